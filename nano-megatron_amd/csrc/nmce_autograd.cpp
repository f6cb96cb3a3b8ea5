// The drop-in loss's one-pass path at TP = 1, the embedding lookup, and the
// distillation loss at TP = 1, as C++ autograd nodes; and the calls of the adjusted and
// the top logits.
//
// Forward and backward of cross_entropy.py:16-65 followed by the wrapper's
// .mean() (:85), for the rows the one-pass kernel takes: one launch of
// nmce_ce_fwd_bwd writes the per-token loss, the row statistics and the
// gradient of the mean for the assumed upstream value; the backward launches
// nmce_ce_grad_rescale_unless (gradient in the logits' storage) or
// nmce_ce_bwd_scaled_unless (a separate buffer), which leave it as it is when
// the upstream value is the assumed one. Host code only: the kernels are
// libnmce.so's, reached through its C ABI (include/nmce.h).
//
// A node written in Python costs the autograd engine a hand-over to the
// interpreter on its device thread for every backward, and the forward's
// Python bookkeeping besides: tens of microseconds per call, which a small
// batch (a step of a few tens of microseconds of kernels) pays in full. The
// Python wrapper still validates the arguments and resolves the upstream
// hint; the target check of cross_entropy.py:79-81 runs here too
// (one_pass_mean_checked).
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <ATen/TensorUtils.h>
#include <ATen/core/DimVector.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <atomic>
#include <chrono>
#include <map>
#include <memory>
#include <mutex>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "nmce.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int status, const char* what) {
  TORCH_CHECK(status == 0, "nmce: ", what, " failed with status ", status, ": ",
              nmce_status_string(status));
}

int dtype_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kFloat) return NMCE_F32;
  if (t.scalar_type() == at::kBFloat16) return NMCE_BF16;
  TORCH_CHECK(false, "nmce: unsupported logits dtype ", t.scalar_type());
  return -1;
}

hipStream_t stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// A saved tensor as it came back, which saved-tensor hooks may have replaced: the
// kernels read it at its address, so it has to be on the device, of the type and of
// the shape that went in. (Strides are its own.)
const at::Tensor& came_back(const at::Tensor& t, const at::Device& device, at::ScalarType type,
                            at::IntArrayRef shape, const char* what) {
  TORCH_CHECK(t.defined() && t.device() == device && t.scalar_type() == type &&
                  t.sizes() == shape,
              "nmce: saved-tensor hooks handed the backward other ", what, " than were saved: ",
              type, " ", shape, " on ", device, " became ",
              t.defined() ? c10::str(t.scalar_type(), " ", t.sizes(), " on ", t.device())
                          : std::string("nothing"));
  return t;
}

// The same for the nodes that are Python's: what they saved, noted at the forward and
// compared at the backward. (In Python the two took 10 us of a small fused step's 137 on
// the host; through pybind's conversion of the tensors 6, taken out of the tuple 3.)
class SavedAs {
 public:
  explicit SavedAs(const pybind11::tuple& tensors) {
    was_.reserve(tensors.size());
    for (size_t i = 0; i < tensors.size(); ++i) {
      PyObject* o = PyTuple_GET_ITEM(tensors.ptr(), i);
      if (o == Py_None) {
        was_.emplace_back();
        continue;
      }
      TORCH_CHECK_TYPE(THPVariable_Check(o), "nmce: saved tensors are tensors or None");
      const at::Tensor& t = THPVariable_Unpack(o);
      was_.push_back(Was{t.device(), t.scalar_type(), at::DimVector(t.sizes())});
    }
  }
  // Whether all of them are contiguous; raises on another tensor than was saved.
  bool check(const pybind11::tuple& tensors) const {
    TORCH_CHECK(tensors.size() == was_.size(), "nmce: ", tensors.size(), " saved tensors, not ",
                was_.size());
    bool contiguous = true;
    for (size_t i = 0; i < was_.size(); ++i) {
      const auto& was = was_[i];
      if (!was) continue;
      PyObject* o = PyTuple_GET_ITEM(tensors.ptr(), i);
      TORCH_CHECK_TYPE(THPVariable_Check(o), "nmce: saved-tensor hooks handed back no tensor");
      const at::Tensor& t = THPVariable_Unpack(o);
      came_back(t, was->device, was->type, was->shape, "tensors");
      contiguous = contiguous && t.is_contiguous();
    }
    return contiguous;
  }

 private:
  struct Was {
    at::Device device;
    at::ScalarType type;
    at::DimVector shape;
  };
  std::vector<c10::optional<Was>> was_;
};

// Optional per-launch timing: HIP event pairs recorded on the launch stream
// around every launch of this file while enabled, read back by
// take_timeline() (the benchmark's per-call times).
std::mutex g_timeline_lock;
std::atomic<bool> g_timing{false};
std::vector<std::tuple<std::string, hipEvent_t, hipEvent_t>> g_timeline;

template <typename Launch>
void timed(const char* name, hipStream_t st, Launch&& launch) {
  if (!g_timing) {
    check(launch(), name);
    return;
  }
  hipEvent_t a = nullptr, b = nullptr;
  const bool made = hipEventCreate(&a) == hipSuccess && hipEventCreate(&b) == hipSuccess;
  if (!made || hipEventRecord(a, st) != hipSuccess) {
    if (a) (void)hipEventDestroy(a);
    if (b) (void)hipEventDestroy(b);
    TORCH_CHECK(false, "nmce: creating or recording a timing event failed");
  }
  const int status = launch();
  if (hipEventRecord(b, st) != hipSuccess) {
    (void)hipEventSynchronize(a);
    (void)hipEventDestroy(a);
    (void)hipEventDestroy(b);
    check(status, name);
    TORCH_CHECK(false, "nmce: recording a timing event failed");
  }
  {
    std::lock_guard<std::mutex> g(g_timeline_lock);
    g_timeline.emplace_back(name, a, b);
  }
  check(status, name);
}

// Rows off the 16-byte grid or of a ragged width take the ragged entries.
bool is_ragged(const at::Tensor& t, int64_t V, int64_t ld) {
  const int64_t es = t.element_size();
  return (V * es) % 16 != 0 || (ld * es) % 16 != 0 ||
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0;
}

struct OnePassMean : public torch::autograd::Function<OnePassMean> {
  // logits [..., V] viewable as [rows, V], V within the kernel's width (for a
  // separate gradient buffer, rows that share its rows' offsets from a 16-byte
  // boundary; the wrapper checked),
  // target the flat contiguous int64 targets, hint the one-element fp32
  // upstream value to assume, bad_flag the address of the target check's
  // device word (0 without a check; not an autograd input), inplace whether
  // the gradient goes into the logits' storage.
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits,
                            const at::Tensor& target, const at::Tensor& hint, int64_t bad_flag,
                            bool inplace, int64_t vocab_start) {
    const c10::DeviceGuard device_guard(logits.device());
    const int64_t V = logits.size(-1);
    const at::Tensor rows = logits.view({-1, V});
    const int64_t n = rows.size(0);
    const int64_t ld = n > 1 ? rows.stride(0) : V;
    const int code = dtype_code(rows);
    at::Tensor out = at::empty({3, n}, rows.options().dtype(at::kFloat));  // loss, max, sum - 1
    at::Tensor loss = out.select(0, 0);
    at::Tensor row_stat = out.slice(0, 1, 3);
    at::Tensor grad = inplace ? rows : at::empty({n, V}, rows.options());
    const int64_t ldg = inplace ? ld : V;
    at::Tensor assumed = at::empty({1}, out.options());
    hipStream_t st = stream_of(rows);
    float* stats = out.data_ptr<float>();
    const bool ragged = is_ragged(rows, V, ld);
    timed(ragged ? "nmce_ce_fwd_bwd_ragged" : "nmce_ce_fwd_bwd", st, [&] {
      return (ragged ? nmce_ce_fwd_bwd_ragged : nmce_ce_fwd_bwd)(
          rows.data_ptr(), grad.data_ptr(), code, n, V, ld, ldg, target.data_ptr<int64_t>(), stats,
          stats + n, stats + 2 * n, hint.data_ptr<float>(), assumed.data_ptr<float>(),
          reinterpret_cast<const int32_t*>(bad_flag), static_cast<float>(n), st);
    });
    ctx->saved_data["inplace"] = inplace;
    ctx->saved_data["hint"] = hint;  // itself: the backward writes into it
    ctx->saved_data["vocab_start"] = vocab_start;
    ctx->saved_data["handed_out"] = false;
    ctx->saved_data["shape"] = logits.sizes().vec();
    ctx->saved_data["rows"] = n;
    ctx->saved_data["type"] = logits.scalar_type();
    if (inplace) {
      // The logits now hold the gradient: autograd nodes that saved them fail
      // their version check rather than read it.
      torch::autograd::impl::bump_version(logits);
      ctx->saved_data["grad_buf"] = logits.detach();
      ctx->saved_data["ld"] = ld;
      ctx->save_for_backward({target, row_stat, assumed});
    } else {
      ctx->save_for_backward({rows, target, row_stat, grad, assumed});
    }
    return loss.mean();
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad_outputs) {
    const c10::DeviceGuard device_guard(grad_outputs[0].device());
    at::Tensor go = grad_outputs[0].reshape({1});
    if (go.scalar_type() != at::kFloat) go = go.to(at::kFloat);
    go = go.contiguous();
    const bool inplace = ctx->saved_data["inplace"].toBool();
    const at::Tensor hint = ctx->saved_data["hint"].toTensor();
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const int64_t V = shape.back();
    const int64_t n = ctx->saved_data["rows"].toInt();
    const at::ScalarType type = ctx->saved_data["type"].toScalarType();
    const at::Device device = grad_outputs[0].device();
    const variable_list saved = ctx->get_saved_variables();
    variable_list grads(6);
    const size_t first = inplace ? 0 : 1;
    const at::Tensor target =
        came_back(saved[first], device, at::kLong, {n}, "targets").contiguous();
    const at::Tensor row_stat =
        came_back(saved[first + 1], device, at::kFloat, {2, n}, "row statistics").contiguous();
    const at::Tensor& assumed = came_back(saved.back(), device, at::kFloat, {1}, "upstream value");
    if (inplace) {
      TORCH_CHECK(!ctx->saved_data["handed_out"].toBool(),
                  "nmce: a second backward through an in-place one-pass loss needs the logits, "
                  "which now hold the gradient; pass inplace=False to differentiate it twice");
      at::Tensor grad = ctx->saved_data["grad_buf"].toTensor();
      const int64_t ld = ctx->saved_data["ld"].toInt();
      hipStream_t st = stream_of(grad);
      const bool ragged = is_ragged(grad, V, ld);
      timed(ragged ? "nmce_ce_grad_rescale_unless_ragged" : "nmce_ce_grad_rescale_unless", st, [&] {
        return (ragged ? nmce_ce_grad_rescale_unless_ragged : nmce_ce_grad_rescale_unless)(
            grad.data_ptr(), dtype_code(grad), n, V, ld, go.data_ptr<float>(),
            assumed.data_ptr<float>(), hint.data_ptr<float>(), st);
      });
      ctx->saved_data["handed_out"] = true;
      ctx->saved_data["grad_buf"] = at::Tensor();
      grads[0] = grad;
      return grads;
    }
    // Saved-tensor hooks may hand back copies of other strides.
    const at::Tensor& held = came_back(saved[0], device, type, {n, V}, "logits");
    const at::Tensor rows = V > 1 && held.stride(1) != 1 ? held.contiguous() : held;
    const at::Tensor grad = came_back(saved[3], device, type, {n, V}, "gradient").contiguous();
    const int64_t ld = n > 1 ? rows.stride(0) : V;
    const int64_t vocab_start = ctx->saved_data["vocab_start"].toInt();
    const float gdiv = static_cast<float>(n > 1 ? n : 1);
    hipStream_t st = stream_of(rows);
    const float* stats = row_stat.data_ptr<float>();
    if (ctx->saved_data["handed_out"].toBool()) {
      // A second backward through the same graph: the first one's buffer
      // belongs to its consumers; a new one from the logits.
      at::Tensor fresh = at::empty({n, V}, rows.options());
      timed("nmce_ce_bwd_scaled", st, [&] {
        return nmce_ce_bwd_scaled(rows.data_ptr(), fresh.data_ptr(), dtype_code(rows), n, V, ld,
                                  V, target.data_ptr<int64_t>(), vocab_start, stats, stats + n,
                                  go.data_ptr<float>(), 0, gdiv, st);
      });
      grads[0] = fresh.view(shape);
      return grads;
    }
    timed("nmce_ce_bwd_scaled_unless", st, [&] {
      return nmce_ce_bwd_scaled_unless(rows.data_ptr(), grad.data_ptr(), dtype_code(rows), n, V,
                                       ld, V, target.data_ptr<int64_t>(), vocab_start, stats,
                                       stats + n, go.data_ptr<float>(), gdiv,
                                       assumed.data_ptr<float>(), hint.data_ptr<float>(), st);
    });
    ctx->saved_data["handed_out"] = true;
    grads[0] = grad.view(shape);
    return grads;
  }
};

// ---- the target check ------------------------------------------------------
// nmce_validate_targets_once counts the targets outside [0, vocab) into a
// pinned host word (for the ValueError) and a device word that the one-pass
// kernel reads before its first store (it writes nothing when it is nonzero),
// on the loss stream just before the kernel. The host waits for the check's
// event after enqueueing the kernel, so the GPU starts on the loss meanwhile.

// The device word per (device, stream): the check and the kernel run on that
// stream one after the other, so calls on one stream can share it.
std::mutex g_flag_lock;
std::map<std::pair<int, hipStream_t>, at::Tensor> g_flags;

at::Tensor flag_word(const at::Tensor& like, hipStream_t st) {
  std::lock_guard<std::mutex> g(g_flag_lock);
  auto key = std::make_pair(static_cast<int>(like.device().index()), st);
  auto it = g_flags.find(key);
  if (it == g_flags.end())
    it = g_flags.emplace(key, at::empty({1}, like.options().dtype(at::kInt))).first;
  return it->second;
}

// Pinned count words with their events, pooled per device (an event belongs
// to one) and reused once a check has been waited for (the kernel writes the
// words through their host mapping). The pool holds as many as were ever in
// flight at once, each with the words of the largest check it served.
struct CheckSlot {
  at::Tensor host;
  hipEvent_t event = nullptr;
  int device = 0;
};
std::mutex g_slot_lock;
std::map<int, std::vector<CheckSlot>> g_slots;

// A slot of at least `words` words. The caller has made `device` the current one.
CheckSlot take_slot(int device, int64_t words) {
  CheckSlot s;
  s.device = device;
  {
    std::lock_guard<std::mutex> g(g_slot_lock);
    std::vector<CheckSlot>& free = g_slots[device];
    if (!free.empty()) {
      s = std::move(free.back());
      free.pop_back();
    }
  }
  if (!s.event)
    TORCH_CHECK(hipEventCreateWithFlags(&s.event, hipEventDisableTiming) == hipSuccess,
                "nmce: hipEventCreateWithFlags failed");
  if (!s.host.defined() || s.host.numel() < words) {
    int64_t room = 1;
    while (room < words) room *= 2;
    try {
      s.host = at::empty({room}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
    } catch (...) {
      (void)hipEventDestroy(s.event);
      throw;
    }
  }
  return s;
}

// Waits for a recorded check on every way out of the call (the kernel writes
// the pinned word until then), and gives the slot back.
class CheckGuard {
 public:
  CheckGuard(CheckSlot s, int64_t words) : slot_(std::move(s)), words_(words) {}
  int32_t* host() { return slot_.host.data_ptr<int32_t>(); }
  hipEvent_t event() const { return slot_.event; }
  void recorded() { recorded_ = true; }
  // The count, once the check has finished. Polls first (the count is
  // usually there within microseconds of the launch), then blocks.
  int64_t wait() {
    if (recorded_) {
      pybind11::gil_scoped_release nogil;
      const auto until = std::chrono::steady_clock::now() + std::chrono::microseconds(200);
      hipError_t q = hipEventQuery(slot_.event);
      while (q == hipErrorNotReady && std::chrono::steady_clock::now() < until)
        q = hipEventQuery(slot_.event);
      if (q == hipErrorNotReady) q = hipEventSynchronize(slot_.event);
      recorded_ = false;
      TORCH_CHECK(q == hipSuccess, "nmce: waiting for the target check failed: ",
                  hipGetErrorString(q));
    }
    const volatile int32_t* word = slot_.host.data_ptr<int32_t>();
    int64_t count = 0;
    for (int64_t i = 0; i < words_; ++i) count += word[i];
    return count;
  }
  ~CheckGuard() {
    if (recorded_) (void)hipEventSynchronize(slot_.event);
    std::lock_guard<std::mutex> g(g_slot_lock);
    g_slots[slot_.device].push_back(std::move(slot_));
  }

 private:
  CheckSlot slot_;
  int64_t words_;
  bool recorded_ = false;
};

// The check of flat contiguous targets on the current stream of their device,
// its event recorded behind it. With `flag`, that stream's device word, one
// workgroup counts into it and one host word; without, as many workgroups as
// there are slots of targets count into a host word each: 3.5 us at any of 64
// to a million targets, where the one workgroup takes 3.8 at 16384, 16 at
// 131072 and 126 at a million.
std::unique_ptr<CheckGuard> launch_check(const at::Tensor& target, int64_t vocab_total,
                                         const at::Tensor* flag, hipStream_t st) {
  const int64_t n = target.numel();
  const int64_t words = flag ? 1 : nmce_validate_slots(n);
  auto guard = std::make_unique<CheckGuard>(take_slot(target.device().index(), words), words);
  timed(flag ? "nmce_validate_targets_once" : "nmce_validate_targets", st, [&] {
    return flag ? nmce_validate_targets_once(target.data_ptr<int64_t>(), n, vocab_total,
                                             guard->host(), flag->data_ptr<int32_t>(), st)
                : nmce_validate_targets(target.data_ptr<int64_t>(), n, vocab_total,
                                        guard->host(), st);
  });
  if (hipEventRecord(guard->event(), st) != hipSuccess) {
    // The check may still write the slot's words: let it finish first.
    (void)hipStreamSynchronize(st);
    TORCH_CHECK(false, "nmce: hipEventRecord failed");
  }
  guard->recorded();
  return guard;
}

// A target check in flight, for the callers that launch their loss kernels
// from Python meanwhile (they write nothing that a bad target must not touch
// until the host has the count, so no kernel reads it): wait() gives the count of bad targets (once the check
// is over) and the slot back; so does the end of its life.
class TargetCheck {
 public:
  // Any tensor may come here (validate_targets is public): the kernel reads it
  // at its device address, as int64 and without strides.
  TargetCheck(const at::Tensor& target, int64_t vocab_total) {
    TORCH_CHECK_VALUE(target.is_cuda(), "nmce: targets must be on a ROCm device, got ",
                      target.device());
    TORCH_CHECK_TYPE(target.scalar_type() == at::kLong, "nmce: target must be int64, got ",
                     target.scalar_type());
    TORCH_CHECK_VALUE(target.is_contiguous() && target.numel() > 0,
                      "nmce: the target check takes a non-empty contiguous tensor");
    const c10::DeviceGuard device_guard(target.device());
    hipStream_t st = stream_of(target);
    guard_ = launch_check(target, vocab_total, nullptr, st);
  }
  bool query() const { return !guard_ || hipEventQuery(guard_->event()) == hipSuccess; }
  int64_t wait() {
    if (guard_) {
      count_ = guard_->wait();
      guard_.reset();
    }
    return count_;
  }

 private:
  std::unique_ptr<CheckGuard> guard_;
  int64_t count_ = 0;
};

at::Tensor one_pass_mean(const at::Tensor& logits, const at::Tensor& target,
                         const at::Tensor& hint, const c10::optional<at::Tensor>& bad_flag,
                         bool inplace, int64_t vocab_start) {
  const int64_t flag = bad_flag.has_value() && bad_flag->defined()
                           ? reinterpret_cast<int64_t>(bad_flag->data_ptr<int32_t>())
                           : 0;
  return OnePassMean::apply(logits, target, hint, flag, inplace, vocab_start);
}

// one_pass_mean with the target check of cross_entropy.py:79-81 in front:
// raises the reference's ValueError, after the kernel has left everything as
// it was, when a target lies outside [0, vocab_total).
at::Tensor one_pass_mean_checked(const at::Tensor& logits, const at::Tensor& target,
                                 const at::Tensor& hint, int64_t vocab_total, bool inplace,
                                 int64_t vocab_start) {
  const c10::DeviceGuard device_guard(logits.device());
  hipStream_t st = stream_of(logits);
  const at::Tensor flag = flag_word(logits, st);
  const std::unique_ptr<CheckGuard> guard = launch_check(target, vocab_total, &flag, st);
  at::Tensor loss = OnePassMean::apply(logits, target, hint,
                                       reinterpret_cast<int64_t>(flag.data_ptr<int32_t>()),
                                       inplace, vocab_start);
  if (guard->wait() != 0)
    throw pybind11::value_error("target token id is outside the model vocabulary");
  return loss;
}

// The assumed upstream value a one-pass loss's forward used, for tests that
// follow which backward kept the forward's gradient: the saved fp32 word.
at::Tensor assumed_of(const at::Tensor& loss) {
  auto fn = loss.grad_fn();
  TORCH_CHECK(fn, "nmce: not a one-pass loss");
  auto* node = dynamic_cast<torch::autograd::CppNode<OnePassMean>*>(fn.get());
  TORCH_CHECK(node, "nmce: not a one-pass loss");
  const variable_list saved = node->ctx_.get_saved_variables();
  return saved[node->ctx_.saved_data.at("inplace").toBool() ? 2 : 4];
}

// ---- the embedding -----------------------------------------------------------
// One shard's lookup (nmce_embedding_fwd) and the weight's dense gradient
// (nmce_embedding_bwd). The gradient is linear in the output's, so its own
// derivative is the lookup again: a backward under create_graph goes through
// EmbeddingGrad and can be differentiated further.

// [..., h] as rows of contiguous elements: a view where they lie so, else a copy.
at::Tensor rows_of(const at::Tensor& t, int64_t* ld) {
  const int64_t h = t.size(-1), n = h ? t.numel() / h : 0;
  at::Tensor rows;
  if (t.stride(-1) == 1 || h == 1) {
    const std::vector<int64_t> shape = {n, h};
    const auto strides = at::detail::computeStride(t.sizes(), t.strides(), shape);
    if (strides && (n <= 1 || (*strides)[0] >= h)) rows = t.view(shape);
  }
  if (!rows.defined()) rows = t.contiguous().view({n, h});
  *ld = n > 1 ? rows.stride(0) : h;
  return rows;
}

at::Tensor lookup(const at::Tensor& weight, const at::Tensor& flat, at::IntArrayRef lead,
                  int64_t vocab_start, double scale, at::ScalarType out_type) {
  const c10::DeviceGuard device_guard(weight.device());
  const at::Tensor w = weight.detach();
  int64_t ld;
  const at::Tensor rows = rows_of(w, &ld);
  const int64_t v = rows.size(0), h = rows.size(1);
  std::vector<int64_t> shape = lead.vec();
  shape.push_back(h);
  at::Tensor out = at::empty(shape, w.options().dtype(out_type));
  hipStream_t st = stream_of(w);
  timed("nmce_embedding_fwd", st, [&] {
    return nmce_embedding_fwd(flat.data_ptr<int64_t>(), flat.numel(), rows.data_ptr(),
                              dtype_code(rows), v, h, ld, vocab_start, static_cast<float>(scale),
                              out.data_ptr(), dtype_code(out), h, st);
  });
  return out;
}

at::Tensor lookup_grad(const at::Tensor& grad, const at::Tensor& flat, int64_t v,
                       int64_t vocab_start, double scale, at::ScalarType weight_type) {
  const c10::DeviceGuard device_guard(grad.device());
  const at::Tensor g = grad.detach();
  int64_t ld;
  const at::Tensor dy = rows_of(g, &ld);
  const int64_t n = flat.numel(), h = dy.size(1);
  at::Tensor dw = at::empty({v, h}, g.options().dtype(weight_type));
  const int64_t need = nmce_embedding_bwd_workspace_bytes(n, v, h);
  at::Tensor ws = at::empty({need > 16 ? need : 16}, g.options().dtype(at::kByte));
  hipStream_t st = stream_of(g);
  timed("nmce_embedding_bwd", st, [&] {
    return nmce_embedding_bwd(flat.data_ptr<int64_t>(), n, dy.data_ptr(), dtype_code(dy), ld, v, h,
                              vocab_start, static_cast<float>(scale), dw.data_ptr(),
                              dtype_code(dw), ws.data_ptr(), ws.numel(), st);
  });
  return dw;
}

at::Tensor embedding(const at::Tensor& weight, const at::Tensor& tokens, int64_t vocab_start,
                     double scale, at::ScalarType out_type);

// The ids of a node, saved by its forward and taken back by its backward.
void save_ids(AutogradContext* ctx, const at::Tensor& tokens) {
  ctx->saved_data["shape"] = tokens.sizes().vec();
  ctx->save_for_backward({tokens});
}

at::Tensor saved_ids(AutogradContext* ctx, const at::Device& device) {
  const at::Tensor ids = ctx->get_saved_variables()[0];
  return came_back(ids, device, at::kLong, ctx->saved_data["shape"].toIntVector(), "token ids");
}

struct EmbeddingGrad : public torch::autograd::Function<EmbeddingGrad> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& grad,
                            const at::Tensor& tokens, int64_t v, int64_t vocab_start, double scale,
                            at::ScalarType weight_type) {
    ctx->saved_data["start"] = vocab_start;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["type"] = grad.scalar_type();
    save_ids(ctx, tokens);
    return lookup_grad(grad, tokens.reshape({-1}).contiguous(), v, vocab_start, scale,
                       weight_type);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    out[0] = embedding(grads[0], saved_ids(ctx, grads[0].device()),
                       ctx->saved_data["start"].toInt(), ctx->saved_data["scale"].toDouble(),
                       ctx->saved_data["type"].toScalarType());
    return out;
  }
};

struct Embedding : public torch::autograd::Function<Embedding> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& weight,
                            const at::Tensor& tokens, int64_t vocab_start, double scale,
                            at::ScalarType out_type) {
    ctx->saved_data["start"] = vocab_start;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["type"] = weight.scalar_type();
    ctx->saved_data["rows"] = weight.size(0);
    save_ids(ctx, tokens);
    return lookup(weight, tokens.reshape({-1}).contiguous(), tokens.sizes(), vocab_start, scale,
                  out_type);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor tokens = saved_ids(ctx, grads[0].device());
    const int64_t start = ctx->saved_data["start"].toInt(), v = ctx->saved_data["rows"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    const at::ScalarType type = ctx->saved_data["type"].toScalarType();
    variable_list out(5);
    out[0] = at::GradMode::is_enabled() && grads[0].requires_grad()
                 ? EmbeddingGrad::apply(grads[0], tokens, v, start, scale, type)
                 : lookup_grad(grads[0], tokens.reshape({-1}).contiguous(), v, start, scale, type);
    return out;
  }
};

at::Tensor embedding(const at::Tensor& weight, const at::Tensor& tokens, int64_t vocab_start,
                     double scale, at::ScalarType out_type) {
  return Embedding::apply(weight, tokens, vocab_start, scale, out_type);
}

// The entry from Python. It reads device addresses: what would hand it another
// kind of tensor is refused here too (the wrapper has checked the rest).
at::Tensor embedding_entry(const at::Tensor& weight, const at::Tensor& tokens,
                           int64_t vocab_start, double scale, bool f32_out) {
  TORCH_CHECK(weight.is_cuda() && tokens.device() == weight.device() && weight.dim() == 2 &&
                  tokens.scalar_type() == at::kLong,
              "nmce: the embedding takes a [vocabulary, hidden] weight and int64 tokens on one "
              "ROCm device (there is no CPU path)");
  return embedding(weight, tokens, vocab_start, scale, f32_out ? at::kFloat : at::kBFloat16);
}

// ---- distillation from a teacher's top logits ------------------------------------------
// On one rank. DistillMean: nmce_distill_fwd_bwd writes the loss, the mean and its
// gradient for the assumed upstream value in one read of the logits, as OnePassMean does.
// Distill: two passes, each token's loss or their mean.

// A batch for the C entries, and the tensors that it points into.
struct DistillArgs {
  at::Tensor rows, teacher, ids, norm;
  nmce_distill_batch batch{};

  DistillArgs(const at::Tensor& logits, const at::Tensor& teacher_logits,
              const at::Tensor& teacher_ids, const c10::optional<at::Tensor>& normalizer,
              double temperature) {
    const int64_t V = logits.size(-1);
    int64_t ld, t_ld, ids_ld;
    rows = rows_of(logits, &ld);
    teacher = rows_of(teacher_logits, &t_ld);
    ids = rows_of(teacher_ids, &ids_ld);
    if (normalizer.has_value() && normalizer->defined())
      norm = normalizer->reshape({-1}).contiguous();
    batch.logits = rows.data_ptr();
    batch.teacher_logits = teacher.data_ptr();
    batch.teacher_ids = ids.data_ptr<int64_t>();
    batch.teacher_log_normalizer = norm.defined() ? norm.data_ptr<float>() : nullptr;
    batch.ld = ld;
    batch.teacher_ld = t_ld;
    batch.ids_ld = ids_ld;
    batch.n_rows = rows.size(0);
    batch.vocab_local = batch.vocab_total = V;
    batch.temperature = temperature;
    batch.k = static_cast<int>(teacher.size(1));
    batch.dtype = dtype_code(rows);
    batch.teacher_dtype = dtype_code(teacher);
  }
  at::Tensor state() const {
    const int64_t bytes = nmce_distill_state_bytes(batch.n_rows, batch.k);
    return at::empty({bytes > 16 ? bytes : 16}, rows.options().dtype(at::kByte));
  }
};

// What a backward hands out: under create_graph it carries a node that raises when the
// kernels, which have no second derivative, are differentiated again.
at::Tensor once(const at::Tensor& grad) {
  if (!at::GradMode::is_enabled()) return grad;
  auto raise = std::make_shared<torch::autograd::DelayedError>(
      "nmce: the distillation loss cannot be differentiated twice", 1);
  return (*raise)({grad.detach().requires_grad_(true)})[0];
}

at::Tensor distill_grad(AutogradContext* ctx, const at::Tensor& rows, at::Tensor out,
                        const at::Tensor& state, const at::Tensor& go, int64_t stride,
                        const float* assumed, float* observed) {
  const int64_t n = rows.size(0), V = rows.size(1);
  hipStream_t st = stream_of(rows);
  timed("nmce_distill_bwd", st, [&] {
    return nmce_distill_bwd(rows.data_ptr(), out.data_ptr(), dtype_code(rows), n, V,
                            n > 1 ? rows.stride(0) : V, n > 1 ? out.stride(0) : V,
                            static_cast<int>(ctx->saved_data["k"].toInt()),
                            ctx->saved_data["temperature"].toDouble(), state.data_ptr(),
                            state.numel(), go.data_ptr<float>(), stride,
                            static_cast<float>(ctx->saved_data["divisor"].toInt()), assumed,
                            observed, st);
  });
  return out;
}

void save_distill(AutogradContext* ctx, const DistillArgs& a, const at::Tensor& logits,
                  const at::Tensor& state, bool inplace, int64_t divisor) {
  ctx->saved_data["inplace"] = inplace;
  ctx->saved_data["k"] = static_cast<int64_t>(a.batch.k);
  ctx->saved_data["temperature"] = a.batch.temperature;
  ctx->saved_data["divisor"] = divisor;
  ctx->saved_data["shape"] = logits.sizes().vec();
  ctx->saved_data["rows"] = a.batch.n_rows;
  ctx->saved_data["type"] = logits.scalar_type();
  ctx->saved_data["state"] = state.numel();
}

struct DistillMean : public torch::autograd::Function<DistillMean> {
  // logits viewable as rows that nmce_distill_fwd_bwd takes (the wrapper checked).
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits,
                            const at::Tensor& teacher_logits, const at::Tensor& teacher_ids,
                            const c10::optional<at::Tensor>& normalizer, const at::Tensor& hint,
                            double temperature, bool inplace) {
    const c10::DeviceGuard device_guard(logits.device());
    const DistillArgs a(logits, teacher_logits, teacher_ids, normalizer, temperature);
    const int64_t n = a.batch.n_rows, V = a.batch.vocab_local;
    const at::Tensor state = a.state();
    const auto f32 = a.rows.options().dtype(at::kFloat);
    at::Tensor loss = at::empty({n}, f32), mean = at::empty({}, f32), assumed = at::empty({1}, f32);
    // Rows that had to be copied (of an expanded tensor) are not the logits' storage.
    inplace = inplace && a.rows.data_ptr() == logits.data_ptr();
    at::Tensor grad = inplace ? a.rows : at::empty({n, V}, a.rows.options());
    hipStream_t st = stream_of(a.rows);
    timed("nmce_distill_fwd_bwd", st, [&] {
      return nmce_distill_fwd_bwd(&a.batch, grad.data_ptr(), inplace ? a.batch.ld : V,
                                  state.data_ptr(), state.numel(), loss.data_ptr<float>(),
                                  mean.data_ptr<float>(), hint.data_ptr<float>(),
                                  assumed.data_ptr<float>(), static_cast<float>(n), st);
    });
    save_distill(ctx, a, logits, state, inplace, n);
    ctx->saved_data["hint"] = hint;  // itself: the backward writes into it
    ctx->saved_data["handed_out"] = false;
    if (inplace) {
      torch::autograd::impl::bump_version(logits);
      ctx->saved_data["grad_buf"] = logits.detach();
      ctx->saved_data["ld"] = a.batch.ld;
      ctx->save_for_backward({assumed});
    } else {
      ctx->save_for_backward({a.rows, state, grad, assumed});
    }
    return mean;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad_outputs) {
    const c10::DeviceGuard device_guard(grad_outputs[0].device());
    const at::Tensor go = grad_outputs[0].detach().reshape({1}).to(at::kFloat).contiguous();
    const at::Tensor hint = ctx->saved_data["hint"].toTensor();
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const int64_t V = shape.back(), n = ctx->saved_data["rows"].toInt();
    const at::Device device = grad_outputs[0].device();
    const at::ScalarType type = ctx->saved_data["type"].toScalarType();
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor& assumed = came_back(saved.back(), device, at::kFloat, {1}, "upstream value");
    variable_list grads(7);
    if (ctx->saved_data["inplace"].toBool()) {
      TORCH_CHECK(!ctx->saved_data["handed_out"].toBool(),
                  "nmce: a second backward through an in-place one-pass loss needs the logits, "
                  "which now hold the gradient; pass inplace=False to differentiate it twice");
      at::Tensor grad = ctx->saved_data["grad_buf"].toTensor();
      const int64_t ld = ctx->saved_data["ld"].toInt();
      hipStream_t st = stream_of(grad);
      const bool ragged = is_ragged(grad, V, ld);
      timed(ragged ? "nmce_ce_grad_rescale_unless_ragged" : "nmce_ce_grad_rescale_unless", st, [&] {
        return (ragged ? nmce_ce_grad_rescale_unless_ragged : nmce_ce_grad_rescale_unless)(
            grad.data_ptr(), dtype_code(grad), n, V, ld, go.data_ptr<float>(),
            assumed.data_ptr<float>(), hint.data_ptr<float>(), st);
      });
      ctx->saved_data["handed_out"] = true;
      ctx->saved_data["grad_buf"] = at::Tensor();
      grads[0] = once(grad);
      return grads;
    }
    // Saved-tensor hooks may hand back copies of other strides.
    const at::Tensor& held = came_back(saved[0], device, type, {n, V}, "logits");
    const at::Tensor rows = V > 1 && held.stride(1) != 1 ? held.contiguous() : held;
    const at::Tensor state = came_back(saved[1], device, at::kByte,
                                       {ctx->saved_data["state"].toInt()}, "state").contiguous();
    if (ctx->saved_data["handed_out"].toBool()) {
      // The first backward's buffer belongs to its consumers; a new one.
      grads[0] = once(distill_grad(ctx, rows, at::empty({n, V}, rows.options()), state, go, 0,
                                   nullptr, nullptr).view(shape));
      return grads;
    }
    const at::Tensor grad = came_back(saved[2], device, type, {n, V}, "gradient").contiguous();
    distill_grad(ctx, rows, grad, state, go, 0, assumed.data_ptr<float>(), hint.data_ptr<float>());
    ctx->saved_data["handed_out"] = true;
    grads[0] = once(grad.view(shape));
    return grads;
  }
};

struct Distill : public torch::autograd::Function<Distill> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits,
                            const at::Tensor& teacher_logits, const at::Tensor& teacher_ids,
                            const c10::optional<at::Tensor>& normalizer, double temperature,
                            bool mean, bool inplace) {
    const c10::DeviceGuard device_guard(logits.device());
    const DistillArgs a(logits, teacher_logits, teacher_ids, normalizer, temperature);
    const int64_t n = a.batch.n_rows;
    const at::Tensor state = a.state();
    at::Tensor loss = at::empty({n}, a.rows.options().dtype(at::kFloat));
    at::Tensor stats = at::empty({n, 5}, a.rows.options().dtype(at::kDouble));
    at::Tensor result = mean && n > 0 ? at::empty({}, loss.options()) : at::Tensor();
    hipStream_t st = stream_of(a.rows);
    timed("nmce_distill_stats", st, [&] {
      return nmce_distill_stats(&a.batch, state.data_ptr(), state.numel(),
                                stats.data_ptr<double>(), st);
    });
    timed("nmce_distill_combine", st, [&] {
      return nmce_distill_combine(state.data_ptr(), state.numel(), n, a.batch.k, temperature,
                                  stats.data_ptr<double>(), 1, loss.data_ptr<float>(),
                                  result.defined() ? result.data_ptr<float>() : nullptr, st);
    });
    // Rows that had to be copied are not the logits' storage.
    inplace = inplace && a.rows.data_ptr() == logits.data_ptr();
    save_distill(ctx, a, logits, state, inplace, mean && n > 1 ? n : 1);
    ctx->saved_data["mean"] = mean;
    if (inplace) ctx->save_for_backward({a.rows, state, logits});
    else ctx->save_for_backward({a.rows, state});
    if (mean) return result.defined() ? result : loss.mean();  // (of no tokens: NaN)
    return loss.view(logits.sizes().slice(0, logits.dim() - 1));
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad_outputs) {
    const c10::DeviceGuard device_guard(grad_outputs[0].device());
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const int64_t V = shape.back(), n = ctx->saved_data["rows"].toInt();
    const at::Device device = grad_outputs[0].device();
    const at::ScalarType type = ctx->saved_data["type"].toScalarType();
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor& held = came_back(saved[0], device, type, {n, V}, "logits");
    const at::Tensor rows = V > 1 && held.stride(1) != 1 ? held.contiguous() : held;
    const at::Tensor state = came_back(saved[1], device, at::kByte,
                                       {ctx->saved_data["state"].toInt()}, "state").contiguous();
    // A broadcast upstream value (a sum's or the mean's) is read where it is.
    at::Tensor go = grad_outputs[0].detach().to(at::kFloat);
    int64_t stride = 0;
    if (!ctx->saved_data["mean"].toBool()) {
      for (int64_t d = 0; d < go.dim(); ++d) stride = go.stride(d) != 0 ? 1 : stride;
      if (stride) go = go.reshape({-1}).contiguous();
    }
    variable_list grads(7);
    const bool inplace = ctx->saved_data["inplace"].toBool();
    at::Tensor original, out;
    if (inplace) {
      original = came_back(saved[2], device, type, shape, "logits");
      int64_t ld;
      out = rows_of(original, &ld);
    } else {
      out = at::empty({n, V}, rows.options());
    }
    distill_grad(ctx, rows, out, state, go, stride, nullptr, nullptr);
    if (inplace && out.data_ptr() == original.data_ptr()) {
      // The logits hold the gradient: readers that saved them fail their version check.
      torch::autograd::impl::bump_version(original);
      grads[0] = once(original.detach());
    } else {
      grads[0] = once(out.view(shape));
    }
    return grads;
  }
};

// The entries from Python. They read device addresses: what would hand them other kinds of
// tensors is refused here too (the wrapper has checked the rest).
void check_distill(const at::Tensor& logits, const at::Tensor& teacher_logits,
                   const at::Tensor& teacher_ids, const c10::optional<at::Tensor>& normalizer) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() > 0 && logits.size(-1) > 0 &&
                  teacher_logits.device() == logits.device() &&
                  teacher_ids.device() == logits.device() &&
                  teacher_ids.scalar_type() == at::kLong && teacher_logits.dim() > 0 &&
                  teacher_ids.sizes() == teacher_logits.sizes() &&
                  teacher_ids.sizes().slice(0, teacher_ids.dim() - 1) ==
                      logits.sizes().slice(0, logits.dim() - 1) &&
                  (!normalizer.has_value() ||
                   (normalizer->device() == logits.device() &&
                    normalizer->scalar_type() == at::kFloat &&
                    normalizer->sizes() == logits.sizes().slice(0, logits.dim() - 1))),
              "nmce: the distillation loss takes logits [..., vocabulary], teacher logits and "
              "int64 ids [..., listed] and fp32 normalisers [...] on one ROCm device (there is no "
              "CPU path)");
}

at::Tensor distill_mean(const at::Tensor& logits, const at::Tensor& teacher_logits,
                        const at::Tensor& teacher_ids,
                        const c10::optional<at::Tensor>& normalizer, const at::Tensor& hint,
                        double temperature, bool inplace) {
  check_distill(logits, teacher_logits, teacher_ids, normalizer);
  return DistillMean::apply(logits, teacher_logits, teacher_ids, normalizer, hint, temperature,
                            inplace);
}

at::Tensor distill(const at::Tensor& logits, const at::Tensor& teacher_logits,
                   const at::Tensor& teacher_ids, const c10::optional<at::Tensor>& normalizer,
                   double temperature, bool mean, bool inplace) {
  check_distill(logits, teacher_logits, teacher_ids, normalizer);
  return Distill::apply(logits, teacher_logits, teacher_ids, normalizer, temperature, mean,
                        inplace);
}

// ---- logits on their way to a sampler ---------------------------------------------------
// No nodes (they have no derivative), but one call from Python each: through ctypes, with
// its outputs made there, a small call took 19 (adjust) and 16 us (top) on the host, and takes 11 and 7.

// Lists [batch, n] of consecutive elements: their address, stride and length.
struct Lists {
  at::Tensor held;
  const void* at = nullptr;
  int64_t stride = 0, n = 0;
  explicit Lists(const c10::optional<at::Tensor>& t) {
    if (!t.has_value() || !t->defined() || t->numel() == 0) return;
    held = t->size(1) > 1 && t->stride(1) != 1 ? t->contiguous() : *t;
    at = held.data_ptr();
    stride = held.stride(0);
    n = held.size(1);
  }
};

// (The wrapper has checked the arguments; what is no address on the device is refused here.)
at::Tensor adjust(const at::Tensor& logits, const c10::optional<at::Tensor>& prompt,
                  const c10::optional<at::Tensor>& output,
                  const c10::optional<at::Tensor>& drafts,
                  const std::vector<c10::optional<at::Tensor>>& penalties,
                  const std::vector<double>& alike, const c10::optional<at::Tensor>& bias_ids,
                  const c10::optional<at::Tensor>& bias,
                  const c10::optional<at::Tensor>& allowed, int64_t vocab_start,
                  int64_t vocab_total, bool inplace) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 3 && penalties.size() == 3 && alike.size() == 3,
              "nmce: logits are adjusted as [batch, rows, vocabulary] on a ROCm device (there is "
              "no CPU path)");
  for (const auto* t : {&prompt, &output, &drafts, &bias_ids, &bias, &allowed, &penalties[0],
                        &penalties[1], &penalties[2]})
    TORCH_CHECK(!t->has_value() || (*t)->device() == logits.device(),
                "nmce: lists, penalties and masks on another device than the logits");
  const c10::DeviceGuard device_guard(logits.device());
  const int64_t v = logits.size(2);
  const at::Tensor x =
      inplace || v == 1 || logits.stride(2) == 1 ? logits.detach() : logits.detach().contiguous();
  at::Tensor out = inplace ? logits : at::empty(logits.sizes(), logits.options());
  const Lists p(prompt), o(output), d(drafts), bi(bias_ids), bv(bias);
  at::Tensor mask, each[3];
  if (allowed.has_value())
    mask = allowed->size(2) > 1 && allowed->stride(2) != 1 ? allowed->contiguous() : *allowed;
  const float* values[3] = {nullptr, nullptr, nullptr};
  for (int i = 0; i < 3; ++i) {
    if (!penalties[i].has_value()) continue;
    each[i] = penalties[i]->contiguous();
    values[i] = each[i].data_ptr<float>();
  }
  nmce_adjust_batch a{};
  a.logits = x.data_ptr();
  a.out = out.data_ptr();
  a.prompt = static_cast<const int64_t*>(p.at);
  a.output = static_cast<const int64_t*>(o.at);
  a.drafts = static_cast<const int64_t*>(d.at);
  a.bias_ids = static_cast<const int64_t*>(bi.at);
  a.bias = static_cast<const float*>(bv.at);
  a.allowed = mask.defined() ? static_cast<const uint32_t*>(mask.data_ptr()) : nullptr;
  a.repetition = values[0];
  a.frequency = values[1];
  a.presence = values[2];
  a.logits_batch_stride = x.stride(0);
  a.logits_row_stride = x.stride(1);
  a.out_batch_stride = out.stride(0);
  a.out_row_stride = out.stride(1);
  a.prompt_stride = p.stride;
  a.output_stride = o.stride;
  a.drafts_stride = d.stride;
  a.bias_ids_stride = bi.stride;
  a.bias_stride = bv.stride;
  a.allowed_batch_stride = mask.defined() ? mask.stride(0) : 0;
  a.allowed_row_stride = mask.defined() ? mask.stride(1) : 0;
  a.n_prompt = p.n;
  a.n_output = o.n;
  a.n_bias = bi.n;
  a.batch = logits.size(0);
  a.rows = logits.size(1);
  a.vocab_local = v;
  a.vocab_start = vocab_start;
  a.vocab_total = vocab_total;
  a.repetition_all = alike[0];
  a.frequency_all = alike[1];
  a.presence_all = alike[2];
  a.dtype = dtype_code(x);
  hipStream_t st = stream_of(x);
  timed("nmce_adjust_logits", st, [&] { return nmce_adjust_logits(&a, st); });
  // (Inference tensors have no version.)
  if (inplace && !logits.is_inference()) torch::autograd::impl::bump_version(logits);
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> top(const at::Tensor& logits, int64_t k,
                                                   double temperature) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() > 0,
              "nmce: top logits are taken on a ROCm device (there is no CPU path)");
  const c10::DeviceGuard device_guard(logits.device());
  std::vector<int64_t> lead = logits.sizes().vec();
  const int64_t v = lead.back();
  lead.pop_back();
  std::vector<int64_t> shape = lead;
  shape.push_back(k);
  at::Tensor values = at::empty(shape, logits.options());
  at::Tensor ids = at::empty(shape, logits.options().dtype(at::kLong));
  at::Tensor norm = at::empty(lead, logits.options().dtype(at::kFloat));
  if (logits.numel() == 0) return {values, ids, norm};
  int64_t ld;
  const at::Tensor rows = rows_of(logits.detach(), &ld);
  const int64_t n = rows.size(0);
  const int64_t bytes = nmce_top_workspace_bytes(n, v, static_cast<int>(k));
  at::Tensor ws = at::empty({bytes > 16 ? bytes : 16}, logits.options().dtype(at::kByte));
  hipStream_t st = stream_of(rows);
  timed("nmce_top_logits", st, [&] {
    return nmce_top_logits(rows.data_ptr(), dtype_code(rows), n, v, ld, 0, static_cast<int>(k),
                           temperature, nullptr, values.data_ptr(), ids.data_ptr<int64_t>(),
                           norm.data_ptr<float>(), ws.data_ptr(), ws.numel(), st);
  });
  return {values, ids, norm};
}

void set_timing(bool on) { g_timing = on; }

// (name, milliseconds) of every launch timed since the last call, in launch
// order; waits for the last of them.
std::vector<std::tuple<std::string, double>> take_timeline() {
  std::vector<std::tuple<std::string, hipEvent_t, hipEvent_t>> events;
  {
    std::lock_guard<std::mutex> g(g_timeline_lock);
    events.swap(g_timeline);
  }
  std::vector<std::tuple<std::string, double>> out;
  bool ok = true;
  for (auto& [name, a, b] : events) {
    float ms = 0.0f;
    ok = ok && hipEventSynchronize(b) == hipSuccess &&
         hipEventElapsedTime(&ms, a, b) == hipSuccess;
    (void)hipEventDestroy(a);
    (void)hipEventDestroy(b);
    out.emplace_back(name, ms);
  }
  TORCH_CHECK(ok, "nmce: reading a launch's HIP events failed");
  return out;
}

// For measurements (no counterpart in the reference): an autograd node that
// stands where the LM-head matmul is (model.py:192). Its forward hands the
// resident logits on as a non-leaf alias, its backward receives d(logits)
// and hands nothing further, as a C++ node, as the matmul's own backward
// is, so a timed step carries no Python node of its own.
struct HeadOutput : public torch::autograd::Function<HeadOutput> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits,
                            const at::Tensor& anchor) {
    (void)ctx;
    (void)anchor;
    return logits.alias();
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    (void)ctx;
    (void)grads;
    return {at::Tensor(), at::Tensor()};
  }
};

at::Tensor head_output(const at::Tensor& logits, const at::Tensor& anchor) {
  return HeadOutput::apply(logits, anchor);
}

}  // namespace

PYBIND11_MODULE(_nmce_autograd, m) {
  m.doc() = "The one-pass loss at TP = 1, the embedding and the distillation loss at TP = 1 as C++ "
            "autograd nodes over libnmce's C ABI.";
  m.def("one_pass_mean", &one_pass_mean, "mean one-pass loss (forward + backward in C++)");
  m.def("one_pass_mean_checked", &one_pass_mean_checked,
        "one_pass_mean after the target check; ValueError on a target outside the vocabulary");
  pybind11::class_<TargetCheck>(m, "TargetCheck",
                                "a target check in flight on the targets' current stream")
      .def(pybind11::init<const at::Tensor&, int64_t>())
      .def("query", &TargetCheck::query, "whether the check is over")
      .def("wait", &TargetCheck::wait, "wait for it; the count of bad targets");
  pybind11::class_<SavedAs>(m, "SavedAs", "device, type and shape of the tensors a node saves")
      .def(pybind11::init<const pybind11::tuple&>())
      .def("check", &SavedAs::check,
           "RuntimeError unless the tensors are such as were saved; whether all are contiguous");
  m.def("assumed_of", &assumed_of, "the assumed upstream value saved by a one-pass loss");
  m.def("embedding", &embedding_entry,
        "a vocabulary shard's scaled lookup, with the weight's dense gradient");
  m.def("distill_mean", &distill_mean, "mean one-pass distillation loss of one rank");
  m.def("distill", &distill, "distillation losses of one rank, or their mean, in two passes");
  m.def("adjust", &adjust, "penalties, biases and masks on logits, in one call");
  m.def("top", &top, "a rank's top logits, their ids and the rows' log-normalisers");
  m.def("set_timing", &set_timing, "time every launch with HIP events while on");
  m.def("take_timeline", &take_timeline, "(name, ms) of the launches timed since the last call");
  m.def("head_output", &head_output,
        "logits as a non-leaf alias through a C++ node whose backward hands nothing on "
        "(stands for the LM-head matmul in measurements)");
}
