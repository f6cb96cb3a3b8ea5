// Penalties for repeated tokens, biases of single ids and masks of allowed ids, on
// the logits of a vocabulary shard, for gfx950. For row i of a sequence (its next
// token's logits, and those after its first i drafted tokens), with count = how
// often an id is among the sequence's output tokens and its first i drafts:
//
//   id in the prompt or count > 0:   x <- x / r where x > 0, else x r
//   count > 0:                       x <- x - f count - p
//   then x + the id's biases (in their order), and -inf where it is not allowed.
//
// Few of a row's ids are touched (those of the lists), so the row goes by in two
// steps: the dense one copies it under its mask, 16 bytes a load, and the sparse one
// writes the touched elements over it, in 64 bits rounded once. What bounds a batch is
// one read and one write of the logits; in place, without a mask, the lists.
//
// A workgroup holds one sequence's counts of a slab of the vocabulary in LDS, so a
// list is read once by every slab (from the L2 after the first) and nothing of the
// vocabulary's size is kept in memory. The counts are integers: their order does not
// matter.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "nmce.h"
#include "nmce_device.h"

namespace nmce {
namespace {

constexpr int kSlab = 8192;               // ids of a workgroup: 32 KiB of counts
constexpr uint32_t kPrompt = 1u << 31;    // of a count: the id is in the prompt,
constexpr uint32_t kBiased = 1u << 30;    // has a bias,
constexpr uint32_t kTimes = kBiased - 1;  // and comes so often in output and drafts
constexpr float kInf = __builtin_huge_valf();

// The bits of kVec allowed ids from global id g on, the first in bit 0.
template <int kVec>
__device__ __forceinline__ uint32_t allowed_bits(const uint32_t* __restrict__ words, int64_t g,
                                                 int64_t total) {
  const int64_t last = g + kVec <= total ? g + kVec - 1 : total - 1;
  const uint64_t lo = words[g >> 5], hi = words[last >> 5];
  return static_cast<uint32_t>((lo | hi << 32) >> (g & 31));
}

// z to T, rounded once: to bf16 through an fp32 whose last bit is set where the
// conversion cut something off (to odd), which a second rounding cannot take for a tie.
__device__ __forceinline__ void store_rounded(float* p, double z) { *p = static_cast<float>(z); }
__device__ __forceinline__ void store_rounded(uint16_t* p, double z) {
  const float f = static_cast<float>(z);
  uint32_t u = __float_as_uint(f);
  const double back = static_cast<double>(f);
  if (back != z && z == z) {
    if (fabs(back) > fabs(z)) --u;  // towards zero
    u |= 1u;
  }
  *p = f32_to_bf16(__uint_as_float(u));
}

struct Penalties {
  double r, f, p;
  __device__ __forceinline__ bool none() const { return r == 1.0 && f == 0.0 && p == 0.0; }
  __device__ __forceinline__ double on(double x, uint32_t word) const {
    const uint32_t times = word & kTimes;
    if ((word & (kPrompt | kTimes)) && r != 1.0) x = x > 0.0 ? x / r : x * r;
    if (times) x = x - f * static_cast<double>(times) - p;
    return x;
  }
};

__device__ __forceinline__ double of_sequence(const float* each, double all, int64_t b) {
  return each ? static_cast<double>(each[b]) : all;
}

// Part `part` of sequence b's rows, slab `slab` of the vocabulary.
template <typename T, int kBlock, bool kInPlace>
__global__ __launch_bounds__(kBlock) void adjust_kernel(nmce_adjust_batch a, int64_t slabs,
                                                        int64_t parts, int64_t rows_each) {
  constexpr int kVec = Elem<T>::kPerVec;
  constexpr int kEach = kSlab / kBlock / kVec;  // vectors of a thread
  __shared__ __align__(16) uint32_t count[kSlab];
  __shared__ uint16_t touched[kSlab];
  __shared__ int n_touched, repeated;
  const int tid = threadIdx.x;
  const int64_t bp = blockIdx.x / slabs, slab = blockIdx.x - bp * slabs;
  const int64_t b = bp / parts, part = bp - b * parts;
  const int64_t first = part * rows_each;
  const int64_t last = first + rows_each < a.rows ? first + rows_each : a.rows;
  const int64_t c0 = slab * kSlab;
  const int64_t left = a.vocab_local - c0;
  const int width = static_cast<int>(left < kSlab ? left : kSlab);
  const int64_t g0 = a.vocab_start + c0;  // the slab's first global id
  const T* x = static_cast<const T*>(a.logits) + b * a.logits_batch_stride + c0;
  T* y = static_cast<T*>(a.out) + b * a.out_batch_stride + c0;

  // The first row's vectors are on their way while the lists are counted.
  u32x4 v[kEach];
  auto load_row = [&](int64_t row) {
    const T* p = x + row * a.logits_row_stride;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int c = (k * kBlock + tid) * kVec;
      if (c + kVec <= width) memcpy(&v[k], p + c, 16);
    }
  };
  if constexpr (!kInPlace) load_row(first);

  for (int i = tid * 4; i < kSlab; i += kBlock * 4)
    *reinterpret_cast<u32x4*>(count + i) = u32x4{0u, 0u, 0u, 0u};
  if (tid == 0) n_touched = repeated = 0;
  __syncthreads();

  Penalties pen;
  pen.r = of_sequence(a.repetition, a.repetition_all, b);
  pen.f = of_sequence(a.frequency, a.frequency_all, b);
  pen.p = of_sequence(a.presence, a.presence_all, b);
  if (!(pen.r > 0.0 && pen.r < static_cast<double>(kInf))) pen.r = 1.0;
  // An id's place in the slab, or kSlab and above.
  auto place = [&](int64_t id) {
    const uint64_t s = static_cast<uint64_t>(id) - static_cast<uint64_t>(g0);
    return s < static_cast<uint64_t>(width) ? static_cast<int>(s) : kSlab;
  };
  auto note = [&](int s, uint32_t old) {
    if (old == 0) touched[atomicAdd(&n_touched, 1)] = static_cast<uint16_t>(s);
  };
  auto count_list = [&](const int64_t* __restrict__ ids, int64_t n, bool prompt) {
    for (int64_t j = tid; j < n; j += kBlock) {
      const int s = place(ids[j]);
      if (s < kSlab) note(s, prompt ? atomicOr(&count[s], kPrompt) : atomicAdd(&count[s], 1u));
    }
  };
  if (!pen.none()) {
    if (pen.r != 1.0) count_list(a.prompt + b * a.prompt_stride, a.n_prompt, true);
    count_list(a.output + b * a.output_stride, a.n_output, false);
    count_list(a.drafts + b * a.drafts_stride, first, false);
  }
  const int64_t* bias_ids = a.bias_ids + b * a.bias_ids_stride;
  const float* bias = a.bias + b * a.bias_stride;
  for (int64_t j = tid; j < a.n_bias; j += kBlock) {
    const int s = place(bias_ids[j]);
    if (s < kSlab && (atomicOr(&count[s], kBiased) & kBiased)) repeated = 1;
  }
  __syncthreads();

  for (int64_t row = first; row < last; ++row) {
    const T* xr = x + row * a.logits_row_stride;
    T* yr = y + row * a.out_row_stride;
    const uint32_t* words =
        a.allowed ? a.allowed + b * a.allowed_batch_stride + row * a.allowed_row_stride : nullptr;
    auto allowed = [&](int s) {
      return !words || (words[(g0 + s) >> 5] >> ((g0 + s) & 31) & 1u);
    };
    if (!kInPlace || words) {
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        const int c = (k * kBlock + tid) * kVec;
        if (c + kVec > width) break;
        constexpr uint32_t kAll = (1u << kVec) - 1;
        const uint32_t bits = words ? allowed_bits<kVec>(words, g0 + c, a.vocab_total) & kAll
                                    : kAll;
        if (kInPlace) {
          // All allowed: nothing to write; none: nothing to read.
          if (bits == kAll) continue;
          if (bits != 0) memcpy(&v[k], xr + c, 16);
        }
        if (bits != kAll) {
          float f[kVec];
          Elem<T>::unpack(v[k], f);
#pragma unroll
          for (int e = 0; e < kVec; ++e) f[e] = bits >> e & 1u ? f[e] : -kInf;
          v[k] = Elem<T>::pack(f);
        }
        memcpy(yr + c, &v[k], 16);
      }
      // The shard's last elements, of no whole vector.
      const int c = width / kVec * kVec + tid;
      if (c < width) {
        if (!allowed(c)) Elem<T>::store1(yr + c, -kInf);
        else if (!kInPlace) yr[c] = xr[c];
      }
      // The dense stores have reached the memory before any thread of the workgroup
      // stores an element over them.
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
    if (!kInPlace && row + 1 < last) load_row(row + 1);
    auto put = [&](int s, uint32_t word, double add) {
      if (!allowed(s)) return;
      const double z = pen.on(static_cast<double>(Elem<T>::load1(xr + s)), word);
      store_rounded(yr + s, z + add);
    };
    const int n = n_touched;
    for (int t = tid; t < n; t += kBlock) {
      const int s = touched[t];
      const uint32_t word = count[s];
      if (!(word & kBiased)) put(s, word, 0.0);
    }
    for (int64_t j = tid; j < a.n_bias; j += kBlock) {
      const int64_t id = bias_ids[j];
      const int s = place(id);
      if (s >= kSlab) continue;
      double add = bias[j];
      if (repeated) {
        // The first entry of an id adds all of them, in their order.
        bool mine = true;
        for (int64_t i = 0; i < j && mine; ++i) mine = bias_ids[i] != id;
        if (!mine) continue;
        for (int64_t i = j + 1; i < a.n_bias; ++i)
          if (bias_ids[i] == id) add += static_cast<double>(bias[i]);
      }
      put(s, count[s], add);
    }
    if (row + 1 < last && !pen.none()) {
      __syncthreads();  // every thread is done with this row's counts
      if (tid == 0) {
        const int s = place(a.drafts[b * a.drafts_stride + row]);
        if (s < kSlab) note(s, atomicAdd(&count[s], 1u));
      }
      __syncthreads();
    }
  }
}

int check_batch(const nmce_adjust_batch* a) {
  if (!a) return NMCE_EINVAL_PTR;
  if (a->dtype != NMCE_F32 && a->dtype != NMCE_BF16) return NMCE_EINVAL_DTYPE;
  const int64_t most = (int64_t{1} << 31) - 1;
  if (a->batch < 0 || a->batch > most || a->rows < 1 || a->rows > most || a->vocab_local < 1 ||
      a->vocab_local > most || a->vocab_start < 0 || a->vocab_total > most ||
      a->vocab_total < a->vocab_local || a->vocab_start > a->vocab_total - a->vocab_local)
    return NMCE_EINVAL_SHAPE;
  // What a count holds; the biases are searched for an id that comes twice.
  if (a->n_prompt < 0 || a->n_output < 0 || a->n_output > (int64_t{1} << 29) ||
      a->rows > (int64_t{1} << 28) || a->n_bias < 0 || a->n_bias > NMCE_ADJUST_MAX_BIASES)
    return NMCE_EINVAL_SHAPE;
  const int64_t slabs = (a->vocab_local + kSlab - 1) / kSlab;
  // A launch's workgroups times their threads fit 32 bits.
  if (a->batch > (int64_t{1} << 21) || a->batch * a->rows > (int64_t{1} << 21) ||
      a->batch * a->rows * slabs > (int64_t{1} << 21))
    return NMCE_EINVAL_SHAPE;
  if (a->batch == 0) return NMCE_OK;
  if (!a->logits || !a->out || (a->n_prompt > 0 && !a->prompt) ||
      (a->n_output > 0 && !a->output) || (a->n_bias > 0 && (!a->bias_ids || !a->bias)))
    return NMCE_EINVAL_PTR;
  const uintptr_t es = a->dtype == NMCE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a->logits) % es || reinterpret_cast<uintptr_t>(a->out) % es ||
      reinterpret_cast<uintptr_t>(a->allowed) % 4)
    return NMCE_EINVAL_ALIGN;
  return NMCE_OK;
}

}  // namespace
}  // namespace nmce

using namespace nmce;

extern "C" {

int nmce_adjust_logits(const nmce_adjust_batch* a, void* stream) {
  if (const int st = check_batch(a)) return st;
  if (a->batch == 0) return NMCE_OK;
  const int64_t slabs = (a->vocab_local + kSlab - 1) / kSlab;
  nmce_adjust_batch g = *a;
  if (!g.drafts) {
    g.drafts_stride = 0;
    if (g.rows > 1) return NMCE_EINVAL_PTR;
  }
  const bool in_place = a->logits == a->out;
  if (in_place && (a->logits_batch_stride != a->out_batch_stride ||
                   a->logits_row_stride != a->out_row_stride))
    return NMCE_EINVAL_SHAPE;
  const int64_t parts = 1, rows_each = a->rows;
  const dim3 grid(static_cast<unsigned>(a->batch * parts * slabs));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto run = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, g, slabs, parts, rows_each);
  };
  if (a->dtype == NMCE_F32)
    in_place ? run(adjust_kernel<float, 256, true>, 256)
             : run(adjust_kernel<float, 256, false>, 256);
  else
    in_place ? run(adjust_kernel<uint16_t, 256, true>, 256)
             : run(adjust_kernel<uint16_t, 256, false>, 256);
  return launch_status();
}

}  // extern "C"
