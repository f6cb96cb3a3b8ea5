// Distillation from a teacher's top logits over a vocabulary shard, forward and
// backward, for gfx950. With q = softmax(z / T) of the student's row over the whole
// vocabulary and the teacher's p at K listed ids (p = exp(t / T - its log-normaliser),
// or softmax(t / T) over the list), r = max(1 - sum p, 0) for the rest as one class,
//
//   loss  = sum p (log p - log q) + r (log r - log s)      s = sum of q outside the list
//   dz    = (P q - p) / T  at the list's ids               P = sum p + r
//         = (P q - r q / s) / T  outside (without normaliser r = 0, P = 1)
//
// Outside the list dz = a exp((z - m) / T) with one factor a per row, so the row is read
// for (m, sum of exp((z - m) / T)) outside, and written from it; the list's few elements
// are formed apart. The list's side of it (p, the student's logits there, their sums, in
// 64 bits) is a wave's work per row, done first. An id that comes several times adds up
// its p, in the list's order, at its first place.
//
// With a sharded vocabulary the ranks exchange 40 bytes a row: (m, sum) outside, (m, sum)
// of the list's ids that they hold, and sum p z there.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "nmce.h"
#include "nmce_device.h"

namespace nmce {
namespace {

constexpr int kMaxK = NMCE_DISTILL_MAX_K;
constexpr int kStat = 5;  // doubles of a rank's statistics of a row
constexpr float kInf = __builtin_huge_valf();

// What the list's side of a row comes to.
struct Taught {
  double r;      // the rest's probability (0 without a normaliser)
  double p;      // sum of p
  double h;      // sum of p log p
  double dot;    // sum of p z / T over this shard's ids
  double sum;    // sum of exp((z - top) / T) over this shard's ids, each id once
  float top;     // the largest z there
  int any;       // 0: no teacher for this row
};

// What the backward needs of a row: dz = a exp((z - m) / T) outside the list,
// exp((z - top) / T) b - p at its ids, each times the upstream value / T.
struct Slope {
  float m, a, top, b;
};

// The parts of the state that a forward leaves for its backward.
struct State {
  Taught* rows;
  Slope* slopes;
  int* column;  // [n][k] of this shard; -1: none, another rank's, or said before
  float* p;
  float* z;
};
__host__ __device__ inline State state_of(void* base, int64_t n, int64_t k) {
  char* b = static_cast<char*>(base);
  State s;
  auto take = [&](int64_t bytes) {
    char* p = b;
    b += (bytes + 255) / 256 * 256;
    return p;
  };
  s.rows = reinterpret_cast<Taught*>(take(n * static_cast<int64_t>(sizeof(Taught))));
  s.slopes = reinterpret_cast<Slope*>(take(n * static_cast<int64_t>(sizeof(Slope))));
  s.column = reinterpret_cast<int*>(take(n * k * 4));
  s.p = reinterpret_cast<float*>(take(n * k * 4));
  s.z = reinterpret_cast<float*>(take(n * k * 4));
  return s;
}

__device__ __forceinline__ double wave_add(double v) {
  for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s);
  return v;
}
__device__ __forceinline__ float wave_maxf(float v) {
  for (int s = 32; s > 0; s >>= 1) v = fmaxf(v, __shfl_xor(v, s));
  return v;
}

// ---- the list's side ------------------------------------------------------------
constexpr int kListWaves = 4;

template <typename T, typename TT>
__global__ __launch_bounds__(kListWaves * 64) void distill_list_kernel(nmce_distill_batch a,
                                                                       int table, State st) {
  extern __shared__ int tables[];  // `table` slots a wave: ids noted, 0 for none
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kListWaves + wave;
  if (row >= a.n_rows) return;  // (waves are on their own: no barrier below)
  int* seen = tables + wave * table;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  const TT* t = static_cast<const TT*>(a.teacher_logits) + row * a.teacher_ld;
  const int64_t* ids = a.teacher_ids + row * a.ids_ld;
  const double c = 1.0 / a.temperature;
  const int64_t base = row * a.k;
  auto held = [&](int64_t id) { return id >= 0 && id < a.vocab_total; };

  for (int i = lane; i < table; i += 64) seen[i] = 0;
  __builtin_amdgcn_wave_barrier();
  float top_t = -kInf, top = -kInf;
  bool any = false, again = false;
  for (int j = lane; j < a.k; j += 64) {
    const int64_t id = ids[j];
    if (!held(id)) continue;
    any = true;
    const float tj = Elem<TT>::load1(t + j);
    top_t = tj > top_t || tj != tj ? tj : top_t;
    const int64_t at = id - a.vocab_start;
    if (at >= 0 && at < a.vocab_local) top = fmaxf(top, Elem<T>::load1(x + at));
    // Whether another place names the id: the table holds each once.
    const int mark = static_cast<int>(id) + 1;
    uint32_t h = static_cast<uint32_t>(mark) * 2654435761u >> 7;
    for (;; ++h) {
      const int old = atomicCAS(&seen[h & (table - 1)], 0, mark);
      if (old == 0) break;
      if (old == mark) {
        again = true;
        break;
      }
    }
  }
  any = __any(any);
  again = __any(again);
  for (int s = 32; s > 0; s >>= 1) {
    const float o = __shfl_xor(top_t, s);
    top_t = o > top_t || o != o ? o : top_t;
  }
  top = wave_maxf(top);
  const bool whole = a.teacher_log_normalizer == nullptr;
  if (whole && top_t == -kInf) any = false;  // no distribution
  double norm = whole ? 0.0 : static_cast<double>(a.teacher_log_normalizer[row]);
  if (whole && any) {
    double sum = 0.0;
    for (int j = lane; j < a.k; j += 64)
      if (held(ids[j]))
        sum += exp2_64((static_cast<double>(Elem<TT>::load1(t + j)) - top_t) * (c * kLog2e64));
    norm = static_cast<double>(top_t) * c + log(wave_add(sum));
  }
  double p_all = 0.0, h = 0.0, dot = 0.0, sum = 0.0;
  for (int j = lane; j < a.k; j += 64) {
    const int64_t id = ids[j];
    int column = -1;
    float pj = 0.0f, zj = 0.0f;
    if (any && held(id)) {
      const double lp = static_cast<double>(Elem<TT>::load1(t + j)) * c - norm;
      const double p = lp > 700.0 ? exp(lp) : exp2_64(lp * kLog2e64);
      p_all += p;
      if (p > 0.0 || p != p) h += p * lp;
      const int64_t at = id - a.vocab_start;
      if (at >= 0 && at < a.vocab_local) {
        zj = Elem<T>::load1(x + at);
        if (p > 0.0 || p != p) dot += p * (static_cast<double>(zj) * c);
        bool first = true;
        double p_id = p;
        if (again) {
          for (int i = 0; i < j && first; ++i) first = ids[i] != id;
          if (first)
            for (int i = j + 1; i < a.k; ++i)
              if (ids[i] == id) {
                const double l = static_cast<double>(Elem<TT>::load1(t + i)) * c - norm;
                p_id += l > 700.0 ? exp(l) : exp2_64(l * kLog2e64);
              }
        }
        if (first) {
          column = static_cast<int>(at);
          pj = static_cast<float>(p_id);
          sum += zj == top ? 1.0 : exp2_64((static_cast<double>(zj) - top) * (c * kLog2e64));
        }
      }
    }
    st.column[base + j] = column;
    st.p[base + j] = pj;
    st.z[base + j] = zj;
  }
  p_all = wave_add(p_all);
  h = wave_add(h);
  dot = wave_add(dot);
  sum = wave_add(sum);
  if (lane == 0) {
    Taught o;
    o.r = whole || !any ? 0.0 : fmax(1.0 - p_all, 0.0);
    o.p = p_all;
    o.h = h;
    o.dot = dot;
    // (Nothing above -inf there weighs nothing.)
    o.sum = top == -kInf && sum == sum ? 0.0 : sum;
    o.top = fmaxf(top, kNegHuge);
    o.any = any;
    st.rows[row] = o;
  }
}

// ---- the statistics outside the list ------------------------------------------------
// A row a workgroup, in stretches whose listed columns are bits in LDS.
constexpr int kBlock = 512;
constexpr int kWaves = kBlock / 64;
constexpr int kStretch = 65536;

template <typename T>
__global__ __launch_bounds__(kBlock) void distill_stats_kernel(nmce_distill_batch a, State st,
                                                               float cl,
                                                               double* __restrict__ stats) {
  using E = Elem<T>;
  constexpr int EPV = E::kPerVec;
  __shared__ uint32_t bits[kStretch / 32];
  __shared__ float wave_m[kWaves];
  __shared__ double wave_s[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  const int* column = st.column + row * a.k;
  float m = kNegHuge, s = 0.0f;
  for (int64_t c0 = 0; c0 < a.vocab_local; c0 += kStretch) {
    const int width = static_cast<int>(
        a.vocab_local - c0 < kStretch ? a.vocab_local - c0 : kStretch);
    for (int i = tid; i < kStretch / 32; i += kBlock) bits[i] = 0;
    __syncthreads();
    for (int j = tid; j < a.k; j += kBlock) {
      const int64_t at = column[j] - c0;
      if (at >= 0 && at < width) atomicOr(&bits[at >> 5], 1u << (at & 31));
    }
    __syncthreads();
    for (int i = tid * EPV; i < width; i += kBlock * EPV) {
      float f[EPV];
      if (i + EPV <= width) {
        u32x4 v;
        memcpy(&v, x + c0 + i, 16);
        E::unpack(v, f);
      } else {
#pragma unroll
        for (int e = 0; e < EPV; ++e) f[e] = i + e < width ? E::load1(x + c0 + i + e) : -kInf;
      }
      const uint32_t on = bits[i >> 5] >> (i & 31) & ((1u << EPV) - 1);
      if (on) {
#pragma unroll
        for (int e = 0; e < EPV; ++e) f[e] = on >> e & 1u ? -kInf : f[e];
      }
      float q = f[0];
#pragma unroll
      for (int e = 1; e < EPV; ++e) q = fmaxf(q, f[e]);
      const float nm = fmaxf(m, q);
      float y[EPV];
#pragma unroll
      for (int e = 0; e < EPV; ++e) y[e] = exp2_hw((f[e] - nm) * cl);
#pragma unroll
      for (int w = 1; w < EPV; w *= 2) {
#pragma unroll
        for (int e = 0; e + w < EPV; e += 2 * w) y[e] += y[e + w];
      }
      s = fmaf(s, exp2_hw((m - nm) * cl), y[0]);
      m = nm;
    }
    __syncthreads();
  }
  float wm = wave_max(m);
  if (lane == 0) wave_m[wave] = wm;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) wm = fmaxf(wm, wave_m[w]);
  double total = wave_add(static_cast<double>(s) * static_cast<double>(exp2_hw((m - wm) * cl)));
  if (lane == 0) wave_s[wave] = total;
  __syncthreads();
  if (tid == 0) {
    total = 0.0;
    for (int w = 0; w < kWaves; ++w) total += wave_s[w];
    const Taught t = st.rows[row];
    double* o = stats + row * kStat;
    o[0] = wm;
    o[1] = total;
    o[2] = t.top;
    o[3] = t.sum;
    o[4] = t.dot;
  }
}

// ---- the loss, and the backward's factors --------------------------------------------
// (m, s) and (o, u) together; sums of 0 have no say.
__device__ __forceinline__ void merge(double& m, double& s, double o, double u, double c) {
  if (o > m) {
    s = fma(s, exp2_64((m - o) * (c * kLog2e64)), u);
    m = o;
  } else {
    s = fma(u, exp2_64((o - m) * (c * kLog2e64)), s);
  }
}

// From the merged statistics of a row: outside the list (m, s), on it (top, sum), and
// sum p z / T. A student's row of only -inf, or with a +inf or NaN, has no distribution:
// NaN. Where it gives
// the rest nothing (nothing outside above -inf) the rest has no class and no term.
__device__ __forceinline__ double loss_and_slope(const Taught& t, double m, double s, double top,
                                                 double sum, double dot, double c, Slope* slope) {
  if (!t.any) {
    *slope = Slope{0.0f, 0.0f, 0.0f, -1.0f};  // (b < 0: no teacher, dz = 0)
    return 0.0;
  }
  double all_m = m, all = s;
  merge(all_m, all, top, sum, c);
  const bool rest = t.r > 0.0 && !(s == 0.0);
  const double p = t.p + (rest ? t.r : 0.0);
  const double log_all = log(all);
  double loss = t.h - dot + t.p * (all_m * c + log_all);
  if (rest) loss += t.r * (log(t.r) - ((m - all_m) * c + log(s) - log_all));
  const double b = p / all;
  slope->m = static_cast<float>(m);
  slope->a = static_cast<float>(b * exp2_64((m - all_m) * (c * kLog2e64)) -
                                (rest ? t.r / s : 0.0));
  slope->top = static_cast<float>(all_m);
  slope->b = static_cast<float>(b);
  if (all == 0.0 || all != all || all_m == static_cast<double>(kInf)) {
    slope->a = slope->b = __builtin_nanf("");
    loss = __builtin_nan("");
  }
  return loss;
}

__global__ __launch_bounds__(256) void distill_combine_kernel(State st, int64_t n, double c,
                                                              const double* __restrict__ stats,
                                                              int ranks,
                                                              float* __restrict__ loss) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (row >= n) return;
  double m = kNegHuge, s = 0.0, top = kNegHuge, sum = 0.0, dot = 0.0;
  for (int k = 0; k < ranks; ++k) {
    const double* o = stats + (k * n + row) * kStat;
    merge(m, s, o[0], o[1], c);
    merge(top, sum, o[2], o[3], c);
    dot += o[4];
  }
  Slope slope;
  loss[row] = static_cast<float>(loss_and_slope(st.rows[row], m, s, top, sum, dot, c, &slope));
  st.slopes[row] = slope;
}

// ---- the backward ------------------------------------------------------------------------
// A row a workgroup: the dense elements, then the list's over them.
template <typename T>
__global__ __launch_bounds__(kBlock) void distill_bwd_kernel(
    const T* x, T* g, int64_t n_rows, int64_t v, int64_t ld, int64_t ldg, int k, State st,
    float cl, const float* __restrict__ gout, int64_t gstride, float gdiv,
    const float* __restrict__ assumed, float* __restrict__ observed) {
  using E = Elem<T>;
  constexpr int EPV = E::kPerVec;
  if (assumed) {
    const float gv = gout[0];
    if (observed && blockIdx.x == 0 && threadIdx.x == 0) observed[0] = gv;
    if (gv == assumed[0]) return;
  }
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < n_rows; row += gridDim.x) {
    const Slope s = st.slopes[row];
    const float up = gout[row * gstride] / gdiv;
    const bool taught = !(s.b < 0.0f);
    const float scale = s.a * up;
    const T* xr = x + row * ld;
    T* gr = g + row * ldg;
    for (int64_t i = tid * EPV; i < v; i += kBlock * EPV) {
      float f[EPV], y[EPV];
      if (i + EPV <= v) {
        u32x4 w;
        memcpy(&w, xr + i, 16);
        E::unpack(w, f);
#pragma unroll
        for (int e = 0; e < EPV; ++e) y[e] = taught ? exp2_hw((f[e] - s.m) * cl) * scale : 0.0f;
        w = E::pack(y);
        memcpy(gr + i, &w, 16);
      } else {
        for (int e = 0; i + e < v; ++e)
          E::store1(gr + i + e,
                    taught ? exp2_hw((E::load1(xr + i + e) - s.m) * cl) * scale : 0.0f);
      }
    }
    // The dense stores have reached the memory before an element is stored over them.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (taught) {
      for (int j = tid; j < k; j += kBlock) {
        const int at = st.column[row * k + j];
        if (at >= 0)
          E::store1(gr + at, (exp2_hw((st.z[row * k + j] - s.top) * cl) * s.b -
                              st.p[row * k + j]) * up);
      }
    }
  }
}

int check_batch(const nmce_distill_batch* a) {
  if (!a) return NMCE_EINVAL_PTR;
  if ((a->dtype != NMCE_F32 && a->dtype != NMCE_BF16) ||
      (a->teacher_dtype != NMCE_F32 && a->teacher_dtype != NMCE_BF16))
    return NMCE_EINVAL_DTYPE;
  const int64_t most = (int64_t{1} << 31) - 1;
  if (a->n_rows < 0 || a->n_rows > (int64_t{1} << 22) || a->vocab_local < 1 ||
      a->vocab_local > most || a->vocab_start < 0 || a->vocab_total >= most ||
      a->vocab_total < a->vocab_local || a->vocab_start > a->vocab_total - a->vocab_local ||
      a->ld < a->vocab_local || a->k < 1 || a->k > kMaxK || a->teacher_ld < 0 || a->ids_ld < 0 ||
      !(a->temperature >= 1e-6 && a->temperature <= 1e6))
    return NMCE_EINVAL_SHAPE;
  if (a->n_rows == 0) return NMCE_OK;
  if (!a->logits || !a->teacher_logits || !a->teacher_ids) return NMCE_EINVAL_PTR;
  if (reinterpret_cast<uintptr_t>(a->logits) % (a->dtype == NMCE_F32 ? 4 : 2) ||
      reinterpret_cast<uintptr_t>(a->teacher_logits) % (a->teacher_dtype == NMCE_F32 ? 4 : 2))
    return NMCE_EINVAL_ALIGN;
  return NMCE_OK;
}

int check_state(const void* state, int64_t bytes, int64_t n, int k) {
  return !state || !aligned16(state) || bytes < nmce_distill_state_bytes(n, k)
             ? NMCE_EINVAL_WORKSPACE
             : NMCE_OK;
}

// exp((x - m) / T) = 2^((x - m) * this).
float log2e_over(double temperature) { return static_cast<float>(kLog2e64 / temperature); }

int launch_list(const nmce_distill_batch& a, const State& st, hipStream_t s) {
  int table = 64;
  while (table < 2 * a.k) table *= 2;
  const dim3 grid(static_cast<unsigned>((a.n_rows + kListWaves - 1) / kListWaves)),
      block(kListWaves * 64);
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, block, kListWaves * table * 4, s, a, table, st);
  };
  const bool f = a.dtype == NMCE_F32, tf = a.teacher_dtype == NMCE_F32;
  if (f)
    tf ? run(distill_list_kernel<float, float>) : run(distill_list_kernel<float, uint16_t>);
  else
    tf ? run(distill_list_kernel<uint16_t, float>) : run(distill_list_kernel<uint16_t, uint16_t>);
  return launch_status();
}

}  // namespace
}  // namespace nmce

using namespace nmce;

extern "C" {

int64_t nmce_distill_state_bytes(int64_t n_rows, int k) {
  if (n_rows < 0 || n_rows > (int64_t{1} << 22) || k < 1 || k > kMaxK) return -1;
  return align256(n_rows * static_cast<int64_t>(sizeof(Taught))) +
         align256(n_rows * static_cast<int64_t>(sizeof(Slope))) + 3 * align256(n_rows * k * 4);
}

int nmce_distill_stats(const nmce_distill_batch* a, void* state, int64_t state_bytes,
                       double* stats, void* stream) {
  if (const int rc = check_batch(a)) return rc;
  if (a->n_rows == 0) return NMCE_OK;
  if (!stats) return NMCE_EINVAL_PTR;
  if (const int rc = check_state(state, state_bytes, a->n_rows, a->k)) return rc;
  const State st = state_of(state, a->n_rows, a->k);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (const int rc = launch_list(*a, st, s)) return rc;
  const dim3 grid(static_cast<unsigned>(a->n_rows)), block(kBlock);
  const float cl = log2e_over(a->temperature);
  if (a->dtype == NMCE_F32)
    hipLaunchKernelGGL(distill_stats_kernel<float>, grid, block, 0, s, *a, st, cl, stats);
  else
    hipLaunchKernelGGL(distill_stats_kernel<uint16_t>, grid, block, 0, s, *a, st, cl, stats);
  return launch_status();
}

int nmce_distill_combine(void* state, int64_t state_bytes, int64_t n_rows, int k,
                         double temperature, const double* stats, int ranks, float* loss,
                         void* stream) {
  if (n_rows < 0 || n_rows > (int64_t{1} << 22) || k < 1 || k > kMaxK ||
      !(temperature >= 1e-6 && temperature <= 1e6))
    return NMCE_EINVAL_SHAPE;
  if (ranks < 1) return NMCE_EINVAL_TP;
  if (n_rows == 0) return NMCE_OK;
  if (!stats || !loss) return NMCE_EINVAL_PTR;
  if (const int rc = check_state(state, state_bytes, n_rows, k)) return rc;
  hipLaunchKernelGGL(distill_combine_kernel, dim3(static_cast<unsigned>((n_rows + 255) / 256)),
                     dim3(256), 0, static_cast<hipStream_t>(stream), state_of(state, n_rows, k),
                     n_rows, 1.0 / temperature, stats, ranks, loss);
  return launch_status();
}

int nmce_distill_bwd(const void* logits, void* grad, int dtype, int64_t n_rows,
                     int64_t vocab_local, int64_t ld, int64_t ld_grad, int k, double temperature,
                     void* state, int64_t state_bytes, const float* grad_output,
                     int64_t gout_stride, float gout_div, const float* assumed, float* observed,
                     void* stream) {
  if (dtype != NMCE_F32 && dtype != NMCE_BF16) return NMCE_EINVAL_DTYPE;
  if (n_rows < 0 || n_rows > (int64_t{1} << 22) || vocab_local < 1 || ld < vocab_local ||
      ld_grad < vocab_local || k < 1 || k > kMaxK || gout_stride < 0 || !(gout_div > 0.0f) ||
      !(temperature >= 1e-6 && temperature <= 1e6) || (grad == logits && ld_grad != ld))
    return NMCE_EINVAL_SHAPE;
  if (n_rows == 0) return NMCE_OK;
  if (!logits || !grad || !grad_output) return NMCE_EINVAL_PTR;
  const uintptr_t es = dtype == NMCE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % es || reinterpret_cast<uintptr_t>(grad) % es)
    return NMCE_EINVAL_ALIGN;
  if (const int rc = check_state(state, state_bytes, n_rows, k)) return rc;
  const State st = state_of(state, n_rows, k);
  const float cl = log2e_over(temperature);
  const float gdiv = gout_div * static_cast<float>(temperature);
  // After a one-pass forward the upstream value is usually the assumed one: a small
  // grid that walks the rows then ends at once.
  const int64_t most = assumed ? 2 * device_cus() : n_rows;
  const dim3 grid(static_cast<unsigned>(n_rows < most ? n_rows : most)), block(kBlock);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == NMCE_F32)
    hipLaunchKernelGGL(distill_bwd_kernel<float>, grid, block, 0, s,
                       static_cast<const float*>(logits), static_cast<float*>(grad), n_rows,
                       vocab_local, ld, ld_grad, k, st, cl, grad_output, gout_stride, gdiv,
                       assumed, observed);
  else
    hipLaunchKernelGGL(distill_bwd_kernel<uint16_t>, grid, block, 0, s,
                       static_cast<const uint16_t*>(logits), static_cast<uint16_t*>(grad), n_rows,
                       vocab_local, ld, ld_grad, k, st, cl, grad_output, gout_stride, gdiv,
                       assumed, observed);
  return launch_status();
}

}  // extern "C"
