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
constexpr int kBufNonTemporal = 2;
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
  float* sums;  // outside the list, as the slope's m has it (of the one-pass forward)
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
  s.sums = reinterpret_cast<float*>(take(n * 4));
  s.column = reinterpret_cast<int*>(take(n * k * 4));
  s.p = reinterpret_cast<float*>(take(n * k * 4));
  s.z = reinterpret_cast<float*>(take(n * k * 4));
  return s;
}

// 16 bytes at any element's alignment, streamed.
typedef u32x4 anywhere __attribute__((aligned(2)));
__device__ __forceinline__ u32x4 load16(const void* p) {
  return __builtin_nontemporal_load(static_cast<const anywhere*>(p));
}
__device__ __forceinline__ void store16(void* p, const u32x4& v) {
  __builtin_nontemporal_store(v, static_cast<anywhere*>(p));
}

// Fold K values into (m, sum of 2^((x - m) cl)).
template <int K>
__device__ __forceinline__ void fold(float& m, float& s, float* f, float cl) {
  float q = f[0];
#pragma unroll
  for (int k = 1; k < K; ++k) q = fmaxf(q, f[k]);
  const float nm = fmaxf(m, q);
#pragma unroll
  for (int k = 0; k < K; ++k) f[k] = exp2_hw((f[k] - nm) * cl);
#pragma unroll
  for (int w = 1; w < K; w *= 2) {
#pragma unroll
    for (int k = 0; k + w < K; k += 2 * w) f[k] += f[k + w];
  }
  s = fmaf(s, exp2_hw((m - nm) * cl), f[0]);
  m = nm;
}

__device__ __forceinline__ double wave_add(double v) {
  for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s);
  return v;
}
// exp(lp) of a log-probability (far above 0, as from a normaliser that is none, infinite).
__device__ __forceinline__ double probability(double lp) {
  return lp > 700.0 ? static_cast<double>(kInf) : exp2_64(lp * kLog2e64);
}

// ---- the list's side ------------------------------------------------------------
constexpr int kListWaves = 4;

// kWhole: no normaliser, the teacher's distribution is over the list. The student's sum is
// in fp32 terms, as the one outside the list is. Latency bounds it (ids, then the logits that
// they name, then fp64 exponentials; waits 0.64 to 0.80 of the waves' time): 256 rows of 20
// 6 us, 8192 of 64 21. A list that names an id twice is compared with itself, K^2 / 64 reads of
// LDS a lane: a step of 4096 rows 839 -> 1625 us where each of K 1024 does, 604 -> 624 of 128.
// `assumed` (of a one-pass forward, else NULL) takes the upstream value to assume: the row
// kernels read it there, since another stream's backward may change the hint under them.
template <typename T, typename TT, bool kWhole>
__global__ __launch_bounds__(kListWaves * 64) void distill_list_kernel(
    nmce_distill_batch a, int table, float cl, State st, const float* __restrict__ expect,
    float* __restrict__ assumed) {
  extern __shared__ int tables[];  // `table` slots a wave: ids noted, 0 for none
  if (assumed && blockIdx.x == 0 && threadIdx.x == 0) assumed[0] = usable_hint(expect[0]);
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
  auto column_of = [&](int64_t id) {
    const int64_t at = id - a.vocab_start;
    return held(id) && at >= 0 && at < a.vocab_local ? static_cast<int>(at) : -1;
  };

  for (int i = lane; i < table; i += 64) seen[i] = 0;
  __builtin_amdgcn_wave_barrier();
  float top_t = -kInf, top = -kInf;
  bool any = false, again = false;
  for (int j = lane; j < a.k; j += 64) {
    const int64_t id = ids[j];
    const int at = column_of(id);
    const float zj = at >= 0 ? Elem<T>::load1(x + at) : -kInf;
    st.z[base + j] = zj;
    top = fmaxf(top, zj);
    if (!held(id)) continue;
    any = true;
    const float tj = Elem<TT>::load1(t + j);
    top_t = tj > top_t || tj != tj ? tj : top_t;
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
  top = wave_max(fmaxf(top, kNegHuge));
  double norm = 0.0;
  if constexpr (kWhole) {
    for (int s = 32; s > 0; s >>= 1) {
      const float o = __shfl_xor(top_t, s);
      top_t = o > top_t || o != o ? o : top_t;
    }
    if (top_t == -kInf) any = false;  // no distribution
    if (any) {
      double sum = 0.0;
      for (int j = lane; j < a.k; j += 64)
        if (held(ids[j]))
          sum += exp2_64((static_cast<double>(Elem<TT>::load1(t + j)) - top_t) * (c * kLog2e64));
      norm = static_cast<double>(top_t) * c + log(wave_add(sum));
    }
  } else {
    norm = static_cast<double>(a.teacher_log_normalizer[row]);
    if (norm == -static_cast<double>(kInf)) any = false;  // (a teacher's row of only -inf)
  }
  // (The table is done with; of a list that names an id twice its logits and ids come there.)
  float* held_t = reinterpret_cast<float*>(seen);
  int* held_id = seen + a.k;
  double p_all = 0.0, h = 0.0, dot = 0.0, sum = 0.0;
  for (int j = lane; j < a.k; j += 64) {
    const int64_t id = ids[j];
    const int at = any ? column_of(id) : -1;
    double p = 0.0;
    float tj = 0.0f;
    if (any && held(id)) {
      tj = Elem<TT>::load1(t + j);
      const double lp = static_cast<double>(tj) * c - norm;
      p = probability(lp);
      p_all += p;
      const bool some = p > 0.0 || p != p;
      if (some) h += p * lp;
      if (at >= 0) {
        const float zj = st.z[base + j];  // (the lane's own store)
        if (some) dot += p * (static_cast<double>(zj) * c);
        sum += exp2_hw((zj - top) * cl);
      }
    }
    st.column[base + j] = at;
    st.p[base + j] = static_cast<float>(p);
    if (again) {
      held_t[j] = tj;
      held_id[j] = any && held(id) ? static_cast<int>(id) : -1;
    }
  }
  if (again) {
    // An id's first place takes all of its p, in their order, for p log p too (of every id of
    // the list, other shards' as well: all ranks have the same); the others are none.
    __builtin_amdgcn_wave_barrier();
    h = 0.0;
    for (int j = lane; j < a.k; j += 64) {
      const int id = held_id[j];
      if (id < 0) continue;
      const int at = column_of(id);
      int before = 0, others = 0;
#pragma unroll 8
      for (int i = 0; i < a.k; ++i) {
        const bool same = held_id[i] == id;
        before += same && i < j;
        others += same && i > j;
      }
      if (before) {
        st.column[base + j] = -1;
        if (at >= 0) sum -= exp2_hw((Elem<T>::load1(x + at) - top) * cl);  // counted at the first
        continue;
      }
      double lp = static_cast<double>(held_t[j]) * c - norm;
      double p = probability(lp);
      if (others) {
        for (int i = j + 1; i < a.k; ++i)
          if (held_id[i] == id)
            p += probability(static_cast<double>(held_t[i]) * c - norm);
        lp = log(p);
        st.p[base + j] = static_cast<float>(p);
      }
      if (p > 0.0 || p != p) h += p * lp;
    }
  }
  p_all = wave_add(p_all);
  h = wave_add(h);
  dot = wave_add(dot);
  sum = wave_add(sum);
  if (lane == 0) {
    Taught o;
    o.r = kWhole || !any ? 0.0 : fmax(1.0 - p_all, 0.0);
    o.p = p_all;
    o.h = h;
    o.dot = dot;
    o.sum = sum;
    o.top = top;
    o.any = any;
    st.rows[row] = o;
  }
}

// ---- the statistics outside the list ------------------------------------------------
// A row a workgroup, in stretches whose listed columns are bits in LDS. Bounded by the read:
// 4096 x 151936 bf16 184 us (6.7 TB/s, VALU busy 0.87).
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
    auto take = [&](int i, const u32x4& v) {
      float f[EPV];
      E::unpack(v, f);
      const uint32_t on = bits[i >> 5] >> (i & 31) & ((1u << EPV) - 1);
      if (on) {
#pragma unroll
        for (int e = 0; e < EPV; ++e) f[e] = on >> e & 1u ? -kInf : f[e];
      }
      fold<EPV>(m, s, f, cl);
    };
    // Two vectors on their way at a time.
    int i = tid * EPV;
    for (; i + kBlock * EPV + EPV <= width; i += 2 * kBlock * EPV) {
      const u32x4 v0 = load16(x + c0 + i), v1 = load16(x + c0 + i + kBlock * EPV);
      take(i, v0);
      take(i + kBlock * EPV, v1);
    }
    for (; i < width; i += kBlock * EPV) {
      if (i + EPV <= width) {
        take(i, load16(x + c0 + i));
      } else {
        for (int j = i; j < width; ++j) {
          float f[1] = {bits[j >> 5] >> (j & 31) & 1u ? -kInf : E::load1(x + c0 + j)};
          fold<1>(m, s, f, cl);
        }
      }
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
// NaN. Where it gives the rest nothing (nothing outside above -inf) the rest has no class
// and no term.
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

// The losses of the one-pass forward, and their mean where one workgroup has all rows; of
// more, distill_mean_kernel's (8192 rows: 25 us in one workgroup, 5 and 4 in the two).
// Sums in a fixed order, in 64 bits.
constexpr int kLossBlock = 1024;
constexpr int kLossRows = 64;  // of a workgroup, where there are several
__device__ __forceinline__ void store_mean(double sum, int64_t n, float* __restrict__ mean) {
  __shared__ double part[kLossBlock / 64];
  sum = wave_add(sum);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < static_cast<int>(blockDim.x >> 6); ++w) sum += part[w];
  mean[0] = static_cast<float>(sum / static_cast<double>(n));
}
__global__ __launch_bounds__(kLossBlock) void distill_loss_kernel(State st, int64_t n, double c,
                                                                  float* __restrict__ loss,
                                                                  float* __restrict__ mean) {
  double sum = 0.0;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (row < n) {
    const Taught t = st.rows[row];
    Slope slope;
    const double one = loss_and_slope(t, t.any ? st.slopes[row].m : 0.0, st.sums[row], t.top,
                                      t.sum, t.dot, c, &slope);
    loss[row] = static_cast<float>(one);
    sum = static_cast<float>(one);
  }
  if (mean) store_mean(sum, n, mean);
}
__global__ __launch_bounds__(kLossBlock) void distill_mean_kernel(const float* __restrict__ loss,
                                                                  int64_t n,
                                                                  float* __restrict__ mean) {
  constexpr int kAhead = 8;
  double sum = 0.0;
  for (int64_t row = threadIdx.x; row < n; row += kAhead * kLossBlock) {
    float one[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t at = row + i * kLossBlock;
      one[i] = loss[at < n ? at : n - 1];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) sum += row + i * kLossBlock < n ? one[i] : 0.0f;
  }
  store_mean(sum, n, mean);
}

constexpr int kBwdAhead = 4;  // vectors of a thread on their way

// ---- the backward ------------------------------------------------------------------------
// A row a workgroup: the dense elements, then the list's over them. For rows off the 16-byte
// grid, and after a one-pass forward, where it mostly ends at once (3 to 5 us).
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
    auto slope_at = [&](float f) { return taught ? exp2_hw((f - s.m) * cl) * scale : 0.0f; };
    auto put = [&](int64_t i, const u32x4& w) {
      float f[EPV];
      E::unpack(w, f);
#pragma unroll
      for (int e = 0; e < EPV; ++e) f[e] = slope_at(f[e]);
      store16(gr + i, E::pack(f));
    };
    constexpr int kStep = kBlock * EPV;
    int64_t i = tid * EPV;
    for (; i + (kBwdAhead - 1) * kStep + EPV <= v; i += kBwdAhead * kStep) {
      u32x4 w[kBwdAhead];
#pragma unroll
      for (int u = 0; u < kBwdAhead; ++u) w[u] = load16(xr + i + u * kStep);
#pragma unroll
      for (int u = 0; u < kBwdAhead; ++u) put(i + u * kStep, w[u]);
    }
    for (; i < v; i += kStep) {
      if (i + EPV <= v) {
        put(i, load16(xr + i));
      } else {
        for (int64_t j = i; j < v; ++j) E::store1(gr + j, slope_at(E::load1(xr + j)));
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

// ---- forward and backward in one read -----------------------------------------------------
// Whole-vocabulary rows (one rank) held by a workgroup of 1024 threads: in registers (up to 8
// vectors a thread; two workgroups a compute unit), or 9 of up to 16 in LDS. Bounded by HBM
// with a whole row between its read and its write: 2047 x 50257 bf16 87 us (4.8 TB/s), 8192 x
// 128256 790 (5.3; a streaming copy 6.5). A step of these takes 101 and 815 us, by two passes 152 and
// 994, in place 101 and 841; one whose upstream value is not the assumed one 192 and 1571.
// The listed elements are set to -inf where they are held, so that the fold sees what is
// outside; each wave does that for its own elements, one listed id after another, and writes
// their gradients over the row's, by the lanes that stored it. The gradient is that of the mean
// for the upstream value assumed[0] (the list kernel's); loss and slopes as from
// distill_combine_kernel, the slopes in fp32. Vectors, edges (kRagged: rows of any width and
// alignment, the gradient's as the logits') and buffer resources as in the cross entropy's
// one-pass kernels. g may be x.
constexpr int kRowBlock = 1024;
constexpr int kRowWaves = kRowBlock / 64;
constexpr int kWideLo = 7, kWideHi = 9;
constexpr int kWideLdsBytes = kWideHi * kRowBlock * 16;
static_assert(kWideLdsBytes + 2 * kRowWaves * 8 <= 160 * 1024, "");
typedef __attribute__((address_space(3))) void lds_void_t;

// Where a row's column is held: vector `slot` of thread `owner`, element e; slot -1: the
// thread's edge element.
struct Place {
  int owner, slot, e;
};
template <int EPV>
__device__ __forceinline__ Place place_of(int column, int head, int nvec) {
  const int rel = column - head;
  if (rel < 0) return {column, -1, 0};
  if (rel >= nvec * EPV) return {EPV + rel - nvec * EPV, -1, 0};
  const int vec = rel / EPV;
  return {vec % kRowBlock, vec / kRowBlock, rel % EPV};
}

// Element e (the same for all lanes) of v to -inf where `on`.
template <typename T>
__device__ __forceinline__ void mask_out(u32x4& v, int e, bool on) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    if constexpr (sizeof(T) == 4) {
      if (e == d) v[d] = on ? 0xff800000u : v[d];
    } else {
      if (e == 2 * d) v[d] = on ? (v[d] & 0xffff0000u) | 0xff80u : v[d];
      if (e == 2 * d + 1) v[d] = on ? (v[d] & 0xffffu) | 0xff800000u : v[d];
    }
  }
}

// (m, s) of the wave, in every lane.
__device__ __forceinline__ void wave_merge(float& m, float& s, float cl) {
  const float wm = wave_max(m);
  s = wave_sum(s * exp2_hw((m - wm) * cl));
  m = wm;
}

// loss_and_slope's slope in fp32, by every wave for itself.
__device__ __forceinline__ Slope slope_of(const Taught& t, float m, float s, float cl) {
  const float top = t.top, sum = static_cast<float>(t.sum), r = static_cast<float>(t.r);
  const float all_m = fmaxf(m, top);
  const float out = exp2_hw((m - all_m) * cl);
  const float all = fmaf(s, out, sum * exp2_hw((top - all_m) * cl));
  const bool rest = r > 0.0f && !(s == 0.0f);
  const float b = (static_cast<float>(t.p) + (rest ? r : 0.0f)) / all;
  Slope o{m, b * out - (rest ? r / s : 0.0f), all_m, b};
  if (all == 0.0f || all != all || all_m == kInf) o.a = o.b = __builtin_nanf("");
  if (!t.any) o = Slope{0.0f, 0.0f, 0.0f, -1.0f};
  return o;
}

// The listed ids of a row that a wave's elements hold, 64 of the list at a time.
template <typename T>
struct Listed {
  static constexpr int EPV = Elem<T>::kPerVec;
  const int* column;
  const float* p;
  const float* z;
  int k, lane, wave;
  int first;  // the list's first 64, asked for early
  float first_p, first_z;

  __device__ __forceinline__ void ask(const State& st, int64_t row, int k_, int lane_, int wave_) {
    column = st.column + row * k_;
    p = st.p + row * k_;
    z = st.z + row * k_;
    k = k_;
    lane = lane_;
    wave = wave_;
    first = lane < k ? column[lane] : -1;
    first_p = lane < k ? p[lane] : 0.0f;
    first_z = lane < k ? z[lane] : 0.0f;
  }
  // use(place, column, value of `each` in the lane that holds the id) for every id of the
  // wave's; the arguments are the same in all lanes.
  template <typename Each, typename Use>
  __device__ __forceinline__ void visit(int head, int nvec, Each&& each, Use&& use) const {
    for (int base = 0; base < k; base += 64) {
      const int j = base + lane;
      const int c = base == 0 ? first : j < k ? column[j] : -1;
      const bool mine = c >= 0 && place_of<EPV>(c, head, nvec).owner >> 6 == wave;
      uint64_t who = __ballot(mine);
      if (who == 0) continue;
      float value = 0.0f;
      if (mine) value = base == 0 ? each(first_p, first_z) : each(p[j], z[j]);
      for (; who; who &= who - 1) {
        const int src = __builtin_ctzll(who);
        const int at = __builtin_amdgcn_readlane(c, src);
        use(place_of<EPV>(at, head, nvec), at,
            __int_as_float(__builtin_amdgcn_readlane(__float_as_int(value), src)));
      }
    }
  }
};

template <typename T, int kVec, bool kRagged>
__global__ __launch_bounds__(kRowBlock, 8) void distill_row_kernel(
    const T* x, T* g, int64_t n_rows, int64_t V, int64_t ld, int64_t ldg, int k, State st,
    float cl, const float* __restrict__ assumed, float gdiv) {
  using E = Elem<T>;
  constexpr int EPV = E::kPerVec;
  __shared__ float sm_m[2][kRowWaves];
  __shared__ float sm_s[2][kRowWaves];
  const float up = assumed[0] / gdiv;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int head = 0;
  int nvec = static_cast<int>(V / EPV);
  const int row_end = static_cast<int>(V * sizeof(T));
  auto rsrc = [&](const T* base, int64_t r, int64_t stride) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base + r * stride), 0, row_end,
                                             0x00020000);
  };
  auto rsrc_k = [&](const T* base, int64_t r, int64_t stride, int i) {
    const int rest = (nvec - i * kRowBlock) * 16;
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<T*>(base + r * stride + head + i * kRowBlock * EPV), 0, rest > 0 ? rest : 0,
        0x00020000);
  };
  const uint32_t voff = static_cast<uint32_t>(tid) * 16u;
  u32x4 cur[kVec];
  int parity = 0;
  for (int64_t row = blockIdx.x; row < n_rows; row += gridDim.x, parity ^= 1) {
    if constexpr (kRagged) {
      head = static_cast<int>(head_elems(x + row * ld, V));
      nvec = (static_cast<int>(V) - head) / EPV;
    }
    Listed<T> listed;
    listed.ask(st, row, k, lane, wave);
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      cur[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc_k(x, row, ld, i), voff, 0,
                                                     kBufNonTemporal);
    const int ec =
        kRagged ? edge_column<EPV>(tid, head, nvec, static_cast<int>(V)) : -1;
    float edge = 0.0f;
    if constexpr (kRagged)
      edge = E::buf_load1(rsrc(x, row, ld), ec >= 0 ? static_cast<uint32_t>(ec) * sizeof(T)
                                                    : static_cast<uint32_t>(row_end));
    const Taught t = st.rows[row];
    listed.visit(head, nvec, [](float, float) { return 0.0f; },
                 [&](const Place& at, int, float) {
                   const bool on = lane == (at.owner & 63);
#pragma unroll
                   for (int i = 0; i < kVec; ++i)
                     if (at.slot == i) mask_out<T>(cur[i], at.e, on);
                   if (kRagged && at.slot < 0) edge = on ? -kInf : edge;
                 });
    float m = kNegHuge, s = 0.0f;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      if (tid + i * kRowBlock < nvec) {
        u32x4 w = cur[i];
        asm volatile("" : "+v"(w));
        float f[EPV];
        E::unpack(w, f);
        fold<EPV>(m, s, f, cl);
      }
    }
    if (kRagged && ec >= 0) {
      float f[1] = {edge};
      fold<1>(m, s, f, cl);
    }
    wave_merge(m, s, cl);
    if (lane == 0) {
      sm_m[parity][wave] = m;
      sm_s[parity][wave] = s;
    }
    __syncthreads();
    m = lane < kRowWaves ? sm_m[parity][lane] : kNegHuge;
    s = lane < kRowWaves ? sm_s[parity][lane] : 0.0f;
    wave_merge(m, s, cl);
    const Slope slope = slope_of(t, m, s, cl);
    const float scale = slope.a * up;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      u32x4 out = {0u, 0u, 0u, 0u};
      if (t.any && tid + i * kRowBlock < nvec) {
        u32x4 w = cur[i];
        asm volatile("" : "+v"(w));  // unpack again from the packed row
        float f[EPV];
        E::unpack(w, f);
#pragma unroll
        for (int e = 0; e < EPV; ++e) f[e] = exp2_hw((f[e] - slope.m) * cl) * scale;
        out = E::pack(f);
      }
      buffer_store_b128<kBufNonTemporal>(out, rsrc_k(g, row, ldg, i), voff);
    }
    const auto rg = rsrc(g, row, ldg);
    if constexpr (kRagged)
      E::buf_store1(t.any ? exp2_hw((edge - slope.m) * cl) * scale : 0.0f, rg,
                    ec >= 0 ? static_cast<uint32_t>(ec) * sizeof(T)
                            : static_cast<uint32_t>(row_end));
    listed.visit(head, nvec,
                 [&](float p, float z) {
                   return (exp2_hw((z - slope.top) * cl) * slope.b - p) * up;
                 },
                 [&](const Place& at, int column, float value) {
                   E::buf_store1(value, rg, lane == (at.owner & 63)
                                                ? static_cast<uint32_t>(column) * sizeof(T)
                                                : static_cast<uint32_t>(row_end));
                 });
    if (tid == kRowBlock - 64) {
      st.slopes[row] = slope;
      st.sums[row] = s;
    }
  }
}

// Rows wider than 8 vectors a thread: vectors 0 .. 6 in registers and 7 .. 15 in LDS, the
// next row's on their way while this one's gradient is written. Every wave fills, reads and
// masks its own part of LDS, so only the statistics need a barrier.
template <typename T, bool kRagged>
__global__ __launch_bounds__(kRowBlock) void distill_wide_row_kernel(
    const T* x, T* g, int64_t n_rows, int64_t V, int64_t ld, int64_t ldg, int k, State st,
    float cl, const float* __restrict__ assumed, float gdiv) {
  using E = Elem<T>;
  constexpr int EPV = E::kPerVec;
  extern __shared__ __align__(16) char lds_dyn[];
  u32x4* hi = reinterpret_cast<u32x4*>(lds_dyn);  // vector kWideLo + i of thread t: hi[i * kRowBlock + t]
  __shared__ float sm_m[2][kRowWaves];
  __shared__ float sm_s[2][kRowWaves];
  const float up = assumed[0] / gdiv;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  struct Geom {
    int head, nvec, cnt;
  };
  auto geom = [&](int64_t r) {
    Geom q;
    q.head = kRagged ? static_cast<int>(head_elems(x + r * ld, V)) : 0;
    q.nvec = (static_cast<int>(V) - q.head) / EPV;
    q.cnt = q.nvec > tid ? (q.nvec - tid + kRowBlock - 1) / kRowBlock : 0;
    return q;
  };
  auto row_rsrc = [&](const T* base, const Geom& q) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base + q.head), 0, q.nvec * 16,
                                             0x00020000);
  };
  const uint32_t voff = static_cast<uint32_t>(tid) * 16u;
  u32x4 cur[kWideLo], nxt[kWideLo];
  auto load_lo = [&](int64_t r, const Geom& q, u32x4 (&v)[kWideLo]) {
    const auto rs = row_rsrc(x + r * ld, q);
#pragma unroll
    for (int i = 0; i < kWideLo; ++i)
      if (i < q.cnt)
        v[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, voff, i * kRowBlock * 16,
                                                     kBufNonTemporal);
  };
  auto load_hi = [&](int64_t r, const Geom& q) {
    const uint64_t addr = reinterpret_cast<uint64_t>(x + r * ld + q.head);
    i32x4_t rs;
    rs[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(addr & 0xffffffffu));
    rs[1] = __builtin_amdgcn_readfirstlane(static_cast<int>(addr >> 32));
    rs[2] = q.nvec * 16;
    rs[3] = 0x00020000;
#pragma unroll
    for (int i = 0; i < kWideHi; ++i)
      if (kWideLo + i < q.cnt)
        raw_buffer_load_lds(rs, (lds_void_t*)(hi + i * kRowBlock + wave * 64), 16,
                            static_cast<int>(voff) + (kWideLo + i) * kRowBlock * 16, 0, 0, 0);
  };
  int64_t row = blockIdx.x;
  Geom q{};
  Listed<T> listed{};
  if (row < n_rows) {
    q = geom(row);
    listed.ask(st, row, k, lane, wave);
    load_lo(row, q, cur);
    load_hi(row, q);
  }
  int parity = 0;
  for (; row < n_rows; row += gridDim.x, parity ^= 1) {
    const Taught t = st.rows[row];
    const int ec =
        kRagged ? edge_column<EPV>(tid, q.head, q.nvec, static_cast<int>(V)) : -1;
    float edge = 0.0f;
    if (kRagged && ec >= 0) edge = E::load1(x + row * ld + ec);
    // The wave's part of the row has landed.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    listed.visit(q.head, q.nvec, [](float, float) { return 0.0f; },
                 [&](const Place& at, int, float) {
                   const bool on = lane == (at.owner & 63);
#pragma unroll
                   for (int i = 0; i < kWideLo; ++i)
                     if (at.slot == i) mask_out<T>(cur[i], at.e, on);
                   if (at.slot >= kWideLo && on)
                     E::store1(reinterpret_cast<T*>(hi + (at.slot - kWideLo) * kRowBlock + tid) +
                                   at.e, -kInf);
                   if (kRagged && at.slot < 0) edge = on ? -kInf : edge;
                 });
    float m = kNegHuge, s = 0.0f;
#pragma unroll
    for (int i = 0; i < kWideLo + kWideHi; ++i) {
      if (i < q.cnt) {
        u32x4 w = i < kWideLo ? cur[i < kWideLo ? i : 0] : hi[(i - kWideLo) * kRowBlock + tid];
        asm volatile("" : "+v"(w));
        float f[EPV];
        E::unpack(w, f);
        fold<EPV>(m, s, f, cl);
      }
    }
    if (kRagged && ec >= 0) {
      float f[1] = {edge};
      fold<1>(m, s, f, cl);
    }
    const int64_t next = row + gridDim.x;
    Geom qn = q;
    Listed<T> then = listed;
    if (next < n_rows) {
      if constexpr (kRagged) qn = geom(next);
      then.ask(st, next, k, lane, wave);
      load_lo(next, qn, nxt);
    }
    wave_merge(m, s, cl);
    if (lane == 0) {
      sm_m[parity][wave] = m;
      sm_s[parity][wave] = s;
    }
    __syncthreads();
    m = lane < kRowWaves ? sm_m[parity][lane] : kNegHuge;
    s = lane < kRowWaves ? sm_s[parity][lane] : 0.0f;
    wave_merge(m, s, cl);
    const Slope slope = slope_of(t, m, s, cl);
    const float scale = slope.a * up;
    const auto grs = row_rsrc(g + row * ldg, q);
    auto write_grad = [&](u32x4 v, int i) {
      float f[EPV];
      E::unpack(v, f);
#pragma unroll
      for (int e = 0; e < EPV; ++e)
        f[e] = t.any ? exp2_hw((f[e] - slope.m) * cl) * scale : 0.0f;
      buffer_store_b128<kBufNonTemporal>(E::pack(f), grs, voff + i * kRowBlock * 16);
    };
#pragma unroll
    for (int i = 0; i < kWideHi; ++i)
      if (kWideLo + i < q.cnt) write_grad(hi[i * kRowBlock + tid], kWideLo + i);
    // The wave has read its part of LDS: the next row's may come.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (next < n_rows) load_hi(next, qn);
#pragma unroll
    for (int i = 0; i < kWideLo; ++i)
      if (i < q.cnt) write_grad(cur[i], i);
    T* gr = g + row * ldg;
    if (kRagged && ec >= 0)
      E::store1(gr + ec, t.any ? exp2_hw((edge - slope.m) * cl) * scale : 0.0f);
    listed.visit(q.head, q.nvec,
                 [&](float p, float z) {
                   return (exp2_hw((z - slope.top) * cl) * slope.b - p) * up;
                 },
                 [&](const Place& at, int column, float value) {
                   if (lane == (at.owner & 63)) E::store1(gr + column, value);
                 });
    if (tid == kRowBlock - 64) {
      st.slopes[row] = slope;
      st.sums[row] = s;
    }
    q = qn;
    listed = then;
#pragma unroll
    for (int i = 0; i < kWideLo; ++i) cur[i] = nxt[i];
  }
}

// The dense elements of rows on the 16-byte grid, a few vectors a workgroup wherever they
// are (4096 x 151936 bf16 492 -> 385 us, 6.4 TB/s: many small workgroups keep more of the
// memory busy), and the list's over them in a launch of their own (128 a row: 14 us, stores of
// 2 bytes anywhere).
constexpr int kFlatBlock = 128, kFlatAhead = 2;
template <typename T>
__global__ __launch_bounds__(kFlatBlock) void distill_flat_kernel(
    const T* x, T* g, uint32_t n_vec, uint32_t per_row, int64_t ld, int64_t ldg,
    const Slope* __restrict__ slopes, float cl, const float* __restrict__ gout, int64_t gstride,
    float gdiv) {
  using E = Elem<T>;
  constexpr int EPV = E::kPerVec;
  const uint32_t base = blockIdx.x * static_cast<uint32_t>(kFlatBlock * kFlatAhead) + threadIdx.x;
  u32x4 v[kFlatAhead];
  uint32_t rows[kFlatAhead], cols[kFlatAhead];
#pragma unroll
  for (int u = 0; u < kFlatAhead; ++u) {
    const uint32_t f = base + u * kFlatBlock;
    rows[u] = f / per_row;
    cols[u] = (f - rows[u] * per_row) * EPV;
    if (f < n_vec)
      v[u] = load_stream(reinterpret_cast<const u32x4*>(x + rows[u] * ld + cols[u]));
  }
#pragma unroll
  for (int u = 0; u < kFlatAhead; ++u) {
    if (base + u * kFlatBlock >= n_vec) continue;
    const Slope s = slopes[rows[u]];
    const float scale = s.a * (gout[rows[u] * gstride] / gdiv);
    float f[EPV];
    E::unpack(v[u], f);
#pragma unroll
    for (int e = 0; e < EPV; ++e)
      f[e] = s.b < 0.0f ? 0.0f : exp2_hw((f[e] - s.m) * cl) * scale;
    store_stream(reinterpret_cast<u32x4*>(g + rows[u] * ldg + cols[u]), E::pack(f));
  }
}

template <typename T>
__global__ __launch_bounds__(256) void distill_listed_kernel(
    T* g, int64_t count, int64_t ldg, int k, State st, float cl, const float* __restrict__ gout,
    int64_t gstride, float gdiv) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= count) return;
  const int at = st.column[i];
  if (at < 0) return;
  const int64_t row = i / k;
  const Slope s = st.slopes[row];
  const float up = gout[row * gstride] / gdiv;
  Elem<T>::store1(g + row * ldg + at, (exp2_hw((st.z[i] - s.top) * cl) * s.b - st.p[i]) * up);
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

int launch_mean(const float* loss, int64_t n, float* mean, hipStream_t s) {
  hipLaunchKernelGGL(distill_mean_kernel, dim3(1), dim3(kLossBlock), 0, s, loss, n, mean);
  return launch_status();
}

int launch_list(const nmce_distill_batch& a, const State& st, const float* expect, float* assumed,
                hipStream_t s) {
  int table = 64;
  while (table < 2 * a.k) table *= 2;
  const dim3 grid(static_cast<unsigned>((a.n_rows + kListWaves - 1) / kListWaves)),
      block(kListWaves * 64);
  auto run = [&](auto element, auto teacher) {
    using T = decltype(element);
    using TT = decltype(teacher);
    const float cl = log2e_over(a.temperature);
    const int lds = kListWaves * table * 4;
    if (a.teacher_log_normalizer)
      hipLaunchKernelGGL((distill_list_kernel<T, TT, false>), grid, block, lds, s, a, table, cl, st,
                         expect, assumed);
    else
      hipLaunchKernelGGL((distill_list_kernel<T, TT, true>), grid, block, lds, s, a, table, cl, st,
                         expect, assumed);
  };
  const bool f = a.dtype == NMCE_F32, tf = a.teacher_dtype == NMCE_F32;
  if (f)
    tf ? run(float{}, float{}) : run(float{}, uint16_t{});
  else
    tf ? run(uint16_t{}, float{}) : run(uint16_t{}, uint16_t{});
  return launch_status();
}

template <typename T, bool kRagged>
int launch_rows(const nmce_distill_batch& a, void* grad, int64_t ldg, const State& st,
                const float* assumed, float gdiv, hipStream_t s) {
  const T* x = static_cast<const T*>(a.logits);
  T* g = static_cast<T*>(grad);
  const float cl = log2e_over(a.temperature);
  const int64_t per_thread = (a.vocab_local / Elem<T>::kPerVec + kRowBlock - 1) / kRowBlock;
  const dim3 block(kRowBlock);
  auto run = [&](auto kernel, int per_cu, int lds) {
    // (Where a workgroup takes one row: a launch's threads fit 32 bits.)
    const int64_t most =
        per_cu ? static_cast<int64_t>(per_cu) * device_cus() : int64_t{1} << 21;
    const dim3 grid(static_cast<unsigned>(a.n_rows < most ? a.n_rows : most));
    hipLaunchKernelGGL(kernel, grid, block, lds, s, x, g, a.n_rows, a.vocab_local, a.ld, ldg, a.k,
                       st, cl, assumed, gdiv);
  };
  if (per_thread > 8) {
    static std::atomic<bool> lds_ok{false};
    const int rc = allow_lds(reinterpret_cast<const void*>(&distill_wide_row_kernel<T, kRagged>),
                             kWideLdsBytes, lds_ok);
    if (rc) return rc;
    run(distill_wide_row_kernel<T, kRagged>, 1, kWideLdsBytes);
  } else if (per_thread > 4) {
    run(distill_row_kernel<T, 8, kRagged>, 0, 0);
  } else {
    run(distill_row_kernel<T, 4, kRagged>, 0, 0);
  }
  return launch_status();
}

}  // namespace
}  // namespace nmce

using namespace nmce;

extern "C" {

int64_t nmce_distill_state_bytes(int64_t n_rows, int k) {
  if (n_rows < 0 || n_rows > (int64_t{1} << 22) || k < 1 || k > kMaxK) return -1;
  return align256(n_rows * static_cast<int64_t>(sizeof(Taught))) +
         align256(n_rows * static_cast<int64_t>(sizeof(Slope))) + align256(n_rows * 4) +
         3 * align256(n_rows * k * 4);
}

int nmce_distill_stats(const nmce_distill_batch* a, void* state, int64_t state_bytes,
                       double* stats, void* stream) {
  if (const int rc = check_batch(a)) return rc;
  if (a->n_rows == 0) return NMCE_OK;
  if (!stats) return NMCE_EINVAL_PTR;
  if (const int rc = check_state(state, state_bytes, a->n_rows, a->k)) return rc;
  const State st = state_of(state, a->n_rows, a->k);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (const int rc = launch_list(*a, st, nullptr, nullptr, s)) return rc;
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
                         float* mean, void* stream) {
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
  if (const int rc = launch_status()) return rc;
  return mean ? launch_mean(loss, n_rows, mean, static_cast<hipStream_t>(stream)) : NMCE_OK;
}

int nmce_distill_fwd_bwd(const nmce_distill_batch* a, void* grad, int64_t ld_grad, void* state,
                         int64_t state_bytes, float* loss, float* mean, const float* expected,
                         float* assumed, float gout_div, void* stream) {
  if (const int rc = check_batch(a)) return rc;
  const int64_t epv = a->dtype == NMCE_F32 ? 4 : 8;
  const uintptr_t es = 16 / epv;
  if (a->vocab_local > NMCE_DISTILL_ONE_PASS_BYTES / static_cast<int64_t>(es) ||
      a->vocab_start != 0 || a->vocab_total != a->vocab_local || ld_grad < a->vocab_local ||
      (grad == a->logits && ld_grad != a->ld) || !(gout_div > 0.0f))
    return NMCE_EINVAL_SHAPE;
  if (a->n_rows == 0) return NMCE_OK;
  if (!grad || !loss || !expected || !assumed) return NMCE_EINVAL_PTR;
  const uintptr_t px = reinterpret_cast<uintptr_t>(a->logits),
                  pg = reinterpret_cast<uintptr_t>(grad);
  // Rows of the gradient lie against 16-byte boundaries as the logits' do.
  if (pg % es || (px - pg) % 16 || ((a->ld - ld_grad) * static_cast<int64_t>(es)) % 16)
    return NMCE_EINVAL_ALIGN;
  if (const int rc = check_state(state, state_bytes, a->n_rows, a->k)) return rc;
  const State st = state_of(state, a->n_rows, a->k);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (const int rc = launch_list(*a, st, expected, assumed, s)) return rc;
  const float gdiv = gout_div * static_cast<float>(a->temperature);
  const bool ragged = px % 16 || a->vocab_local % epv || a->ld % epv || ld_grad % epv;
  int rc;
  if (a->dtype == NMCE_F32)
    rc = ragged ? launch_rows<float, true>(*a, grad, ld_grad, st, assumed, gdiv, s)
                : launch_rows<float, false>(*a, grad, ld_grad, st, assumed, gdiv, s);
  else
    rc = ragged ? launch_rows<uint16_t, true>(*a, grad, ld_grad, st, assumed, gdiv, s)
                : launch_rows<uint16_t, false>(*a, grad, ld_grad, st, assumed, gdiv, s);
  if (rc) return rc;
  const bool one = a->n_rows <= kLossBlock && mean;
  const int threads = one ? static_cast<int>(round_up(a->n_rows, 64)) : kLossRows;
  const dim3 blocks(static_cast<unsigned>((a->n_rows + threads - 1) / threads));
  hipLaunchKernelGGL(distill_loss_kernel, blocks, dim3(threads), 0, s, st, a->n_rows,
                     1.0 / a->temperature, loss, one ? mean : nullptr);
  if (const int rc2 = launch_status()) return rc2;
  return mean && !one ? launch_mean(loss, a->n_rows, mean, s) : NMCE_OK;
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
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t epv = 16 / static_cast<int64_t>(es), per_row = vocab_local / epv;
  if (!assumed && vocab_local % epv == 0 && ld % epv == 0 && ld_grad % epv == 0 &&
      aligned16(logits) && aligned16(grad) && n_rows * per_row < (int64_t{1} << 31) &&
      n_rows * k < (int64_t{1} << 31)) {
    const uint32_t n_vec = static_cast<uint32_t>(n_rows * per_row);
    constexpr int kEach = kFlatBlock * kFlatAhead;
    auto run = [&](auto element) {
      using T = decltype(element);
      hipLaunchKernelGGL(distill_flat_kernel<T>, dim3((n_vec + kEach - 1) / kEach),
                         dim3(kFlatBlock), 0, s, static_cast<const T*>(logits),
                         static_cast<T*>(grad), n_vec, static_cast<uint32_t>(per_row), ld, ld_grad,
                         st.slopes, cl, grad_output, gout_stride, gdiv);
      if (const int rc = launch_status()) return rc;
      hipLaunchKernelGGL(distill_listed_kernel<T>,
                         dim3(static_cast<unsigned>((n_rows * k + 255) / 256)), dim3(256), 0, s,
                         static_cast<T*>(grad), n_rows * k, ld_grad, k, st, cl, grad_output,
                         gout_stride, gdiv);
      return launch_status();
    };
    return dtype == NMCE_F32 ? run(float{}) : run(uint16_t{});
  }
  // After a one-pass forward the upstream value is usually the assumed one: a small
  // grid that walks the rows then ends at once.
  const int64_t most = assumed ? 2 * device_cus() : n_rows;
  const dim3 grid(static_cast<unsigned>(n_rows < most ? n_rows : most)), block(kBlock);
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
