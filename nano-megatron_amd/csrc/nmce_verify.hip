// Verification of drafted tokens against the target model's probabilities, from
// given uniform numbers, for gfx950. With p = softmax(x / T) of the target's
// logits and q = softmax(y / T) of the draft model's at a position,
//
//   the drafted token d stands while  u q(d) < p(d);
//   at the first that does not, the next token is drawn from max(p - q, 0)
//   (normalised); after the last draft, from p:
//   the first id j whose running sum of weights passes u' times all of them.
//
// T = 0 compares with the largest logit's id instead. Without draft logits q is
// one at the drafted token (a copied draft).
//
// Everything is 64 bits wide from the difference x - max on. A drawn id is the
// place where a running sum over the vocabulary passes a level: its neighbours'
// borders are 1e-5 and less apart, so sums off by 1e-7 would give other ids for
// the same numbers. The card's fp64 rate is that of its unpacked fp32; a logit costs
// 26 instructions, 16 of them fp64 sums and products, whose issue bounds the pass over
// the logits (64 x 11 rows of 128256 bf16 82 us, 2.2 TB/s, a third of the memory's rate;
// the VALU is busy 0.78 of the time).
//
// Three launches. The rows are cut into slabs of 8192 logits, a workgroup each,
// which holds its slab in registers: (1) every slab's (maximum, sum of
// exponentials, drafted token's logit, id of the maximum); (2) per sequence, from
// those, what stands and which row the next token comes from, and that row's
// weights summed by slab; (3) the slab in which the level lies, and the id
// within. With a sharded vocabulary the ranks exchange (1)'s and (2)'s results,
// 48 bytes a slab, and no logits.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "nmce.h"
#include "nmce_device.h"

namespace nmce {
namespace {

constexpr int kSlab = 8192;               // logits of a workgroup
constexpr int kStat = 4;                  // doubles of a slab's statistics
constexpr float kInf = __builtin_huge_valf();

// exp((x - m) / T) with c = log2(e) / T > 0; a masked logit's (-inf) is 0, for which
// m has to be a number (finite_max).
__device__ __forceinline__ double weight_of(float x, double m, double c) {
  return exp2_64((static_cast<double>(x) - m) * c);
}
__device__ __forceinline__ double finite_max(float m) {
  return m == -kInf ? 0.0 : static_cast<double>(m);
}

// A probability: its weight times the row's 1 / sum, rounded. Kept out of a fused
// multiply-add, so that p and q of equal rows are equal and p - q is nothing.
__device__ __forceinline__ double probability(double w, double inv) {
#pragma clang fp contract(off)
  return w * inv;
}

// What 64-bit rounding can leave of max(p - q, 0) over equal distributions.
constexpr double kNothing = 1e-14;

// The temperature of sequence b: not above zero (or NaN) is greedy, whose
// log-probabilities are those of T = 1.
__device__ __forceinline__ double inverse_temperature(const nmce_verify_batch& a, int64_t b,
                                                      bool* greedy) {
  const double t = a.temperature ? static_cast<double>(a.temperature[b]) : a.temperature_all;
  *greedy = !(t > 0.0);
  // (An infinite one is merely very large: every finite logit weighs 1. At the
  // smallest ones all below the largest weigh 0: two logits differ by 2^-149 or more.)
  return *greedy ? 1.0 : fmin(fmax(1.0 / t, 1e-300), 1e300);
}

// A uniform number: outside [0, 1) the nearest inside, NaN 0.
__device__ __forceinline__ double uniform(float u) {
  return u > 0.0f ? fmin(static_cast<double>(u), 1.0 - 0x1p-53) : 0.0;
}

__device__ __forceinline__ bool is_id(int64_t d, const nmce_verify_batch& a) {
  return d >= 0 && d < a.vocab_total;
}

// 16 bytes of logits at any element's alignment (the loads may straddle the
// 16-byte grid: rows of odd widths start anywhere).
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
  u32x4 v;
  memcpy(&v, p, 16);
  Elem<T>::unpack(v, f);
}

// A slab's logits from element c0 of the row, kSlab / kBlock a thread; -inf past its
// end. kInOrder: a thread's are consecutive; otherwise its vectors lie a block apart.
template <typename T, int kBlock, bool kInOrder>
__device__ __forceinline__ int64_t place(int64_t c0, int i) {
  constexpr int kEach = kSlab / kBlock;
  constexpr int kVec = Elem<T>::kPerVec;
  if constexpr (kInOrder) return c0 + threadIdx.x * kEach + i;
  return c0 + (static_cast<int64_t>(i / kVec) * kBlock + threadIdx.x) * kVec + i % kVec;
}
template <typename T, int kBlock, bool kInOrder>
__device__ __forceinline__ void load_slab(const T* __restrict__ row, int64_t c0, int64_t v,
                                          float* f) {
  constexpr int kVec = Elem<T>::kPerVec;
  constexpr int kEach = kSlab / kBlock;
#pragma unroll
  for (int i = 0; i < kEach; i += kVec) {
    const int64_t c = place<T, kBlock, kInOrder>(c0, i);
    if (c + kVec <= v) {
      load_vec(row + c, f + i);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) f[i + e] = c + e < v ? Elem<T>::load1(row + c + e) : -kInf;
    }
  }
}

__device__ __forceinline__ double wave_add(double v) {
  for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s);
  return v;
}

// ---- 1: every slab's statistics ---------------------------------------------
// Rows: the targets' (batch x (drafts + 1)), then the drafts' (batch x drafts).
// stats[row][slab] = {maximum, sum of exp((x - maximum) / T), the drafted token's
// logit (-inf where it is not in the slab), the lowest id of the maximum (of greedy
// sequences)}.
template <typename T, int kBlock>
__global__ __launch_bounds__(kBlock) void verify_stats_kernel(nmce_verify_batch a, int64_t slabs,
                                                              double* __restrict__ stats) {
  constexpr int kEach = kSlab / kBlock, kWaves = kBlock / 64;
  __shared__ float wave_m[kWaves];
  __shared__ double wave_s[kWaves];
  __shared__ int wave_i[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x / slabs, slab = blockIdx.x - row * slabs;
  const int64_t targets = a.batch * (a.drafts + 1);
  const bool target = row < targets;
  const int64_t per = target ? a.drafts + 1 : a.drafts;
  const int64_t r = target ? row : row - targets;
  const int64_t b = r / per, i = r - b * per;
  const T* x = target ? static_cast<const T*>(a.target) + b * a.target_batch_stride +
                            i * a.target_row_stride
                      : static_cast<const T*>(a.draft) + b * a.draft_batch_stride +
                            i * a.draft_row_stride;
  const int64_t c0 = slab * kSlab;
  float f[kEach];
  load_slab<T, kBlock, false>(x, c0, a.vocab_local, f);
  bool greedy;
  const double c = inverse_temperature(a, b, &greedy) * kLog2e64;
  float m = -kInf;
#pragma unroll
  for (int e = 0; e < kEach; ++e) m = fmaxf(m, f[e]);
  for (int s = 32; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
  if (lane == 0) wave_m[wave] = m;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, wave_m[w]);
  double sum = 0.0;
  const double at_m = finite_max(m);
#pragma unroll
  for (int e = 0; e < kEach; ++e) sum += weight_of(f[e], at_m, c);
  sum = wave_add(sum);
  int best = kSlab;
  if (greedy) {
#pragma unroll
    for (int e = kEach - 1; e >= 0; --e)
      if (f[e] == m) best = static_cast<int>(place<T, kBlock, false>(0, e));
    for (int s = 32; s > 0; s >>= 1) {
      const int o = __shfl_xor(best, s);
      best = o < best ? o : best;
    }
  }
  if (lane == 0) {
    wave_s[wave] = sum;
    wave_i[wave] = best;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWaves; ++w) {
      sum += wave_s[w];
      best = wave_i[w] < best ? wave_i[w] : best;
    }
    float xd = -kInf;
    if (i < a.drafts) {
      const int64_t d = a.draft_tokens[b * a.drafts + i];
      if (is_id(d, a)) {
        const int64_t at = d - a.vocab_start;
        if (at >= c0 && at < c0 + kSlab && at < a.vocab_local) xd = Elem<T>::load1(x + at);
      }
    }
    double* o = stats + blockIdx.x * static_cast<int64_t>(kStat);
    o[0] = m;
    o[1] = sum;
    o[2] = xd;
    o[3] = static_cast<double>(a.vocab_start + c0 + best);
  }
}

// ---- 2: what stands, and the next token's weights ------------------------------
struct Row {
  double m, s, xd, arg;
};

// (m, s) and (o.m, o.s) together. Where a maximum is -inf its sum is 0, or NaN.
__device__ __forceinline__ void merge(Row& a, const Row& o, double c) {
  if (o.m > a.m) {
    a.s = a.m == -kInf ? a.s + o.s : fma(a.s, exp2_64((a.m - o.m) * c), o.s);
    a.m = o.m;
    a.arg = o.arg;
  } else {
    a.s = o.m == -kInf ? a.s + o.s : fma(o.s, exp2_64((o.m - a.m) * c), a.s);
    if (o.m == a.m && o.arg < a.arg) a.arg = o.arg;
  }
  a.xd = fmax(a.xd, o.xd);
}

// Whether a row is a distribution: some logit above -inf, none +inf or NaN.
__device__ __forceinline__ bool is_distribution(const Row& r) {
  return r.m > -kInf && r.m < kInf && r.s > 0.0 && r.s < static_cast<double>(kInf);
}

// A row's statistics over all ranks' slabs, by 16 lanes; lane `sub` = 0 has them.
__device__ __forceinline__ Row merged_row(const double* __restrict__ stats, int64_t row,
                                          int64_t rows, int64_t slabs, int ranks, int sub,
                                          double c) {
  Row r{-static_cast<double>(kInf), 0.0, -static_cast<double>(kInf), 0.0};
  const int64_t parts = slabs * ranks;
  for (int64_t p = sub; p < parts; p += 16) {
    const int64_t rank = p / slabs, slab = p - rank * slabs;
    const double* o = stats + ((rank * rows + row) * slabs + slab) * kStat;
    merge(r, Row{o[0], o[1], o[2], o[3]}, c);
  }
  for (int s = 8; s > 0; s >>= 1) {
    const Row o{__shfl_xor(r.m, s), __shfl_xor(r.s, s), __shfl_xor(r.xd, s),
                __shfl_xor(r.arg, s)};
    merge(r, o, c);
  }
  return r;
}

enum Kind : int { kNone, kGreedy, kPlain, kRest, kWithout };

// Where the next token comes from. kNone: the target's row is no distribution;
// kGreedy: its largest logit's id; kPlain: p; kRest: max(p - q, 0); kWithout: p
// without the drafted token.
struct Decision {
  double pm, ps, qm, qs, arg;
  int64_t accepted, draft;
  int kind;
};

template <typename T>
struct Weights {
  const T* x;
  const T* y;
  double pm, pi, qm, qi, c;  // maxima, reciprocals of the sums, log2(e) / T
  int64_t skip;              // local id left out, or -1
  bool rest;

  __device__ __forceinline__ void init(const nmce_verify_batch& a, int64_t b, const Decision& d,
                                       double c_) {
    x = static_cast<const T*>(a.target) + b * a.target_batch_stride +
        d.accepted * a.target_row_stride;
    y = d.kind == kRest ? static_cast<const T*>(a.draft) + b * a.draft_batch_stride +
                              d.accepted * a.draft_row_stride
                        : nullptr;
    pm = d.pm;
    pi = 1.0 / d.ps;
    qm = d.qm;
    qi = 1.0 / d.qs;
    c = c_;
    skip = d.kind == kWithout ? d.draft - a.vocab_start : -1;
    rest = d.kind == kRest;
  }
};

template <typename T, int kBlock>
__global__ __launch_bounds__(kBlock) void verify_masses_kernel(
    nmce_verify_batch a, int64_t slabs, int ranks, const double* __restrict__ stats,
    Decision* __restrict__ decisions, double* __restrict__ masses, int64_t* __restrict__ tokens,
    int64_t* __restrict__ accepted, float* __restrict__ logprobs) {
  constexpr int kEach = kSlab / kBlock, kWaves = kBlock / 64;
  constexpr int kAtOnce = kBlock / 16;
  __shared__ bool stands[kAtOnce];
  __shared__ Decision dec[kAtOnce];
  __shared__ float logp[kAtOnce];
  __shared__ Decision chosen;
  __shared__ double wave_r[kWaves], wave_p[kWaves];
  const int64_t b = blockIdx.x / slabs, slab = blockIdx.x - b * slabs;
  const int64_t rows = a.batch * (a.drafts + 1) + (a.draft ? a.batch * a.drafts : 0);
  const int64_t k = a.drafts;
  bool greedy;
  const double it = inverse_temperature(a, b, &greedy);
  const double c = it * kLog2e64;
  const int slot = threadIdx.x >> 4, sub = threadIdx.x & 15;
  const bool first = slab == 0;

  // A position for every 16 threads at a time, until one does not stand.
  for (int64_t base = 0; base <= k; base += kAtOnce) {
    const int64_t i = base + slot;
    if (i <= k) {
      const Row p = merged_row(stats, b * (k + 1) + i, rows, slabs, ranks, sub, c);
      const bool has = i < k && is_id(a.draft_tokens[b * k + (i < k ? i : 0)], a);
      Row q{0.0, 1.0, 0.0, 0.0};
      if (has && a.draft)
        q = merged_row(stats, a.batch * (k + 1) + b * k + i, rows, slabs, ranks, sub, c);
      if (sub == 0) {
        const bool pv = is_distribution(p), qv = !a.draft || is_distribution(q);
        Decision d{p.m, p.s, q.m, q.s, p.arg, i, has ? a.draft_tokens[b * k + i] : -1, kNone};
        bool ok = false;
        if (pv && greedy) {
          d.kind = kGreedy;
          ok = has && static_cast<double>(d.draft) == p.arg;
        } else if (pv) {
          d.kind = has && qv ? (a.draft ? kRest : kWithout) : kPlain;
          if (has && qv) {
            const double pd = p.xd == -kInf ? 0.0 : exp2_64((p.xd - p.m) * c) / p.s;
            const double qd = !a.draft ? 1.0
                              : q.xd == -kInf ? 0.0 : exp2_64((q.xd - q.m) * c) / q.s;
            ok = uniform(a.accept_u[b * k + i]) * qd < pd;
          }
        }
        stands[slot] = ok;
        dec[slot] = d;
        logp[slot] = ok ? static_cast<float>((p.xd - p.m) * it - log(p.s)) : 0.0f;
      }
    }
    __syncthreads();
    const int64_t here = k + 1 - base < kAtOnce ? k + 1 - base : kAtOnce;
    int n = 0;
    while (n < here && stands[n]) ++n;  // every thread counts the same
    if (first && threadIdx.x < n) {
      tokens[b * (k + 1) + base + threadIdx.x] = dec[threadIdx.x].draft;
      logprobs[b * (k + 1) + base + threadIdx.x] = logp[threadIdx.x];
    }
    if (n < here) {
      if (threadIdx.x == 0) chosen = dec[n];
      __syncthreads();
      break;
    }
    __syncthreads();  // the next positions reuse the arrays
  }
  // (Position k holds no draft, so one is always found.)
  if (first) {
    if (threadIdx.x == 0) {
      accepted[b] = chosen.accepted;
      decisions[b] = chosen;
    }
    for (int64_t i = chosen.accepted + threadIdx.x; i <= k; i += kBlock) {
      tokens[b * (k + 1) + i] = -1;
      logprobs[b * (k + 1) + i] = 0.0f;
    }
  }
  double rest = 0.0, plain = 0.0;
  if (chosen.kind >= kPlain) {
    Weights<T> w;
    w.init(a, b, chosen, c);
    const int64_t c0 = slab * kSlab;
    float f[kEach];
    load_slab<T, kBlock, false>(w.x, c0, a.vocab_local, f);
    if (w.rest) {
      float g[kEach];
      load_slab<T, kBlock, false>(w.y, c0, a.vocab_local, g);
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const double p = probability(weight_of(f[e], w.pm, c), w.pi);
        plain += p;
        rest += fmax(p - probability(weight_of(g[e], w.qm, c), w.qi), 0.0);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const double p = probability(weight_of(f[e], w.pm, c), w.pi);
        plain += p;
        rest += place<T, kBlock, false>(c0, e) == w.skip ? 0.0 : p;
      }
    }
  }
  rest = wave_add(rest);
  plain = wave_add(plain);
  if ((threadIdx.x & 63) == 0) {
    wave_r[threadIdx.x >> 6] = rest;
    wave_p[threadIdx.x >> 6] = plain;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWaves; ++w) {
      rest += wave_r[w];
      plain += wave_p[w];
    }
    masses[2 * blockIdx.x] = rest;
    masses[2 * blockIdx.x + 1] = plain;
  }
}

// ---- 3: the next token ---------------------------------------------------------
// masses [ranks][batch][slabs][2]. A workgroup per sequence finds the slab, and,
// where it is this rank's, the id within: picked[b] = {id, log-probability}, or
// {-1, -inf} on the other ranks. Without `picked` (one rank) the outputs
// themselves are written.
template <typename T, int kBlock>
__global__ __launch_bounds__(kBlock) void verify_pick_kernel(
    nmce_verify_batch a, int64_t slabs, int ranks, int rank,
    const Decision* __restrict__ decisions, const double* __restrict__ masses,
    int64_t* __restrict__ tokens, float* __restrict__ logprobs, double* __restrict__ picked) {
  constexpr int kEach = kSlab / kBlock, kWaves = kBlock / 64;
  __shared__ double part[kBlock];
  __shared__ double wave_sum[kWaves];
  __shared__ int last_s[kWaves];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Decision d = decisions[b];
  bool greedy;
  const double it = inverse_temperature(a, b, &greedy);
  const double c = it * kLog2e64;
  auto put = [&](double id, double lp) {
    if (picked) {
      picked[2 * b] = id;
      picked[2 * b + 1] = lp;
    } else {
      tokens[b * (a.drafts + 1) + d.accepted] = static_cast<int64_t>(id);
      logprobs[b * (a.drafts + 1) + d.accepted] = id < 0.0 ? 0.0f : static_cast<float>(lp);
    }
  };
  if (d.kind <= kGreedy) {
    if (tid == 0)
      put(d.kind == kGreedy ? d.arg : -1.0,
          d.kind == kGreedy ? -log(d.ps) : -static_cast<double>(kInf));
    return;
  }
  // The slabs' masses in the vocabulary's order: their totals, then the slab in
  // which the level is passed.
  const int64_t parts = slabs * ranks;
  auto mass = [&](int64_t p, int which) {
    const int64_t r = p / slabs, s = p - r * slabs;
    return masses[((r * a.batch + b) * slabs + s) * 2 + which];
  };
  double total = 0.0;
  int which = d.kind == kPlain ? 1 : 0;
  for (;; which = 1) {
    total = 0.0;
    for (int64_t p0 = 0; p0 < parts; p0 += kBlock) {
      part[tid] = p0 + tid < parts ? mass(p0 + tid, which) : 0.0;
      __syncthreads();
      const int n = static_cast<int>(parts - p0 < kBlock ? parts - p0 : kBlock);
      for (int j = 0; j < n; ++j) total += part[j];
      __syncthreads();
    }
    // Nothing left of p above q (both rule the draft out): from p.
    if (which == 1 || total > (d.kind == kRest ? kNothing : 0.0)) break;
  }
  const double goal = uniform(a.sample_u[b]) * total;
  double before = 0.0, at_before = 0.0;
  int64_t at = -1;
  for (int64_t p0 = 0; p0 < parts && (at < 0 || before <= goal); p0 += kBlock) {
    part[tid] = p0 + tid < parts ? mass(p0 + tid, which) : 0.0;
    __syncthreads();
    const int n = static_cast<int>(parts - p0 < kBlock ? parts - p0 : kBlock);
    for (int j = 0; j < n && before <= goal; ++j) {
      if (part[j] > 0.0) {  // the last one with weight, if rounding passes none
        at = p0 + j;
        at_before = before;
      }
      before += part[j];
    }
    __syncthreads();
  }
  const int64_t owner = at / slabs;
  if (at < 0 || owner != rank) {
    if (tid == 0) put(-1.0, -static_cast<double>(kInf));
    return;
  }
  const double level = goal - at_before;
  const int64_t c0 = (at - owner * slabs) * kSlab;

  Weights<T> w;
  w.init(a, b, d, c);
  float f[kEach];
  load_slab<T, kBlock, true>(w.x, c0, a.vocab_local, f);
  double wt[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) wt[e] = probability(weight_of(f[e], w.pm, c), w.pi);
  if (which == 0 && w.rest) {
    float g[kEach];
    load_slab<T, kBlock, true>(w.y, c0, a.vocab_local, g);
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      wt[e] = fmax(wt[e] - probability(weight_of(g[e], w.qm, c), w.qi), 0.0);
  } else if (which == 0) {
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (place<T, kBlock, true>(c0, e) == w.skip) wt[e] = 0.0;
  }
  // Sums before each thread's 32, and the last thread with any weight.
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) sum += wt[e];
  double incl = sum;
  for (int s = 1; s < 64; s <<= 1) {
    const double o = __shfl_up(incl, s);
    if (lane >= s) incl += o;
  }
  const uint64_t some = __ballot(sum > 0.0);
  if (lane == 63) wave_sum[wave] = incl;
  if (lane == 0) last_s[wave] = some ? wave * 64 + 63 - __clzll(some) : -1;
  __syncthreads();
  double ahead = 0.0;
  int last = -1;
  for (int v = 0; v < kWaves; ++v) {
    if (v < wave) ahead += wave_sum[v];
    last = last_s[v] > last ? last_s[v] : last;
  }
  const double upto = ahead + incl, from = upto - sum;
  // The first thread whose sums pass the level, the last with weight if none does.
  const uint64_t passes = __ballot(upto > level && sum > 0.0);
  __syncthreads();
  if (lane == 0)
    last_s[wave] = passes ? wave * 64 + __builtin_ctzll(passes) : kBlock;
  __syncthreads();
  int who = kBlock;
  for (int v = 0; v < kWaves; ++v) who = last_s[v] < who ? last_s[v] : who;
  if (who == kBlock) who = last;
  if (tid == who) {
    double run = from;
    int pick = -1;
    bool done = false;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (!done && wt[e] > 0.0) {
        pick = e;
        run += wt[e];
        done = run > level;
      }
    }
    float x = 0.0f;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (e == pick) x = f[e];
    put(static_cast<double>(a.vocab_start + c0 + tid * kEach + pick),
        (static_cast<double>(x) - d.pm) * it - log(d.ps));
  }
}

// The ranks' picks, merged by their maximum, into the outputs.
__global__ __launch_bounds__(256) void verify_finish_kernel(
    const double* __restrict__ picked, const Decision* __restrict__ decisions, int64_t batch,
    int64_t drafts, int64_t* __restrict__ tokens, float* __restrict__ logprobs) {
  const int64_t b = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (b >= batch) return;
  const double id = picked[2 * b];
  const int64_t o = b * (drafts + 1) + decisions[b].accepted;
  tokens[o] = static_cast<int64_t>(id);
  logprobs[o] = id < 0.0 ? 0.0f : static_cast<float>(picked[2 * b + 1]);
}

// ---- host -------------------------------------------------------------------
inline int64_t slabs_of(int64_t v) { return (v + kSlab - 1) / kSlab; }

int check_batch(const nmce_verify_batch* a) {
  if (!a) return NMCE_EINVAL_PTR;
  if (a->dtype != NMCE_F32 && a->dtype != NMCE_BF16) return NMCE_EINVAL_DTYPE;
  const int64_t most = (int64_t{1} << 31) - 1;
  if (a->batch < 0 || a->batch > most || a->drafts < 0 || a->drafts > most || a->vocab_local < 1 ||
      a->vocab_local > most || a->vocab_start < 0 || a->vocab_total > most ||
      a->vocab_total < a->vocab_local || a->vocab_start > a->vocab_total - a->vocab_local)
    return NMCE_EINVAL_SHAPE;
  // A launch's workgroups times their threads fit 32 bits.
  if ((2 * a->drafts + 1) * a->batch > (int64_t{1} << 23) ||
      (2 * a->drafts + 1) * a->batch * slabs_of(a->vocab_local) > (int64_t{1} << 23))
    return NMCE_EINVAL_SHAPE;
  if (a->batch == 0) return NMCE_OK;
  if (!a->target || !a->sample_u || (a->drafts > 0 && (!a->draft_tokens || !a->accept_u)))
    return NMCE_EINVAL_PTR;
  const uintptr_t es = a->dtype == NMCE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a->target) % es || reinterpret_cast<uintptr_t>(a->draft) % es)
    return NMCE_EINVAL_ALIGN;
  return NMCE_OK;
}

// A slab a workgroup of 256 threads, 32 logits each; of 1024 and 8 where there is no
// workgroup for every compute unit, and one thread's chain of exponentials is the
// time: one sequence of four drafts over 50257 fp32 takes 6, 12 and 8 us in the three
// kernels, and 8, 16 and 14 with 256 threads.
inline bool few(int64_t workgroups) { return workgroups <= device_cus(); }

int64_t rows_of(const nmce_verify_batch& a) {
  return a.batch * (a.drafts + 1) + (a.draft ? a.batch * a.drafts : 0);
}

}  // namespace
}  // namespace nmce

using namespace nmce;

extern "C" {

int64_t nmce_verify_slabs(int64_t vocab_local) {
  return vocab_local < 1 ? -1 : slabs_of(vocab_local);
}

int64_t nmce_verify_workspace_bytes(int64_t batch) {
  return batch < 0 ? -1 : align256(batch * static_cast<int64_t>(sizeof(Decision)));
}

int nmce_verify_stats(const nmce_verify_batch* a, double* stats, void* stream) {
  if (const int st = check_batch(a)) return st;
  if (a->batch == 0) return NMCE_OK;
  if (!stats) return NMCE_EINVAL_PTR;
  const int64_t slabs = slabs_of(a->vocab_local);
  const dim3 grid(static_cast<unsigned>(rows_of(*a) * slabs));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool small = few(grid.x);
  auto run = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, *a, slabs, stats);
  };
  if (a->dtype == NMCE_F32)
    small ? run(verify_stats_kernel<float, 1024>, 1024) : run(verify_stats_kernel<float, 256>, 256);
  else
    small ? run(verify_stats_kernel<uint16_t, 1024>, 1024) : run(verify_stats_kernel<uint16_t, 256>, 256);
  return launch_status();
}

int nmce_verify_masses(const nmce_verify_batch* a, const double* stats, int ranks, double* masses,
                       int64_t* tokens, int64_t* accepted, float* logprobs, void* workspace,
                       int64_t workspace_bytes, void* stream) {
  if (const int st = check_batch(a)) return st;
  if (ranks < 1) return NMCE_EINVAL_TP;
  if (a->batch == 0) return NMCE_OK;
  if (!stats || !masses || !tokens || !accepted || !logprobs) return NMCE_EINVAL_PTR;
  if (!workspace || !aligned16(workspace) ||
      workspace_bytes < nmce_verify_workspace_bytes(a->batch))
    return NMCE_EINVAL_WORKSPACE;
  const int64_t slabs = slabs_of(a->vocab_local);
  const dim3 grid(static_cast<unsigned>(a->batch * slabs));
  hipStream_t s = static_cast<hipStream_t>(stream);
  Decision* dec = static_cast<Decision*>(workspace);
  const bool small = few(grid.x);
  auto run = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, *a, slabs, ranks, stats, dec, masses, tokens, accepted, logprobs);
  };
  if (a->dtype == NMCE_F32)
    small ? run(verify_masses_kernel<float, 1024>, 1024) : run(verify_masses_kernel<float, 256>, 256);
  else
    small ? run(verify_masses_kernel<uint16_t, 1024>, 1024) : run(verify_masses_kernel<uint16_t, 256>, 256);
  return launch_status();
}

int nmce_verify_pick(const nmce_verify_batch* a, const double* masses, int ranks, int rank,
                     const void* workspace, int64_t workspace_bytes, int64_t* tokens,
                     float* logprobs, double* picked, void* stream) {
  if (const int st = check_batch(a)) return st;
  if (ranks < 1 || rank < 0 || rank >= ranks) return NMCE_EINVAL_TP;
  if (a->batch == 0) return NMCE_OK;
  if (!masses || (!picked && (!tokens || !logprobs || ranks > 1))) return NMCE_EINVAL_PTR;
  if (!workspace || !aligned16(workspace) ||
      workspace_bytes < nmce_verify_workspace_bytes(a->batch))
    return NMCE_EINVAL_WORKSPACE;
  const int64_t slabs = slabs_of(a->vocab_local);
  const dim3 grid(static_cast<unsigned>(a->batch));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Decision* dec = static_cast<const Decision*>(workspace);
  const bool small = few(grid.x);
  auto run = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, *a, slabs, ranks, rank, dec, masses, tokens, logprobs, picked);
  };
  if (a->dtype == NMCE_F32)
    small ? run(verify_pick_kernel<float, 1024>, 1024) : run(verify_pick_kernel<float, 256>, 256);
  else
    small ? run(verify_pick_kernel<uint16_t, 1024>, 1024) : run(verify_pick_kernel<uint16_t, 256>, 256);
  return launch_status();
}

int nmce_verify_finish(const double* picked, const void* workspace, int64_t workspace_bytes,
                       int64_t batch, int64_t drafts, int64_t* tokens, float* logprobs,
                       void* stream) {
  if (batch < 0 || drafts < 0 || batch > (int64_t{1} << 23)) return NMCE_EINVAL_SHAPE;
  if (batch == 0) return NMCE_OK;
  if (!picked || !tokens || !logprobs) return NMCE_EINVAL_PTR;
  if (!workspace || !aligned16(workspace) || workspace_bytes < nmce_verify_workspace_bytes(batch))
    return NMCE_EINVAL_WORKSPACE;
  const dim3 grid(static_cast<unsigned>((batch + 255) / 256)), block(256);
  hipLaunchKernelGGL(verify_finish_kernel, grid, block, 0, static_cast<hipStream_t>(stream),
                     picked, static_cast<const Decision*>(workspace), batch, drafts, tokens,
                     logprobs);
  return launch_status();
}

}  // extern "C"
