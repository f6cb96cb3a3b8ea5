// 8-bit rows and their product for gfx950: logits from an 8-bit LM head.
//
//   quantise   s_r = max_k |x[r, k]| / 127,  q[r, k] = x[r, k] / s_r to the nearest
//              integer, halves to the even one
//   product    y[n, v] = (sum_k q[n, k] w[v, k]) * sx[n] * sw[v]
//
// q is formed from 127 x / max|x|, whose halves are exact: an element of half
// the largest magnitude gives 63.5 (bf16 has only 8 bits, so such elements are
// common), which a quotient by the rounded scale would send to either side. The
// integer sums are exact in 32 bits up to K = 131072 (127^2 K < 2^31); the
// conversion to fp32 and the two scales round once each.
//
// The product runs on the 16-bit products' core (nmce_gemm.h), whose fragments
// are 16 bytes a lane whatever they hold, at twice the rate.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include <type_traits>

#include "nmce.h"
#include "nmce_device.h"
#include "nmce_gemm.h"

namespace nmce {
namespace {

constexpr int64_t kMaxK = 131072;
constexpr int kFewTokens = 128;  // up to here the weight streams through registers
constexpr int kPadK = 256;  // the tokens' rows are padded to it with zeros: whole steps of K

// A vector's elements as x * 127 / top to the nearest integer, halves to even, as
// the exact quotient rounds; the result is one byte an element. Adding 1.5 * 2^23
// rounds to the integers, whose low byte then lies in the sum's own.
constexpr float kRound = 12582912.0f;

__device__ __forceinline__ uint32_t bytes_of(float a, float b, float c, float d) {
  // v_perm_b32: bytes 0-3 are the second operand's, 4-7 the first's
  const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x04000c0cu);
  return lo | hi;
}

// fp32: the product with inv = 127 / top is off by at most 127 * 2^-23 = 1.6e-5.
// Only where one of the elements lies that near to a half its side of it is settled:
// 127 |x| against h top for the half h, as the fp32 sum of 127 |x| - hi (hi its
// rounding) and hi - h top, both exact (the second cancels at least 16 bits of a
// 32-bit product), whose sign is therefore exact.
__device__ __forceinline__ void quantise(const float (&x)[4], float top, uint32_t* q) {
  constexpr float kNear = 2e-5f;
  const float inv = 127.0f / top;
  float u[4], off = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float t = x[e] * inv;
    u[e] = t + kRound;
    off = fmaxf(off, fabsf(t - (u[e] - kRound)));
  }
  if (off > 0.5f - kNear) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = fabsf(x[e]), t = a * inv, k = floorf(t), h = k + 0.5f;
      if (fabsf(t - h) < kNear) {
        const float hi = 127.0f * a, lo = fmaf(127.0f, a, -hi);
        const float s = fmaf(-h, top, hi) + lo;
        const bool up = s > 0.0f || (s == 0.0f && (static_cast<int>(k) & 1));
        u[e] = (x[e] < 0.0f ? -(up ? k + 1.0f : k) : (up ? k + 1.0f : k)) + kRound;
      }
    }
  }
  q[0] = bytes_of(u[0], u[1], u[2], u[3]);
}

// bf16: halves are common (every element of half the largest magnitude), and 127 x
// is exact in fp32. t = 127 x / top is formed by its reciprocal and corrected by its
// exact remainder, which gives every quotient that fp32 holds, halves among them.
// The others differ from every half by 1.5e-5 of it or more (over all pairs of
// mantissas; the nearest are next to 126.5 and to 1/2), and t is off by 1.2e-7 of
// itself at most. The correction is for the halves: a bare product with the
// reciprocal leaves them on either side.
__device__ __forceinline__ void quantise(const float (&x)[8], float top, uint32_t* q) {
  const float inv = 1.0f / top;
  float u[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float p = 127.0f * x[e], t = p * inv;
    u[e] = fmaf(fmaf(-t, top, p), inv, t) + kRound;
  }
  q[0] = bytes_of(u[0], u[1], u[2], u[3]);
  q[1] = bytes_of(u[4], u[5], u[6], u[7]);
}

// Where those would leave fp32's range: the quotient in fp64, where 127 x is exact
// and a 31-bit over a 24-bit number is a half only if it is one exactly.
template <int kVec>
__device__ __forceinline__ void quantise_wide(const float (&x)[kVec], float top, uint32_t* q) {
  float u[kVec];
#pragma unroll
  for (int e = 0; e < kVec; ++e)
    u[e] = static_cast<float>(
               rint(127.0 * static_cast<double>(x[e]) / static_cast<double>(top))) + kRound;
#pragma unroll
  for (int w = 0; w < kVec / 4; ++w)
    q[w] = bytes_of(u[4 * w], u[4 * w + 1], u[4 * w + 2], u[4 * w + 3]);
}

// The largest magnitude as the integer of its bits, which puts infinities and NaNs
// above every number: running maxima of a vector's elements (bf16: of its even and
// odd ones), and the fp32 bits of the largest of them.
__device__ __forceinline__ void raise(uint32_t& top, const u32x4& v, float) {
  const u32x4 m = v & 0x7fffffffu;
  const uint32_t a = m.x > m.y ? m.x : m.y, b = m.z > m.w ? m.z : m.w;
  const uint32_t c = a > b ? a : b;
  top = c > top ? c : top;
}
__device__ __forceinline__ void raise(uint32_t& top, const u32x4& v, uint16_t) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  // (By value: of a vector's element itself the cast takes the first one's bits.)
  auto pair = [](uint32_t w) { return __builtin_bit_cast(u16x2, w & 0x7fff7fffu); };
  u16x2 t = __builtin_bit_cast(u16x2, top);
  t = __builtin_elementwise_max(t, pair(v.x));
  t = __builtin_elementwise_max(t, pair(v.y));
  t = __builtin_elementwise_max(t, pair(v.z));
  t = __builtin_elementwise_max(t, pair(v.w));
  top = __builtin_bit_cast(uint32_t, t);
}
__device__ __forceinline__ uint32_t top_bits(uint32_t top, float) { return top; }
__device__ __forceinline__ uint32_t top_bits(uint32_t top, uint16_t) {
  const uint32_t lo = top << 16, hi = top & 0xffff0000u;
  return lo > hi ? lo : hi;
}

// kRow threads quantise a row: its largest magnitude, then the elements, which a
// thread holds in registers (32 of them; kHeld = false: longer rows, read twice). A
// row with an infinity or a NaN gets the scale NaN and zeros, so its products are
// NaN; a row of zeros gets the scale 0. A wave or a part of one needs no barrier;
// four waves are faster for few rows. 50257 rows of 1600 bf16 take 47 us (5.2 TB/s),
// of fp32 73 (5.5); read twice an element at a time by a workgroup each, 136.
constexpr int kQuantEach = 32;

template <typename T, int kRow, bool kHeld>
__global__ __launch_bounds__(kRow < 256 ? 256 : kRow) void quantize_rows_kernel(
    const T* __restrict__ x, int64_t n, int64_t k, int64_t ldx, int8_t* __restrict__ q,
    int64_t ldq, float* __restrict__ scale, bool whole_stores) {
  constexpr int kVec = Elem<T>::kPerVec;
  constexpr int kWaves = kRow < 64 ? 1 : kRow / 64;
  constexpr int kRowsAtOnce = (kRow < 256 ? 256 : kRow) / kRow;
  constexpr int kSpan = kRow * kVec;           // columns a round of vectors covers
  constexpr int kVecs = kQuantEach / kVec;
  // 16 bytes of elements at any element's alignment.
  typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
  typedef typename std::conditional<kHeld, int, int64_t>::type col_t;
  __shared__ uint32_t wave_top[kWaves];
  const int t = threadIdx.x % kRow;
  const col_t cols = static_cast<col_t>(k);
  auto get = [&](const T* row, col_t c) {
    if (c + kVec <= cols) {
      const u32x4_any v = *reinterpret_cast<const u32x4_any*>(row + c);
      return u32x4{v.x, v.y, v.z, v.w};
    }
    float f[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) f[e] = c + e < cols ? Elem<T>::load1(row + c + e) : 0.0f;
    return Elem<T>::pack(f);
  };
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kRowsAtOnce + threadIdx.x / kRow; r < n;
       r += static_cast<int64_t>(gridDim.x) * kRowsAtOnce) {
    const T* row = x + r * ldx;
    u32x4 held[kHeld ? kVecs : 1];
    uint32_t top = 0;
    if constexpr (kHeld) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) held[i] = get(row, i * kSpan + t * kVec);
#pragma unroll
      for (int i = 0; i < kVecs; ++i) raise(top, held[i], T());
    } else {
      for (int64_t c = t * kVec; c < k; c += kSpan) raise(top, get(row, c), T());
    }
    top = top_bits(top, T());
    for (int s = (kRow < 64 ? kRow : 64) / 2; s > 0; s >>= 1) {
      const uint32_t o = __shfl_xor(top, s);
      top = o > top ? o : top;
    }
    if constexpr (kWaves > 1) {
      if ((t & 63) == 0) wave_top[t >> 6] = top;
      __syncthreads();
      for (int w = 0; w < kWaves; ++w) top = wave_top[w] > top ? wave_top[w] : top;
      __syncthreads();
    }
    const bool finite = top < 0x7f800000u;
    const float most = __uint_as_float(top);
    if (t == 0)
      scale[r] = finite ? static_cast<float>(static_cast<double>(most) / 127.0)
                        : __uint_as_float(0x7fc00000u);
    const bool any = finite && top != 0;
    const bool wide = !(most > 1e-25f && most < 1e36f);
    int8_t* out = q + r * ldq;
    // kVec columns from c on, zeros past the row's.
    auto put = [&](int64_t c, const u32x4& v) {
      uint32_t word[kVec / 4] = {};
      if (any) {
        float f[kVec];
        Elem<T>::unpack(v, f);
        if (wide)
          quantise_wide<kVec>(f, most, word);
        else
          quantise(f, most, word);
      }
      if (whole_stores && c + kVec <= ldq) {
        typedef uint32_t word_t __attribute__((ext_vector_type(kVec / 4)));
        word_t w;
        memcpy(&w, word, kVec);
        *reinterpret_cast<word_t*>(out + c) = w;
      } else {
        for (int e = 0; e < kVec && c + e < ldq; ++e)
          out[c + e] = static_cast<int8_t>(word[e / 4] >> (8 * (e % 4)));
      }
    };
    if constexpr (kHeld) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int c = i * kSpan + t * kVec;
        if (c < ldq) put(c, held[i]);
      }
    }
    for (int64_t c = (kHeld ? int64_t{kQuantEach} * kRow : 0) + t * kVec; c < ldq; c += kSpan)
      put(c, kHeld ? u32x4{0, 0, 0, 0} : get(row, static_cast<col_t>(c)));
  }
}

struct LinearArgs {
  const int8_t* q;      // [n, kp], zeros from K on
  const float* sx;      // [n]
  const int8_t* w;      // [v, ldw]
  const float* sw;      // [v]
  void* out;            // [n, ldo]
  int64_t n, v, kp, ldw, ldo, w_chunks;
};

// A 256 x 256 tile of the logits (rows: tokens). [2048, 4096] x [128256, 4096] takes
// 805 us among other calls and 930 in an unbroken row (2.67 and 2.3 POP/s: the core's
// MFMA stream, as in bf16, and the clock that the chip's power leaves it), [4096, 64] x
// [50304, 64], all epilogue, 130 (3.2 TB/s of logits).
template <typename O, bool kVec>
__global__ __launch_bounds__(kThreads, 1) void int8_linear_kernel(LinearArgs a) {
  extern __shared__ __align__(16) char lds[];
  const int tiles_m = static_cast<int>((a.n + kBM - 1) / kBM);
  const int tiles_n = static_cast<int>((a.v + kBN - 1) / kBN);
  int tm, tn;
  tile_coords(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int64_t m0 = static_cast<int64_t>(tm) * kBM, n0 = static_cast<int64_t>(tn) * kBN;
  Acc acc;
  gemm_mainloop<false, false, /*kRows=*/true, /*kI8=*/true>(
      reinterpret_cast<const uint16_t*>(a.q), a.kp / 2, a.n,
      reinterpret_cast<const uint16_t*>(a.w), a.ldw / 2, a.v, a.kp / 2, m0, n0, lds, acc,
      a.kp / 16, a.w_chunks);
  // The scales: of the lane's rows 16 i + l % 16, of its columns 16 j + 4 g + e.
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row0 = m0 + (wave / kWavesN) * kWaveM + (lane & 15);
  const int64_t col0 = n0 + (wave % kWavesN) * kWaveN + 4 * (lane >> 4);
  float sx[kF];
#pragma unroll
  for (int i = 0; i < kF; ++i) {
    const int64_t r = row0 + 16 * i;
    sx[i] = a.sx[r < a.n ? r : a.n - 1];
  }
#pragma unroll
  for (int j = 0; j < kF; ++j) {
    float sw[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t c = col0 + 16 * j + e;
      sw[e] = a.sw[c < a.v ? c : a.v - 1];
    }
#pragma unroll
    for (int i = 0; i < kF; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc.c[i][j][e] = static_cast<float>(__float_as_int(acc.c[i][j][e])) * sx[i] * sw[e];
  }
  // Rows of any width and start: 16-byte stores need no more than their element's
  // alignment here, so only a tile that reaches past the last column goes element by
  // element.
  if constexpr (std::is_same<O, float>::value) {
    float* out = static_cast<float*>(a.out);
    if (kVec && n0 + kBN <= a.v)
      store_f32_tile<1, kVec>(acc, lds, out, nullptr, a.ldo, a.n, a.v, m0, n0);
    else
      store_f32_tile<1, false>(acc, lds, out, nullptr, a.ldo, a.n, a.v, m0, n0);
  } else {
    store_bf16_tile<true>(acc, lds, static_cast<uint16_t*>(a.out), a.ldo, a.n, a.v, m0, n0);
  }
}

// ---- few tokens -------------------------------------------------------------
// Up to kFewTokens tokens the weight's read is the time: every wave takes 16
// vocabulary rows of it straight into registers, 256-byte steps of K ahead, and
// all eight share the tokens' steps in LDS, loaded there directly, kDepth of them.
// A compute unit so has 64 to 128 KiB of the weight in flight. Over [128256, 4096]
// the product of one token takes 98 us (5.4 TB/s), quantised and all 104; 16 take 109,
// 64 123, 128 142. With the waves splitting K instead, each with its tokens from L2,
// one took 102, 16 124, 64 212; with 32 rows a wave 116, 118 and 183; the 256 x 256
// tiles of the core 136 for any.
//
// Fragments as in the core: A is 16 vocabulary rows, B 16 tokens, lane l holds row
// (token) l % 16, bytes 16 (l / 16) .. of each 64; the result's lane l has token
// l % 16, rows 4 (l / 16) + e. A token's step is 16 chunks of 16 bytes, chunk c of
// token t at c ^ (t % 16): the 16 tokens that 16 lanes read are on distinct bank
// groups.
constexpr int kStepK = 256;
constexpr int kFewWavesWg = 8;
typedef int i32x4v __attribute__((ext_vector_type(4)));

template <typename O, int kTokFrags, int kDepth>
__global__ __launch_bounds__(64 * kFewWavesWg, 4) void int8_few_kernel(LinearArgs a) {
  constexpr int kStage = 16 * kTokFrags * kStepK;
  constexpr int kBlocks = kStage / 1024;       // 1 KiB: four tokens' steps
  constexpr int kSlices = kStepK / 64;
  // A resource's size, past every offset here; a step past the last reads at it,
  // which is out of range: no memory access, and the loads in flight stay counted.
  constexpr uint32_t kPast = 1u << 31;
  __shared__ __align__(16) char lds[kDepth][kStage];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int64_t v0 = (static_cast<int64_t>(blockIdx.x) * kFewWavesWg + wave) * 16;
  const int64_t base = v0 < a.v ? v0 : a.v - 1;  // waves past the last row repeat it
  const int64_t more = a.v - 1 - base;           // and so do rows
  const uint32_t w_off = static_cast<uint32_t>((c < more ? c : more) * a.ldw);
  const auto w_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<int8_t*>(a.w) + base * a.ldw, 0, static_cast<int>(kPast), 0x00020000);
  i32x4_t q_rsrc;
  {
    const uint64_t p = reinterpret_cast<uint64_t>(a.q);
    q_rsrc = i32x4_t{static_cast<int>(p & 0xffffffffu), static_cast<int>(p >> 32),
                     static_cast<int>(kPast), 0x00020000};
  }
  // Blocks `wave`, + 8, ... of the tokens' step (where there are four, two waves
  // load each: no branch, and every wave has the same loads in flight): lane p fills
  // token 4 b + p / 16, physical chunk p % 16.
  constexpr int kMine = (kBlocks + kFewWavesWg - 1) / kFewWavesWg;
  static_assert(kBlocks == kMine * kFewWavesWg || kBlocks == kFewWavesWg / 2, "whole rounds");
  const int block0 = wave % (kBlocks < kFewWavesWg ? kBlocks : kFewWavesWg);
  uint32_t q_off[kMine];
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    const int64_t t = 4 * (block0 + kFewWavesWg * j) + (lane >> 4);
    const int chunk = (lane & 15) ^ static_cast<int>(t & 15);
    q_off[j] = static_cast<uint32_t>((t < a.n ? t : a.n - 1) * a.kp) + 16 * chunk;
  }
  const int steps = static_cast<int>(a.kp / kStepK);
  const int last_chunk = static_cast<int>(a.w_chunks) - 1;

  struct Weights {
    i32x4v w[kSlices];
  };
  // Workgroups begin at different steps: rows 4096 bytes apart, all read at the same
  // columns, would keep to a few of the memory's channels.
  const int first = static_cast<int>(blockIdx.x % static_cast<unsigned>(steps));
  auto load = [&](Weights& s, int buf, int i) {
    int k = first + i;
    if (k >= steps) k -= steps;
    const uint32_t past = i < steps ? 0u : kPast;
#pragma unroll
    for (int j = 0; j < kMine; ++j)
      raw_buffer_load_lds(q_rsrc,
                          (lds_void_t*)(lds[buf] + (block0 + kFewWavesWg * j) * 1024), 16,
                          static_cast<int>(q_off[j] + k * kStepK + past), 0, 0, 0);
#pragma unroll
    for (int h = 0; h < kSlices; ++h) {
      // Chunks past a row's last read that one: the tokens hold zeros there.
      int chunk = 16 * k + 4 * h + g;
      chunk = chunk < last_chunk ? chunk : last_chunk;
      s.w[h] = __builtin_bit_cast(
          i32x4v, __builtin_amdgcn_raw_buffer_load_b128(w_rsrc, w_off + 16 * chunk + past, 0, 0));
    }
  };
  i32x4v acc[kTokFrags];
#pragma unroll
  for (int t = 0; t < kTokFrags; ++t) acc[t] = i32x4v{0, 0, 0, 0};
  auto mul = [&](const Weights& s, int buf) {
    const char* st = lds[buf] + c * kStepK;
#pragma unroll
    for (int h = 0; h < kSlices; ++h)
#pragma unroll
      for (int t = 0; t < kTokFrags; ++t) {
        const i32x4v q = *reinterpret_cast<const i32x4v*>(st + t * 16 * kStepK +
                                                          (((4 * h + g) ^ c) << 4));
        acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.w[h], q, acc[t], 0, 0, 0);
      }
  };
  // Step k: its loads have landed (all but the newer steps' are waited for), in
  // every wave, and every wave is done with the step whose buffer step k +
  // kDepth - 1 takes.
  constexpr int kNewer = (kDepth - 2) * (kSlices + kMine);
  auto arrive = [&] {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kNewer) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  Weights s[kDepth];
#pragma unroll
  for (int d = 0; d + 1 < kDepth; ++d) load(s[d], d, d);
  int k = 0;
  for (; k + kDepth <= steps; k += kDepth) {  // no branch inside: the loads stay counted
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      arrive();
      constexpr int kLast = kDepth - 1;
      load(s[(d + kLast) % kDepth], (d + kLast) % kDepth, k + d + kLast);
      __builtin_amdgcn_sched_barrier(0);
      mul(s[d], d);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int d = 0; d + 1 < kDepth; ++d)
    if (k + d < steps) mul(s[d], d);
  // Four consecutive logits a lane.
  O* out = static_cast<O*>(a.out);
  const int64_t v = v0 + 4 * g;
  if (v >= a.v) return;
  float sw[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) sw[e] = a.sw[v + e < a.v ? v + e : v];
#pragma unroll
  for (int t = 0; t < kTokFrags; ++t) {
    const int64_t tok = 16 * t + c;
    if (tok >= a.n) continue;
    const float sx = a.sx[tok];
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = static_cast<float>(acc[t][e]) * sx * sw[e];
    O* dst = out + tok * a.ldo + v;
    if (v + 4 <= a.v) {  // at the element's alignment
      if constexpr (std::is_same<O, float>::value) {
        typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
        *reinterpret_cast<f32x4_any*>(dst) = f32x4_any{y[0], y[1], y[2], y[3]};
      } else {
        typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
        *reinterpret_cast<u32x2_any*>(dst) =
            u32x2_any{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
      }
    } else {
      for (int e = 0; e < 4 && v + e < a.v; ++e) Elem<O>::store1(dst + e, y[e]);
    }
  }
}

inline bool dtype_ok(int d) { return d == NMCE_F32 || d == NMCE_BF16; }
inline int64_t size_of(int d) { return d == NMCE_F32 ? 4 : 2; }

template <typename T, int kRow, bool kHeld>
int launch_quantize_as(const void* x, int64_t n, int64_t k, int64_t ldx, int8_t* q, int64_t ldq,
                       float* scale, hipStream_t s) {
  constexpr int kBlock = kRow < 256 ? 256 : kRow, kRows = kBlock / kRow;
  const int64_t most = 1 << 21, want = (n + kRows - 1) / kRows;
  // A vector's bytes leave in one store where every row starts on such a boundary.
  constexpr int kVec = Elem<T>::kPerVec;
  const bool whole = reinterpret_cast<uintptr_t>(q) % kVec == 0 && ldq % kVec == 0;
  hipLaunchKernelGGL((quantize_rows_kernel<T, kRow, kHeld>),
                     dim3(static_cast<unsigned>(want < most ? want : most)), dim3(kBlock), 0, s,
                     static_cast<const T*>(x), n, k, ldx, q, ldq, scale, whole);
  return launch_status();
}

template <typename T>
int launch_quantize_of(const void* x, int64_t n, int64_t k, int64_t ldx, int8_t* q, int64_t ldq,
                       float* scale, hipStream_t s) {
  // A wave a row, or for short rows a part of one, where its registers hold the row
  // and there are rows for two waves on every SIMD; else four, sixteen, or sixteen
  // that read twice. The fewest threads that hold a row win: a wave's others would
  // idle. 2^18 rows of 256 bf16 take 34 us with 8 threads a row, 44 with 16 and 171
  // with 64; 2^17 of 512 33 with 16 and 81 with 64; 65536 of 1024 34 with 32 and 44
  // with 64.
  if (k <= 64 * kQuantEach && n >= 2048) {
    if (k <= 8 * kQuantEach)
      return launch_quantize_as<T, 8, true>(x, n, k, ldx, q, ldq, scale, s);
    if (k <= 16 * kQuantEach)
      return launch_quantize_as<T, 16, true>(x, n, k, ldx, q, ldq, scale, s);
    if (k <= 32 * kQuantEach)
      return launch_quantize_as<T, 32, true>(x, n, k, ldx, q, ldq, scale, s);
    return launch_quantize_as<T, 64, true>(x, n, k, ldx, q, ldq, scale, s);
  }
  if (k <= 256 * kQuantEach)
    return launch_quantize_as<T, 256, true>(x, n, k, ldx, q, ldq, scale, s);
  if (k <= 1024 * kQuantEach)
    return launch_quantize_as<T, 1024, true>(x, n, k, ldx, q, ldq, scale, s);
  return launch_quantize_as<T, 1024, false>(x, n, k, ldx, q, ldq, scale, s);
}

int launch_quantize(const void* x, int dtype, int64_t n, int64_t k, int64_t ldx, int8_t* q,
                    int64_t ldq, float* scale, hipStream_t s) {
  return dtype == NMCE_F32 ? launch_quantize_of<float>(x, n, k, ldx, q, ldq, scale, s)
                           : launch_quantize_of<uint16_t>(x, n, k, ldx, q, ldq, scale, s);
}

template <typename O, bool kVec>
int launch_tiles(const LinearArgs& a, hipStream_t s) {
  static std::atomic<bool> lds_set{false};
  if (const int rc = allow_lds(reinterpret_cast<const void*>(&int8_linear_kernel<O, kVec>),
                               kLdsBytes, lds_set))
    return rc;
  // A launch's workgroups times their threads fit 32 bits: large batches go in parts.
  const int64_t tiles_n = (a.v + kBN - 1) / kBN;
  const int64_t most = ((int64_t{1} << 23) / tiles_n > 0 ? (int64_t{1} << 23) / tiles_n : 1) * kBM;
  for (int64_t r = 0; r < a.n; r += most) {
    LinearArgs p = a;
    p.q += r * a.kp;
    p.sx += r;
    p.out = static_cast<O*>(a.out) + r * a.ldo;
    p.n = a.n - r < most ? a.n - r : most;
    hipLaunchKernelGGL((int8_linear_kernel<O, kVec>),
                       dim3(static_cast<unsigned>((p.n + kBM - 1) / kBM * tiles_n)),
                       dim3(kThreads), kLdsBytes, s, p);
    if (const int st = launch_status()) return st;
  }
  return NMCE_OK;
}

// Three steps of up to 32 tokens at a time; of more, whose steps take more LDS, two
// (three leave fewer workgroups a compute unit: 64 tokens the same, 128 6% slower).
template <typename O, int kTokFrags>
int launch_few(const LinearArgs& a, hipStream_t s) {
  constexpr int kDepth = kTokFrags <= 2 ? 3 : 2;
  constexpr int kRows = 16 * kFewWavesWg;
  const dim3 grid(static_cast<unsigned>((a.v + kRows - 1) / kRows));
  hipLaunchKernelGGL((int8_few_kernel<O, kTokFrags, kDepth>), grid, dim3(64 * kFewWavesWg), 0, s,
                     a);
  return launch_status();
}

template <typename O>
int launch_linear(const LinearArgs& a, bool vec, hipStream_t s) {
  // (A launch's threads, 512 for 128 vocabulary rows, have to fit 32 bits.)
  if (a.n <= kFewTokens && a.v <= (int64_t{1} << 29)) {
    if (a.n <= 16) return launch_few<O, 1>(a, s);
    if (a.n <= 32) return launch_few<O, 2>(a, s);
    if (a.n <= 64) return launch_few<O, 4>(a, s);
    return launch_few<O, 8>(a, s);
  }
  if constexpr (std::is_same<O, float>::value)
    if (!vec) return launch_tiles<O, false>(a, s);
  return launch_tiles<O, true>(a, s);
}

int64_t linear_workspace(int64_t n, int64_t k) {
  return align256(n * round_up(k, kPadK)) + align256(n * 4);
}

}  // namespace
}  // namespace nmce

using namespace nmce;

extern "C" {

int nmce_quantize_rows(const void* x, int dtype, int64_t n_rows, int64_t columns, int64_t ldx,
                       int8_t* q, int64_t ldq, float* scale, void* stream) {
  if (!dtype_ok(dtype)) return NMCE_EINVAL_DTYPE;
  if (n_rows < 0 || columns < 1 || ldx < columns || ldq < columns) return NMCE_EINVAL_SHAPE;
  if (n_rows == 0) return NMCE_OK;
  if (!x || !q || !scale) return NMCE_EINVAL_PTR;
  if (reinterpret_cast<uintptr_t>(x) % size_of(dtype) || reinterpret_cast<uintptr_t>(scale) % 4)
    return NMCE_EINVAL_ALIGN;
  return launch_quantize(x, dtype, n_rows, columns, ldx, q, ldq, scale,
                         static_cast<hipStream_t>(stream));
}

int64_t nmce_int8_linear_workspace_bytes(int64_t n_rows, int64_t columns) {
  if (n_rows < 0 || columns < 1 || columns > kMaxK) return -1;
  return linear_workspace(n_rows, columns);
}

int nmce_int8_linear(const void* x, int dtype, int64_t n_rows, int64_t columns, int64_t ldx,
                     const int8_t* weight, int64_t vocab_local, int64_t ldw, const float* w_scale,
                     void* out, int out_dtype, int64_t ldo, void* workspace,
                     int64_t workspace_bytes, void* stream) {
  if (!dtype_ok(dtype) || !dtype_ok(out_dtype)) return NMCE_EINVAL_DTYPE;
  const int64_t most = (int64_t{1} << 31) - 1;
  // One 256-row tile's bytes are addressed with 32 bits.
  if (n_rows < 0 || n_rows > most || columns < 1 || columns > kMaxK || ldx < columns ||
      vocab_local < 1 || vocab_local > most || ldw < columns || ldw >= (int64_t{1} << 23) ||
      ldo < vocab_local)
    return NMCE_EINVAL_SHAPE;
  if (n_rows == 0) return NMCE_OK;
  if (!x || !weight || !w_scale || !out) return NMCE_EINVAL_PTR;
  if (reinterpret_cast<uintptr_t>(x) % size_of(dtype) || !aligned16(weight) || ldw % 16 ||
      reinterpret_cast<uintptr_t>(w_scale) % 4 ||
      reinterpret_cast<uintptr_t>(out) % size_of(out_dtype))
    return NMCE_EINVAL_ALIGN;
  char* ws = static_cast<char*>(workspace);
  if (!ws || !aligned16(ws) || workspace_bytes < linear_workspace(n_rows, columns))
    return NMCE_EINVAL_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);

  LinearArgs a{};
  a.kp = round_up(columns, kPadK);
  int8_t* q = reinterpret_cast<int8_t*>(ws);
  float* sx = reinterpret_cast<float*>(ws + align256(n_rows * a.kp));
  if (const int st = launch_quantize(x, dtype, n_rows, columns, ldx, q, a.kp, sx, s)) return st;
  a.q = q;
  a.sx = sx;
  a.w = weight;
  a.sw = w_scale;
  a.out = out;
  a.n = n_rows;
  a.v = vocab_local;
  a.ldw = ldw;
  a.ldo = ldo;
  a.w_chunks = (columns + 15) / 16;
  // store_f32_tile addresses a pass's rows with 32 bits.
  if (out_dtype == NMCE_BF16) return launch_linear<uint16_t>(a, true, s);
  return launch_linear<float>(a, ldo * 4 * 512 < (int64_t{1} << 32), s);
}

}  // extern "C"
