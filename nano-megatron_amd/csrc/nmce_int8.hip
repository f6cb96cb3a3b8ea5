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

#include <type_traits>

#include "nmce.h"
#include "nmce_device.h"
#include "nmce_gemm.h"

namespace nmce {
namespace {

constexpr int64_t kMaxK = 131072;
constexpr int kQuantBlock = 256;
constexpr int kPadK = 128;  // bytes of a stage: tokens' rows are padded to it with zeros

// x * (127 / top) to the nearest integer, halves to even, as the exact quotient
// 127 x / top rounds. The fp32 product is off by less than 2e-5 (three roundings of
// at most 127): only where it lies that near to a half (or 127 / top is not
// finite) the quotient is formed, in fp64, where 127 x is exact and the quotient
// of a 31-bit and a 24-bit number is a half only if it is one exactly.
__device__ __forceinline__ int quantised(float x, float top, float inv) {
  const float t = x * inv;
  const float r = rintf(t);
  if (fabsf(fabsf(t - r) - 0.5f) >= 1e-4f) return static_cast<int>(r);
  return static_cast<int>(rint(127.0 * static_cast<double>(x) / static_cast<double>(top)));
}

// A workgroup quantises one row: its largest magnitude, then the elements, read
// again. Magnitudes are compared as the integers of their bits, which put
// infinities and NaNs above every number: such a row gets the scale NaN and
// zeros, so its products are NaN. A row of zeros gets the scale 0.
template <typename T, bool kVec>
__global__ __launch_bounds__(kQuantBlock) void quantize_rows_kernel(
    const T* __restrict__ x, int64_t n, int64_t k, int64_t ldx, int8_t* __restrict__ q,
    int64_t ldq, float* __restrict__ scale) {
  __shared__ uint32_t wave_top[kQuantBlock / 64];
  for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
    const T* row = x + r * ldx;
    uint32_t top = 0;
    for (int64_t c = threadIdx.x; c < k; c += kQuantBlock) {
      const uint32_t b = __float_as_uint(Elem<T>::load1(row + c)) & 0x7fffffffu;
      top = b > top ? b : top;
    }
    for (int s = 32; s > 0; s >>= 1) {
      const uint32_t o = __shfl_xor(top, s);
      top = o > top ? o : top;
    }
    if ((threadIdx.x & 63) == 0) wave_top[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int w = 0; w < kQuantBlock / 64; ++w) top = wave_top[w] > top ? wave_top[w] : top;
    __syncthreads();
    const bool finite = top < 0x7f800000u;
    const float most = __uint_as_float(top);
    if (threadIdx.x == 0)
      scale[r] = finite ? static_cast<float>(static_cast<double>(most) / 127.0)
                        : __uint_as_float(0x7fc00000u);
    const bool any = finite && top != 0;
    const float inv = 127.0f / most;
    for (int64_t c = threadIdx.x; c < ldq; c += kQuantBlock)
      q[r * ldq + c] = static_cast<int8_t>(
          any && c < k ? quantised(Elem<T>::load1(row + c), most, inv) : 0);
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

// A 256 x 256 tile of the logits (rows: tokens).
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
  if constexpr (std::is_same<O, float>::value)
    store_f32_tile<1, kVec>(acc, lds, static_cast<float*>(a.out), nullptr, a.ldo, a.n, a.v, m0,
                            n0);
  else
    store_bf16_tile(acc, lds, static_cast<uint16_t*>(a.out), a.ldo, a.n, a.v, m0, n0);
}

inline bool dtype_ok(int d) { return d == NMCE_F32 || d == NMCE_BF16; }
inline int64_t size_of(int d) { return d == NMCE_F32 ? 4 : 2; }

int launch_quantize(const void* x, int dtype, int64_t n, int64_t k, int64_t ldx, int8_t* q,
                    int64_t ldq, float* scale, hipStream_t s) {
  const int64_t most = 1 << 20;
  const dim3 grid(static_cast<unsigned>(n < most ? n : most)), block(kQuantBlock);
  if (dtype == NMCE_F32)
    hipLaunchKernelGGL((quantize_rows_kernel<float, false>), grid, block, 0, s,
                       static_cast<const float*>(x), n, k, ldx, q, ldq, scale);
  else
    hipLaunchKernelGGL((quantize_rows_kernel<uint16_t, false>), grid, block, 0, s,
                       static_cast<const uint16_t*>(x), n, k, ldx, q, ldq, scale);
  return launch_status();
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
  if (out_dtype == NMCE_BF16) return launch_tiles<uint16_t, true>(a, s);
  // store_f32_tile's conditions for 16-byte stores.
  const bool vec = vocab_local % 4 == 0 && ldo % 4 == 0 && aligned16(out) &&
                   ldo * 4 * 512 < (int64_t{1} << 32);
  return vec ? launch_tiles<float, true>(a, s) : launch_tiles<float, false>(a, s);
}

}  // extern "C"
