// The GEMM core of libnmce's products on gfx950, C[m, n] = sum_k A[m, k] *
// B[n, k], and the epilogues that store a product.
//
// Main loop: a 256x256 output tile per 256-lane workgroup (four waves, 2x2,
// one per SIMD, each 128x128 = 64 accumulators of 16x16 held in AGPRs), K in
// steps of 64. Each wave reads its next fragments from LDS under the MFMAs of
// the current ones (two register sets), and the reads and the next stages'
// loads have fixed places between the MFMAs. Operand tiles move HBM/L2 -> LDS
// with 16-byte direct-to-LDS loads (MUBUF buffer_load_dwordx4 ... lds, no VGPR
// staging), A triple- and B double-buffered. A K-contiguous operand sits in
// rows of 128 bytes with the 16-byte chunks XOR-swizzled by ((row >> 1) & 7).
// gfx950's LDS has 64 banks, so a ds_read_b128 serves 16 lanes (16 consecutive
// rows of a fragment) per cycle; this swizzle puts those 16 rows on 16 distinct
// 16-byte bank groups (row parity picks the half of the banks, the swizzled
// chunk the group). An MN-contiguous operand sits in 64 k-rows of 512 bytes
// and its fragments come from gfx950's transposing LDS read,
// ds_read_b64_tr_b16, with the same fragments, so the two layouts give the
// same bits. Workgroups are mapped to tiles so that each XCD (one L2) owns a
// contiguous band of tiles walked in groups that share operands.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "nmce_device.h"

namespace nmce {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;

constexpr int kBM = 256;          // tile rows (GEMM M)
constexpr int kBN = 256;          // tile columns (GEMM N)
constexpr int kBK = 64;           // K per stage (128 bytes of bf16 per row)
// Four waves, one per SIMD, each 128 x 128 of the tile (2 x 2). Against eight
// waves of 128 x 64 (two per SIMD) a wave reads a third less from LDS per
// product, and that and the smaller MFMA (below) are what a chip at its power
// cap turns into clock: 1190 -> 1525 TFLOP/s on 16384 x 16384 x 8192, 1175 ->
// 1538 on 4096 x 4096 x 65536.
constexpr int kWavesM = 2;
constexpr int kWavesN = 2;
constexpr int kWaves = kWavesM * kWavesN;
constexpr int kThreads = 64 * kWaves;
constexpr int kWaveM = kBM / kWavesM;  // 128
constexpr int kWaveN = kBN / kWavesN;  // 128
constexpr int kF = kWaveM / 16;        // 8 fragments of 16 rows (columns) a side
static_assert(kWaveM == kWaveN, "a wave's tile is square");
constexpr int kStage = kBM * kBK * 2;  // bytes of one operand's stage: 32 KiB
static_assert(kBM == kBN, "the operands' stages have one size");
// A's stages in three buffers, B's in two: all of a compute unit's LDS. A
// stage's A loads are then issued before the barrier that frees B's buffer,
// which spreads a stage's loads over the whole K step (gemm_mainloop).
constexpr int kBufsA = 3;
constexpr int kBufsB = 2;
constexpr int kLdsBytes = (kBufsA + kBufsB) * kStage;  // dynamic LDS: 160 KiB
static_assert(kLdsBytes <= 160 * 1024, "the stages fit a compute unit's LDS");
// 1 KiB LDS blocks per stage and operand, and per wave of them.
constexpr int kBlocks = kStage / 1024;
constexpr int kBlocksPerWave = kBlocks / kWaves;
// Tile rows per raster group inside an XCD band: 4 of 2, 4 and 8 is the
// fastest for the products of many tiles (16384 x 16384 x 8192: 1545 TFLOP/s
// against 1476 with 8; the [16384, 4096] x [128256, 4096] step 39.3 ms against
// 39.6 with 8 and 39.9 with 2) and no slower than 1.5% elsewhere.
constexpr int kGroupM = 4;
constexpr int kXcds = 8;

// A wave's 128 x 128 results: c[i][j] is the 16 x 16 block of rows 16 i and
// columns 16 j; lane l holds column l % 16, rows 4 (l / 16) + e of it, or,
// from a main loop with kRows, row l % 16, columns 4 (l / 16) + e.
struct Acc {
  f32x4_t c[kF][kF];
};

// acc += A B^T of one 16 x 16 block, K = 32, as an instruction that updates
// its accumulator registers in place. With the builtin the compiler gives 64
// accumulators results in other registers than their inputs and moves them
// back (360 moves per K step, 1055-1200 instead of 1440 TFLOP/s). The 16 x 16
// form moves half the accumulator bytes per product that the 32 x 32 x 16 form
// does, with the same sums: 1440 against 1240 TFLOP/s in the same loop.
// The compiler puts no wait states around an instruction that it does not know
// for an MFMA: its fragments come from LDS reads, whose waits it counts, and
// nothing else touches the accumulators within the loop (gemm_mainloop waits
// before the first and after the last; a test looks at the generated code).
__device__ __forceinline__ void mfma_16x16x32(f32x4_t& c, const bf16x8_t& a, const bf16x8_t& b) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

// The same on 8-bit integers, K = 64: its fragments are the same 16 bytes a
// lane (row l % 16, bytes 16 (l / 16) .. + 15 of 64), its accumulators 32-bit
// integers in the same places, and it takes the same 16 cycles. So the whole
// core runs on bytes: an operand of 8-bit elements is one of half as many
// 16-bit ones, and c holds the integers' bits.
__device__ __forceinline__ void mfma_i8_16x16x64(f32x4_t& c, const bf16x8_t& a,
                                                 const bf16x8_t& b) {
  asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

// Tile index for workgroup b. The dispatcher deals workgroups to the 8 XCDs
// round-robin (block b runs on XCD b % 8); give each XCD a contiguous band of
// tile ids, and inside the band walk groups of kGroupM tile rows column by
// column, so the tiles that run together on one L2 share A and B stripes.
__device__ __forceinline__ void tile_coords(int b, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int total = tiles_m * tiles_n;
  const int xcd = b % kXcds;
  const int q = total / kXcds, r = total % kXcds;
  const int tid = xcd * q + (xcd < r ? xcd : r) + b / kXcds;
  const int group = kGroupM * tiles_n;
  const int g = tid / group;
  const int first_m = g * kGroupM;
  const int gm = (tiles_m - first_m) < kGroupM ? (tiles_m - first_m) : kGroupM;
  const int in_g = tid - g * group;
  tm = first_m + in_g % gm;
  tn = in_g / gm;
}

// The loads of one operand's stages (64 k each) into LDS by this wave: 1 KiB
// blocks blk0 .. blk0 + 7, one MUBUF direct-to-LDS load each.
//
// K-contiguous (kMN = false): a block is 8 rows of 128 bytes; lane p writes
// row p / 8, physical chunk p % 8, which holds logical chunk
// (p % 8) ^ ((row >> 1) & 7). The K position goes in the scalar offset, so a
// stage needs no per-lane arithmetic. MN-contiguous: a block is k-rows 2 b and
// 2 b + 1 of 512 bytes; lane p writes row 2 b + p / 32, physical chunk p % 32,
// which holds logical chunk (p % 32) ^ 4 (row & 3) ^ 2 ((row >> 3) & 1). The
// resource's base moves by 64 rows per stage (the offset would pass 32 bits).
//
// The buffer resource has no stride and no range limit (every offset is
// clamped in bounds) and gfx9's data format word.
//
// kTail (K-contiguous): a row's 16-byte chunks may end inside the last stage;
// those past the last are read as the last, and the other operand holds zeros
// there.
template <bool kMN, bool kTail = false>
struct StageLoads {
  i32x4_t rsrc;
  const char* base;
  int64_t row_bytes, krows;
  uint32_t off[kBlocksPerWave];
  int row0, last_chunk, lane, soff;

  __device__ __forceinline__ void set_base(const char* p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    rsrc[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(a & 0xffffffffu));
    rsrc[1] = __builtin_amdgcn_readfirstlane(static_cast<int>(a >> 32));
  }
  __device__ __forceinline__ int krow(int j) const { return row0 + 2 * j; }
  __device__ __forceinline__ int chunk_bytes(int j) const {
    int chunk = (lane & 31) ^ (4 * (krow(j) & 3)) ^ (2 * ((krow(j) >> 3) & 1));
    if (chunk > last_chunk) chunk = last_chunk;
    return chunk * 16;
  }
  // first: the operand's element at the tile's first row (column), k = 0;
  // rows: the operand's rows (columns) from there on; krows_: its k-rows (kMN)
  // or a row's 16-byte chunks (kTail).
  __device__ __forceinline__ void init(const uint16_t* first, int64_t ld, int64_t rows,
                                       int64_t krows_, int wave, int lane_) {
    lane = lane_;
    base = reinterpret_cast<const char*>(first);
    row_bytes = ld * 2;
    krows = krows_;
    soff = 0;
    const int blk0 = wave * kBlocksPerWave;
    if constexpr (kTail) row0 = blk0 * 8 + (lane >> 3);
    if constexpr (kMN) {
      row0 = 2 * blk0 + (lane >> 5);
      const int64_t last = (rows + 7) / 8 - 1;  // >= 0
      last_chunk = static_cast<int>(last < 31 ? last : 31);
#pragma unroll
      for (int j = 0; j < kBlocksPerWave; ++j)
        off[j] = static_cast<uint32_t>(krow(j) * row_bytes + chunk_bytes(j));
    } else {
#pragma unroll
      for (int j = 0; j < kBlocksPerWave; ++j) {
        const int tile_row = (blk0 + j) * 8 + (lane >> 3);
        const int chunk = (lane & 7) ^ ((tile_row >> 1) & 7);
        const int64_t r = tile_row < rows ? tile_row : rows - 1;
        off[j] = static_cast<uint32_t>(r * row_bytes + chunk * 16);
      }
    }
    set_base(base);
    rsrc[2] = -1;
    rsrc[3] = 0x00020000;
  }
  // The number of leading stages whose k-rows all exist.
  __device__ __forceinline__ int full_stages(int stages) const {
    if constexpr (!kMN && !kTail) return stages;
    const int64_t f = krows / (kMN ? kBK : kBK / 8);
    return f < stages ? static_cast<int>(f) : stages;
  }
  // Stage kt (all of its k-rows exist) is the next one to be loaded.
  __device__ __forceinline__ void at(int kt) {
    if constexpr (kMN)
      set_base(base + kt * (kBK * row_bytes));
    else
      soff = __builtin_amdgcn_readfirstlane(kt * (kBK * 2));
  }
  __device__ __forceinline__ void load(char* dst, int j) const {
    raw_buffer_load_lds(rsrc, (lds_void_t*)(dst + j * 1024), 16, static_cast<int>(off[j]), soff, 0,
                        0);
  }
  // A whole stage at once, whose k-rows may end before it does (kMN): those
  // past the last are read as the last.
  __device__ __forceinline__ void stage(char* dst, int kt) {
    const int64_t k0 = static_cast<int64_t>(kt) * kBK;
    if (kMN && k0 + kBK > krows) {
      const int64_t b0 = k0 < krows ? k0 : krows - 1;
      set_base(base + b0 * row_bytes);
#pragma unroll
      for (int j = 0; j < kBlocksPerWave; ++j) {
        int64_t row = k0 + krow(j);
        if (row > krows - 1) row = krows - 1;
        raw_buffer_load_lds(rsrc, (lds_void_t*)(dst + j * 1024), 16,
                            static_cast<int>((row - b0) * row_bytes) + chunk_bytes(j), 0, 0, 0);
      }
      return;
    }
    if constexpr (kTail) {
      if ((kt + 1) * static_cast<int64_t>(kBK / 8) > krows) {
#pragma unroll
        for (int j = 0; j < kBlocksPerWave; ++j) {
          const int chunk = (lane & 7) ^ (((row0 + 8 * j) >> 1) & 7);
          int64_t c = static_cast<int64_t>(kt) * (kBK / 8) + chunk;
          if (c > krows - 1) c = krows - 1;
          raw_buffer_load_lds(rsrc, (lds_void_t*)(dst + j * 1024), 16,
                              static_cast<int>(off[j] + (c - chunk) * 16), 0, 0, 0);
        }
        return;
      }
    }
    at(kt);
#pragma unroll
    for (int j = 0; j < kBlocksPerWave; ++j) load(dst, j);
  }
};

// One operand's fragments of 16 rows (columns) and 32 k from its stage: lane l
// gets row l % 16, k 8 (l / 16) .. + 7. K-contiguous: one ds_read_b128 of the
// row's logical chunk 4 s + l / 16 (sub-step s); 16 consecutive rows of one
// chunk are on distinct 16-byte bank groups. MN-contiguous: two
// ds_read_b64_tr_b16, each giving a lane 4 consecutive k of its column (in a
// group of 16 lanes, lanes 4 r .. 4 r + 3 read the 16 columns of k-row r and
// lane j receives column j of the 4 rows). Lane 16 g + 4 r + u reads k-row
// 8 g + r (+ 4 for the second, + 32 s), columns 4 u .. 4 u + 3 of the
// fragment; the swizzle puts the 8 k-rows that half of the lanes read (rows
// 0-3 and 8-11) on distinct 32 bytes of the 256 that the banks span.
template <bool kMN>
struct Frags {
  int off0, off1;  // K-contiguous: the lane's byte offset in sub-step 0 and 1
  int lane;
  int col0;        // first row (column) of the wave's 128

  __device__ __forceinline__ void init(int first, int lane_) {
    lane = lane_;
    col0 = first;
    const int r = lane & 15, q = lane >> 4;
    off0 = (first + r) * 128 + ((q ^ ((r >> 1) & 7)) << 4);
    off1 = (first + r) * 128 + (((4 + q) ^ ((r >> 1) & 7)) << 4);
  }
  // K-contiguous: the whole fragment f of sub-step s.
  __device__ __forceinline__ bf16x8_t read(const char* st, int s, int f) const {
    return *reinterpret_cast<const bf16x8_t*>(st + (s ? off1 : off0) + f * 16 * 128);
  }
  // MN-contiguous: its half h (k 4 h .. 4 h + 3 of the lane's eight).
  __device__ __forceinline__ s16x4_t read_half(const char* st, int s, int f, int h) const {
    const int g = lane >> 4, r = (lane >> 2) & 3, u = lane & 3;
    // k-rows 8 g + r and 8 g + 4 + r share the swizzle (row & 3 = r,
    // (row >> 3) & 1 = g & 1); 32 s does not change it either.
    const int chunk = (((col0 + 16 * f) >> 3) + (u >> 1)) ^ (4 * r) ^ (2 * (g & 1));
    const char* p = st + (8 * g + r) * 512 + chunk * 16 + 8 * (u & 1) + s * (32 * 512);
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4_t*)(p + h * (4 * 512)));
  }
  static __device__ __forceinline__ bf16x8_t join(const s16x4_t& lo, const s16x4_t& hi) {
    typedef short s16x8_t __attribute__((ext_vector_type(8)));
    const s16x8_t v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8_t, v);
  }
};

// The main loop: acc = A[m0:m0+256, 0:K] * B[n0:n0+256, 0:K]^T, each operand
// K-contiguous (A[m, k] at A + m * lda + k; kAMN = false) or MN-contiguous
// (A[m, k] at A + k * lda + m; kAMN = true), and B likewise.
// K-contiguous operands: rows >= M (N) are read from the last valid row; their
// results are masked by the epilogues. MN-contiguous operands: columns are
// read in 8-element chunks up to the one holding column M - 1 (N - 1), so the
// rows must be allocated to a multiple of 8 elements past it; later chunks
// repeat that one. An MN-contiguous operand may hold fewer k-rows than K
// (ka_rows, kb_rows): k-rows past its last are read as its last, so the other
// operand must hold zeros there. Requires K % 64 == 0, lda and ldb multiples of 8 elements,
// 16-byte aligned A and B, and 256 * ld * 2 < 2^32 bytes (K-contiguous) or
// 64 * ld * 2 < 2^32 bytes (MN-contiguous).
//
// A K step is two sub-steps of 32 k, 64 MFMAs each. One wave per SIMD has
// nothing else to hide a wait, so the stream is fixed: after every third MFMA
// one fragment of the next sub-step is read from LDS (the 16 reads are done
// by the 48th of 64 MFMAs, so none is waited for), and after every sixth one
// of the stage's 16 loads is issued (issued together they fill the address
// unit's queue and the wave stalls: 1370 against 1450 TFLOP/s with one every
// second MFMA, 1525 spread over both sub-steps, on 16384 x 16384 x 8192).
// Stage kt + 2's A goes into the buffer that stage kt - 1 had, during the first
// sub-step of kt; its B into stage kt's buffer, after the barrier at which every
// wave has read the last of stage kt. That barrier waits for all but the wave's
// newest eight loads (stage kt + 2's A).
//
// kRows hands the MFMA its operands the other way round, which gives the lane
// four columns of one row instead of four rows of one column (the same sums):
// what an epilogue wants that stores rows.
//
// kI8: 8-bit integers, two to a 16-bit element (lda, ldb and K count pairs);
// ka_rows and kb_rows are then the 16-byte chunks that each operand's rows hold.
template <bool kAMN, bool kBMN, bool kRows = false, bool kI8 = false>
__device__ __forceinline__ void gemm_mainloop(const uint16_t* __restrict__ A, int64_t lda,
                                              int64_t M, const uint16_t* __restrict__ B,
                                              int64_t ldb, int64_t N, int64_t K, int64_t m0,
                                              int64_t n0, char* lds, Acc& acc,
                                              int64_t ka_rows = 0, int64_t kb_rows = 0) {
  const int lane = threadIdx.x & 63;
  // The wave index is uniform across the wave; say so, so that the load
  // bases and LDS destinations below live in scalar registers.
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / kWavesN, wn = wave % kWavesN;

  StageLoads<kAMN, kI8> la;
  StageLoads<kBMN, kI8> lb;
  la.init(kAMN ? A + m0 : A + m0 * lda, lda, M - m0, ka_rows, wave, lane);
  lb.init(kBMN ? B + n0 : B + n0 * ldb, ldb, N - n0, kb_rows, wave, lane);
  Frags<kAMN> fa;
  Frags<kBMN> fb;
  fa.init(wm * kWaveM, lane);
  fb.init(wn * kWaveN, lane);

  char* const lds_b = lds + kBufsA * kStage;
  const int lds_w = wave * (kBlocksPerWave * 1024);
  const int kt_n = static_cast<int>(K / kBK);

  la.stage(lds + lds_w, 0);
  lb.stage(lds_b + lds_w, 0);
  if (kt_n > 1) {
    la.stage(lds + kStage + lds_w, 1);
    lb.stage(lds_b + kStage + lds_w, 1);
  }
#pragma unroll
  for (int i = 0; i < kF; ++i)
#pragma unroll
    for (int j = 0; j < kF; ++j) acc.c[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  // The compiler does not know that mfma_16x16x32 reads them as an MFMA does:
  // the zeros are written, and have settled, before the first one.
#pragma unroll
  for (int i = 0; i < kF; ++i)
#pragma unroll
    for (int j = 0; j < kF; ++j) asm volatile("" : "+a"(acc.c[i][j]));
  asm volatile("s_nop 7" ::: "memory");
  // Stage 0 is what the first reads need; the compiler puts a wait for nearly
  // all loads in flight before the barrier of its own accord, stage 1's among
  // them.
  if (kt_n > 1)
    asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
  else
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();

  struct Set {
    bf16x8_t a[kF], b[kF];
  };
  // Fragment q of a sub-step in the order the MFMAs first use them, b0 a0 b1
  // a1 ...: part 1 completes it, part 0 reads a transposed one's first half.
  s16x4_t half;
  auto read = [&](const char* pa, const char* pb, int s, Set& f, int q, int part) {
    if (q & 1) {
      if constexpr (!kAMN) {
        if (part == 1) f.a[q >> 1] = fa.read(pa, s, q >> 1);
      } else if (part == 0) {
        half = fa.read_half(pa, s, q >> 1, 0);
      } else {
        f.a[q >> 1] = fa.join(half, fa.read_half(pa, s, q >> 1, 1));
      }
    } else {
      if constexpr (!kBMN) {
        if (part == 1) f.b[q >> 1] = fb.read(pb, s, q >> 1);
      } else if (part == 0) {
        half = fb.read_half(pb, s, q >> 1, 0);
      } else {
        f.b[q >> 1] = fb.join(half, fb.read_half(pb, s, q >> 1, 1));
      }
    }
  };
  // One sub-step: the 64 MFMAs of `cur`, the 16 fragment reads of the next
  // sub-step after every third of them (a transposed fragment's two halves
  // after the second and the third), and kLoads loads, six MFMAs apart, after
  // MFMAs that no read follows: an MFMA's 16 cycles hide about three other
  // instructions.
  constexpr int kLoadGap = 6;
  auto mma = [&](int i, int j, const Set& f) {
    if constexpr (kI8) {
      static_assert(kRows || !kI8, "8-bit products are stored");
      mfma_i8_16x16x64(acc.c[i][j], f.b[j], f.a[i]);
    } else if constexpr (kRows) {
      mfma_16x16x32(acc.c[i][j], f.b[j], f.a[i]);
    } else {
      mfma_16x16x32(acc.c[i][j], f.a[i], f.b[j]);
    }
  };
  auto step = [&](const char* pa, const char* pb, int s, Set& next, const Set& cur, auto loads,
                  auto&& load) {
    constexpr int kLoads = decltype(loads)::value;
#pragma unroll
    for (int x = 0; x < kF * kF; ++x) {
      const int i = x / kF, j = (i & 1) ? kF - 1 - x % kF : x % kF;
      mma(i, j, cur);
      if (x % 3 != 0 && x / 3 < 2 * kF) read(pa, pb, s, next, x / 3, x % 3 - 1);
      if (x % kLoadGap == 0 && x / kLoadGap < kLoads) load(x / kLoadGap);
      if (kAMN || kBMN || x % 3 == 2) __builtin_amdgcn_sched_barrier(0);
    }
  };
  using NoLoads = std::integral_constant<int, 0>;
  using Loads = std::integral_constant<int, kBlocksPerWave>;
  auto none = [](int) {};

  Set f0, f1;
#pragma unroll
  for (int q = 0; q < 2 * kF; ++q) {
    read(lds, lds_b, 0, f0, q, 0);
    read(lds, lds_b, 0, f0, q, 1);
  }
  int a_cur = 0;               // byte offset of stage kt's A buffer
  auto next_a = [](int o) { return o == (kBufsA - 1) * kStage ? 0 : o + kStage; };
  auto prev_a = [](int o) { return o == 0 ? (kBufsA - 1) * kStage : o - kStage; };
  // Stages [0, full) have all their k-rows: their loads run inside the
  // sub-steps. The last one or two steps load with clamped rows, or nothing.
  const int full_a = la.full_stages(kt_n), full_b = lb.full_stages(kt_n);
  const int full = full_a < full_b ? full_a : full_b;
  int kt = 0;
  for (; kt + 2 < full; ++kt) {
    const int a_nxt = next_a(a_cur);
    const int b_cur = (kt & 1) * kStage;
    char* da = lds + prev_a(a_cur) + lds_w;
    la.at(kt + 2);
    step(lds + a_cur, lds_b + b_cur, 1, f1, f0, Loads{}, [&](int l) { la.load(da, l); });
    asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    char* db = lds_b + b_cur + lds_w;
    lb.at(kt + 2);
    step(lds + a_nxt, lds_b + (kStage - b_cur), 0, f0, f1, Loads{},
         [&](int l) { lb.load(db, l); });
    a_cur = a_nxt;
  }
  static_assert(kBlocksPerWave == 8, "the loop's wait leaves one stage's A loads in flight");
  for (; kt + 1 < kt_n; ++kt) {
    const int a_nxt = next_a(a_cur);
    const int b_cur = (kt & 1) * kStage;
    if (kt + 2 < kt_n) la.stage(lds + prev_a(a_cur) + lds_w, kt + 2);
    step(lds + a_cur, lds_b + b_cur, 1, f1, f0, NoLoads{}, none);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (kt + 2 < kt_n) lb.stage(lds_b + b_cur + lds_w, kt + 2);
    step(lds + a_nxt, lds_b + (kStage - b_cur), 0, f0, f1, NoLoads{}, none);
    a_cur = a_nxt;
  }
  step(lds + a_cur, lds_b + (kt & 1) * kStage, 1, f1, f0, NoLoads{}, none);
#pragma unroll
  for (int x = 0; x < kF * kF; ++x) mma(x / kF, x % kF, f1);
  // The compiler does not know the MFMAs' latency: let the last ones finish
  // before anything reads the accumulators.
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int i = 0; i < kF; ++i)
#pragma unroll
    for (int j = 0; j < kF; ++j) asm volatile("" : "+a"(acc.c[i][j]));
}

// Row (within the wave's 128 rows) of accumulator row block i, element e, for
// a lane in 16-lane group g: the 16x16 result gives lane l column l % 16 and
// rows 4 (l / 16) + e.
__device__ __forceinline__ int acc_row(int i, int e, int g) { return 16 * i + 4 * g + e; }

// The stored products' epilogues take the results row by row (kRows): lane l
// holds, of each 16x16 block, row l % 16 and columns 4 g .. 4 g + 3 (g = l /
// 16), and stages them through the freed LDS, so that whole row segments of
// 512 bytes (bf16) or 1 KiB (fp32) leave. Stored straight from the registers
// they are segments of 64 bytes: 1358 against 1415 TFLOP/s with fp32 out on
// 128256 x 4096 x 4096, 1457 against 1485 with bf16.
//
// The fp32 epilogues (modes 1-3 of gemm_store_kernel). The 256x256 fp32 tile
// goes through the freed LDS in two passes of 128 rows: pass q takes row
// blocks i = 4q .. 4q + 3 of every wave, i.e. tile rows 64 q .. 64 q + 63
// and 128 + 64 q .. 128 + 64 q + 63, so each pass reads its own half of the
// accumulator registers. Staged row r (1 KiB) is tile row
// 128 (r >> 6) + 64 q + (r & 63); its 16-byte chunk c sits at c ^ (r & 15),
// which puts the 16 rows that 16 lanes write on distinct 16-byte bank groups
// (the lane's four columns of a block are one chunk). Every thread then moves
// 32 chunks:
// staged row 4 p + wave, chunk lane, so a wave's access is one 1 KiB row
// segment of Cf (or 512 bytes of C).
// kVec (N % 4 == 0, ldc % 4 == 0, Cf 16-byte and C 8-byte aligned, 512 rows
// within 32-bit offsets): buffer resources on the wave's first row, the
// lane's column in the one offset register and the row step in the scalar
// offset of the loads (the 16-byte stores take it in the per-lane offset:
// buffer_store_b128). The hardware range check covers the per-lane offset
// only, so rows past M (passes p >= np, uniform) are skipped explicitly, and
// a lane whose columns lie past N gets the offset 2^31, more than a resource's
// size and no row step takes it past 32 bits: its accesses are out of range (no
// memory access, a load reads 0, a store is dropped) whether or not the row
// step takes part in the check. (As a product of the row stride it made the
// compiler carry the stride in a lane register and loop over its values at
// every load.) Every access left is inside the matrix. In modes 2 and 3 the 32 loads of Cf are
// issued before the pass is staged, so that their latency runs under the
// staging and 128 KiB are in flight. Cf is streamed (non-temporal) both ways.
// Without kVec the pass leaves element by element.
// kFull: all of the tile's rows exist, nothing is tested. Behind a branch the
// compiler cannot count what is in flight and waits for everything, which with
// each row's load issued behind an earlier row's store was a memory round trip
// a row. Accumulating launches, us: K = 512 on [16348, 2368] 138 -> 95, on
// [128256, 4096] 1383 -> 924; K = 4096 on [128256, 4096] 3531 -> 3255 (mode 2),
// 3469 -> 3121 (mode 3). With the loads in flight, reading the tile's lines
// ahead under the last K steps only costs: 3348 and 3197.
//   kMode 1: Cf = acc;  kMode 2: Cf += acc;  kMode 3: C = bf16(Cf + acc)
template <int kMode, bool kVec, bool kFull>
__device__ __forceinline__ void store_f32_pass(const Acc& acc, int q, char* lds,
                                               float* __restrict__ Cf, uint16_t* __restrict__ C,
                                               int64_t ldc, int64_t M, int64_t N, int64_t m0,
                                               int64_t n0) {
  static_assert(kMode >= 1 && kMode <= 3, "fp32 epilogue modes");
  static_assert(kBN == 256 && kWavesM == 2 && kF == 8 && 128 * kBN * 4 <= kLdsBytes,
                "two passes of 128 rows fit the stages");
  constexpr int kRowsPerPass = kThreads / 64;  // 4
  constexpr int kPasses = 128 / kRowsPerPass;  // 32
  constexpr int kNt = 2;                       // cache policy: non-temporal
  constexpr uint32_t kPast = 1u << 31;         // a lane past N: beyond every resource here
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / kWavesN, wn = wave % kWavesN;
  const int g = lane >> 4;
  float* S = reinterpret_cast<float*>(lds);
  const bool col_ok = n0 + 4 * lane < N;
  // Tile rows of staged rows 4 p + wave, relative to the pass's first row.
  auto row_off = [](int p) { return 4 * p + 64 * (p >> 4); };
  const int64_t row0 = m0 + 64 * q + wave;  // tile row of staged row `wave`
  // valid passes: a prefix, rows increase with p
  int np = kPasses;
  if constexpr (!kFull) {
    np = 0;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) np += (row0 + row_off(p) < M) ? 1 : 0;
    np = __builtin_amdgcn_readfirstlane(np);
  }
  const int64_t lim = np == 0 ? 0 : (np < kPasses ? row_off(np) : row_off(kPasses - 1) + 1);
  const uint32_t vf = col_ok ? static_cast<uint32_t>(lane) * 16u : kPast;
  float* cf_base = Cf + (np > 0 ? row0 : 0) * ldc + n0;
  u32x4 old[kPasses];
  __amdgpu_buffer_rsrc_t rf;
  if constexpr (kVec) {
    rf = __builtin_amdgcn_make_buffer_rsrc(cf_base, 0, static_cast<int>(lim * ldc * 4), 0x00020000);
    if constexpr (kMode >= 2) {
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        if (kFull || p < np)
          old[p] = __builtin_amdgcn_raw_buffer_load_b128(
              rf, vf, static_cast<uint32_t>(row_off(p) * ldc * 4), kNt);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kF; ++j)
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const int r = wm * 64 + 16 * f + (lane & 15);
      const int c = (wn * (kWaveN / 4) + 4 * j + g) ^ (lane & 15);
      *reinterpret_cast<f32x4_t*>(S + r * kBN + 4 * c) = acc.c[4 * q + f][j];
    }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int r = p * kRowsPerPass + wave;
    const u32x4 sv =
        *reinterpret_cast<const u32x4*>(S + r * kBN + ((lane ^ ((4 * p + wave) & 15)) << 2));
    if constexpr (!kVec) {
      const int64_t row = row0 + row_off(p);
      const float sf[4] = {__uint_as_float(sv.x), __uint_as_float(sv.y), __uint_as_float(sv.z),
                           __uint_as_float(sv.w)};
      for (int j = 0; j < 4; ++j) {
        const int64_t col = n0 + 4 * lane + j;
        if (row >= M || col >= N) continue;
        const int64_t o = row * ldc + col;
        if constexpr (kMode == 1) Cf[o] = sf[j];
        if constexpr (kMode == 2) Cf[o] += sf[j];
        if constexpr (kMode == 3) C[o] = f32_to_bf16(Cf[o] + sf[j]);
      }
    } else {
      if (!kFull && p >= np) continue;
      const uint32_t so = static_cast<uint32_t>(row_off(p) * ldc * 4);
      if constexpr (kMode == 1) {
        buffer_store_b128<kNt>(sv, rf, vf + so);
      } else {
        const u32x4 o = old[p];
        const float v0 = __uint_as_float(sv.x) + __uint_as_float(o.x);
        const float v1 = __uint_as_float(sv.y) + __uint_as_float(o.y);
        const float v2 = __uint_as_float(sv.z) + __uint_as_float(o.z);
        const float v3 = __uint_as_float(sv.w) + __uint_as_float(o.w);
        if constexpr (kMode == 2) {
          buffer_store_b128<kNt>(
              u32x4{__float_as_uint(v0), __float_as_uint(v1), __float_as_uint(v2),
                    __float_as_uint(v3)},
              rf, vf + so);
        } else {
          typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
          const auto rh = __builtin_amdgcn_make_buffer_rsrc(
              C + (np > 0 ? row0 : 0) * ldc + n0, 0, static_cast<int>(lim * ldc * 2), 0x00020000);
          __builtin_amdgcn_raw_buffer_store_b64(
              u32x2{pack_bf16x2(v0, v1), pack_bf16x2(v2, v3)}, rh,
              col_ok ? static_cast<uint32_t>(lane) * 8u : kPast,
              static_cast<uint32_t>(row_off(p) * ldc * 2), 0);
        }
      }
    }
  }
  __syncthreads();  // the next pass reuses S
}

template <int kMode, bool kVec>
__device__ __forceinline__ void store_f32_tile(const Acc& acc, char* lds, float* __restrict__ Cf,
                                               uint16_t* __restrict__ C, int64_t ldc, int64_t M,
                                               int64_t N, int64_t m0, int64_t n0) {
  __syncthreads();  // every wave is done with the operand buffers
  if (kVec && m0 + kBM <= M) {
    store_f32_pass<kMode, kVec, true>(acc, 0, lds, Cf, C, ldc, M, N, m0, n0);
    store_f32_pass<kMode, kVec, true>(acc, 1, lds, Cf, C, ldc, M, N, m0, n0);
  } else {
    store_f32_pass<kMode, kVec, false>(acc, 0, lds, Cf, C, ldc, M, N, m0, n0);
    store_f32_pass<kMode, kVec, false>(acc, 1, lds, Cf, C, ldc, M, N, m0, n0);
  }
}

// bf16 out: rows of 512 bytes whose 16-byte chunk c sits at c ^ (row & 15):
// the 16 rows of a block that 32 lanes write 8 bytes of each are on distinct
// 16-byte bank groups. The stores are non-temporal: the product is read by a
// later kernel, if at all, and its lines would take L2 from the next tiles'
// operands. Against words of two rows, unscrambled on the way out, and cached
// stores: K = 512 875 -> 1030 TFLOP/s, K = 1600 1166 -> 1247, K = 4096 1445 ->
// 1459. Tiles that reach past M or N, and outputs that are not 16-byte
// aligned, test every row and column. kAny: those outputs leave 16 bytes at a time
// all the same, at their element's alignment (rows of an odd width).
template <bool kAny = false>
__device__ __forceinline__ void store_bf16_tile(const Acc& acc, char* lds,
                                                uint16_t* __restrict__ C, int64_t ldc, int64_t M,
                                                int64_t N, int64_t m0, int64_t n0) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wm = wave / kWavesN, wn = wave % kWavesN;
  const int g = lane >> 4, c = lane & 15;
  const bool vec_ok = (ldc & 7) == 0 && (reinterpret_cast<uintptr_t>(C) & 15) == 0;
  __syncthreads();  // every wave is done with the operand buffers
  char* row = lds + (wm * kWaveM + c) * (kBN * 2) + 8 * (g & 1);
#pragma unroll
  for (int j = 0; j < kF; ++j) {
    char* at = row + (((wn * (kWaveN / 8) + 2 * j + (g >> 1)) ^ c) << 4);
#pragma unroll
    for (int i = 0; i < kF; ++i)
      *reinterpret_cast<u32x2*>(at + i * (16 * kBN * 2)) =
          u32x2{pack_bf16x2(acc.c[i][j][0], acc.c[i][j][1]),
                pack_bf16x2(acc.c[i][j][2], acc.c[i][j][3])};
  }
  __syncthreads();
  constexpr int kRowStep = kThreads / (kBN / 8);  // 8 rows of 32 chunks at a time
  constexpr int kIters = kBM / kRowStep;
  const int r0 = static_cast<int>(threadIdx.x) / (kBN / 8);
  const int q = static_cast<int>(threadIdx.x) % (kBN / 8);
  auto staged = [&](int it) {
    const int r = r0 + it * kRowStep;
    return *reinterpret_cast<const u32x4*>(lds + r * (kBN * 2) + ((q ^ (r & 15)) << 4));
  };
  if (vec_ok && m0 + kBM <= M && n0 + kBN <= N) {  // every store in bounds: no tests
    uint16_t* dst = C + (m0 + r0) * ldc + n0 + 8 * q;
#pragma unroll 8
    for (int it = 0; it < kIters; ++it) {
      store_stream(reinterpret_cast<u32x4*>(dst), staged(it));
      dst += kRowStep * ldc;
    }
    return;
  }
  const int64_t col = n0 + 8 * q;
#pragma unroll 2
  for (int it = 0; it < kIters; ++it) {
    const u32x4 w = staged(it);
    const int64_t r = m0 + r0 + it * kRowStep;
    if (r >= M || col >= N) continue;
    uint16_t* dst = C + r * ldc + col;
    if (vec_ok && col + 8 <= N) {
      store_stream(reinterpret_cast<u32x4*>(dst), w);
    } else if (kAny && col + 8 <= N) {
      typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
      *reinterpret_cast<u32x4_any*>(dst) = u32x4_any{w.x, w.y, w.z, w.w};
    } else {
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
      for (int e = 0; e < 8 && col + e < N; ++e)
        dst[e] = static_cast<uint16_t>(e & 1 ? ws[e >> 1] >> 16 : ws[e >> 1] & 0xffffu);
    }
  }
}

}  // namespace
}  // namespace nmce
