// Embedding lookup over a vocabulary shard, with scaling, and the weight's
// gradient, for gfx950.
//
// Forward   out[i] = scale * W[t_i - start]   for ids of the shard, else 0
//           (the masked lookup whose rows the TP group sums).
// Backward  dW[v] = scale * sum over the i with t_i = start + v of dY[i],
//           written whole: rows that no id names are zero.
//
// Both move bytes and do next to no arithmetic: the forward is bound by the
// rows it reads and writes, the backward by dY's rows and the whole of dW.
//
// The backward adds no values with atomics: the order of a row's sum would
// change from run to run. Positions are sorted by id instead (a stable radix
// sort, so a row's positions ascend), and the sorted list is cut into chunks of
// equal length, whatever ids they hold: a wave walks one chunk for 512 columns
// and writes each id's sum that begins and ends inside. Sums that cross chunks
// leave one fp32 partial per chunk, added in order by a last kernel. A common
// id with thousands of positions is so spread over as many waves as its rows
// need, and the result depends on the inputs alone.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "nmce.h"
#include "nmce_device.h"

namespace nmce {
namespace {

constexpr int kSlab = 512;         // columns of a wave: 8 a lane
constexpr int kPerLane = kSlab / 64;
constexpr int kBlock = 256;        // four waves, each on its own
constexpr int64_t kMaxBlocks = 1 << 22;  // grid-stride past this many
constexpr int64_t kMaxHidden = 1 << 24;

// The 8 columns of `slab` that a lane holds: kVec: 8 in a row (16-byte
// accesses); otherwise every 64th (any alignment; coalesced).
template <bool kVec>
__device__ __forceinline__ int64_t column(int64_t slab, int lane, int e) {
  return slab * kSlab + (kVec ? lane * kPerLane + e : lane + 64 * e);
}

// A lane's 8 columns of one row as they were loaded, so that several rows' loads
// are in flight before the first is unpacked.
template <typename T, bool kVec, bool kStream = false>
struct Row {
  static constexpr int kVecs = kPerLane / Elem<T>::kPerVec;
  u32x4 v[kVec ? kVecs : 1];
  T e[kVec ? 1 : kPerLane];

  __device__ __forceinline__ void load(const T* __restrict__ row, int64_t slab, int lane,
                                       int64_t h) {
    if constexpr (kVec) {
      const int64_t c0 = column<true>(slab, lane, 0);
      if (c0 + kPerLane <= h) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          const u32x4* p = reinterpret_cast<const u32x4*>(row + c0 + i * Elem<T>::kPerVec);
          v[i] = kStream ? load_stream(p) : *p;
        }
      } else {  // the row's last columns, fewer than 8
        float f[kPerLane];
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
          f[i] = c0 + i < h ? Elem<T>::load1(row + c0 + i) : 0.0f;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) v[i] = Elem<T>::pack(f + i * Elem<T>::kPerVec);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int64_t c = column<false>(slab, lane, i);
        e[i] = c < h ? row[c] : T(0);
      }
    }
  }
  __device__ __forceinline__ void get(float* f) const {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) Elem<T>::unpack(v[i], f + i * Elem<T>::kPerVec);
    } else {
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) f[i] = Elem<T>::load1(&e[i]);
    }
  }
};

template <typename T, bool kVec, bool kStream = false>
__device__ __forceinline__ void store_row(T* __restrict__ row, int64_t slab, int lane, int64_t h,
                                          const float* f) {
  if (kVec && column<true>(slab, lane, kPerLane - 1) < h) {
    T* p = row + column<true>(slab, lane, 0);
#pragma unroll
    for (int v = 0; v < kPerLane; v += Elem<T>::kPerVec) {
      u32x4* q = reinterpret_cast<u32x4*>(p + v);
      if (kStream)
        store_stream(q, Elem<T>::pack(f + v));
      else
        *q = Elem<T>::pack(f + v);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < kPerLane; ++e) {
    const int64_t c = column<kVec>(slab, lane, e);
    if (c < h) Elem<T>::store1(row + c, f[e]);
  }
}

// The row of id `t` in the shard, or `vocab` for an id of another one. (The
// difference is taken without a sign: any 64-bit id is told apart.)
__device__ __forceinline__ uint32_t local_row(int64_t t, int64_t start, int64_t vocab) {
  const uint64_t d = static_cast<uint64_t>(t) - static_cast<uint64_t>(start);
  return static_cast<uint32_t>(d < static_cast<uint64_t>(vocab) ? d
                                                                : static_cast<uint64_t>(vocab));
}

// A wave copies 512 columns (blockIdx.y's) of kRows tokens' rows, whose loads are
// in flight together. With one row a wave, its three dependent accesses (id, row,
// output) and nothing beside them, 131072 bf16 rows of 1024 took 87 us; with eight
// 69, and 54 (5.5 TB/s) with the outputs past the caches. Fewer tokens than fill the
// chip that way take one each, and leave their rows in the caches.
template <typename W, typename O, bool kVec, int kRows>
__global__ __launch_bounds__(kBlock) void embed_fwd_kernel(
    const int64_t* __restrict__ tokens, int64_t n, const W* __restrict__ weight, int64_t vocab,
    int64_t h, int64_t ldw, int64_t start, float scale, O* __restrict__ out, int64_t ldo) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t slab = blockIdx.y;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kBlock / 64) * kRows;
  for (int64_t i0 = (static_cast<int64_t>(blockIdx.x) * (kBlock / 64) + wave) * kRows; i0 < n;
       i0 += step) {
    const int mine = lane % kRows;
    const uint32_t my_row =
        local_row(tokens[i0 + mine < n ? i0 + mine : n - 1], start, vocab);
    Row<W, kVec> rows[kRows];
    uint32_t at[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      at[r] = __builtin_amdgcn_readlane(my_row, r);
      if (at[r] < vocab) rows[r].load(weight + at[r] * ldw, slab, lane, h);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (i0 + r >= n) break;
      float f[kPerLane] = {};
      if (at[r] < vocab) {
        rows[r].get(f);
#pragma unroll
        for (int e = 0; e < kPerLane; ++e) f[e] *= scale;
      }
      store_row<O, kVec, (kRows > 1)>(out + (i0 + r) * ldo, slab, lane, h, f);
    }
  }
}

// ---- the sort ---------------------------------------------------------------
// Stable least-significant-digit radix sort of (row, position) by row, digits
// of at most 9 bits. A pass cuts the list into at most 128 tiles, one workgroup
// each: one kernel counts every tile's digits, the next reads all tiles' counts,
// forms where its own digits start, and moves its keys. A wave walks a
// contiguous eighth of the tile 64 keys at a time; equal digits among the 64
// are found with one ballot per digit bit, which ranks them in order. 131072 ids in
// two passes take 33 us; in tiles of 4096, half as many, 43.
constexpr int kSortBlock = 512;
constexpr int kSortWaves = kSortBlock / 64;
constexpr int kMaxDigit = 9;
constexpr int kBins = 1 << kMaxDigit;
static_assert(kBins == kSortBlock, "a thread per bin");
constexpr int kMaxTiles = 128;
constexpr int kMinTile = 2048;

// dW's zeros, written by the workgroups of a sort launch that have no tile: 16
// bytes a thread (again a launch further on where dW is larger than that), dW's
// last bytes, fewer than 16, one by one. The sort keeps half of the chip at most, and
// waits for memory more than it reads: under the fill it costs nothing. More
// stores a thread leave the launch's writes further apart: lookup and gradient of
// 16384 ids with 1.05 GB of dW take 262 us with one, 279 with two, 312 with four.
struct Fill {
  char* to;
  int64_t bytes;
};
constexpr int64_t kMaxFillThreads = int64_t{1} << 31;

__device__ __forceinline__ void fill_zeros(const Fill& f, int64_t block) {
  const int64_t vecs = f.bytes / 16;
  const int64_t first = block * blockDim.x + threadIdx.x;
  for (int64_t i = first; i < vecs; i += kMaxFillThreads)
    store_stream(reinterpret_cast<u32x4*>(f.to) + i, u32x4{0, 0, 0, 0});
  if (first < f.bytes - vecs * 16) f.to[vecs * 16 + first] = 0;
}

struct SortArgs {
  const int64_t* tokens;  // first pass: the ids; later: keys and positions
  const uint32_t* keys;
  const uint32_t* pos;
  uint32_t* keys_out;
  uint32_t* pos_out;
  uint32_t* hist;         // [tiles][kBins]
  Fill fill;              // this launch's share of dW
  int64_t n, start, vocab, tile;
  int tiles, shift, bits;
};

// A sort launch's workgroups behind the tiles fill; true for those.
__device__ __forceinline__ bool filled(const SortArgs& a) {
  if (static_cast<int>(blockIdx.x) < a.tiles) return false;
  fill_zeros(a.fill, static_cast<int>(blockIdx.x) - a.tiles);
  return true;
}

template <bool kFirst>
__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, int64_t i) {
  if constexpr (kFirst) return local_row(a.tokens[i], a.start, a.vocab);
  return a.keys[i];
}

// This wave's keys of the tile: [*lo, *hi).
__device__ __forceinline__ void wave_range(const SortArgs& a, int wave, int64_t* lo, int64_t* hi) {
  const int64_t share = a.tile / kSortWaves;  // a multiple of 64
  const int64_t first = blockIdx.x * a.tile + wave * share;
  *lo = first < a.n ? first : a.n;
  *hi = first + share < a.n ? first + share : a.n;
}

// cnt[w][d]: how many of wave w's keys have digit d.
template <bool kFirst>
__device__ __forceinline__ void count_digits(const SortArgs& a, uint32_t (*cnt)[kBins], int wave,
                                             int lane) {
  for (int w = 0; w < kSortWaves; ++w) cnt[w][threadIdx.x] = 0;
  __syncthreads();
  int64_t lo, hi;
  wave_range(a, wave, &lo, &hi);
  const uint32_t mask = (1u << a.bits) - 1;
  for (int64_t i = lo + lane; i < hi; i += 64)
    atomicAdd(&cnt[wave][(sort_key<kFirst>(a, i) >> a.shift) & mask], 1u);
  __syncthreads();
}

template <bool kFirst>
__global__ __launch_bounds__(kSortBlock) void sort_count_kernel(SortArgs a) {
  __shared__ uint32_t cnt[kSortWaves][kBins];
  if (filled(a)) return;
  count_digits<kFirst>(a, cnt, threadIdx.x >> 6, threadIdx.x & 63);
  uint32_t sum = 0;
  for (int w = 0; w < kSortWaves; ++w) sum += cnt[w][threadIdx.x];
  a.hist[static_cast<int64_t>(blockIdx.x) * kBins + threadIdx.x] = sum;
}

template <bool kFirst>
__global__ __launch_bounds__(kSortBlock) void sort_move_kernel(SortArgs a) {
  __shared__ uint32_t cnt[kSortWaves][kBins];
  __shared__ uint32_t scan[kBins];
  if (filled(a)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = threadIdx.x;
  count_digits<kFirst>(a, cnt, wave, lane);
  // Keys of smaller digits, of the same digit in earlier tiles, and in this
  // tile's earlier waves come first.
  uint32_t before = 0, all = 0;
#pragma unroll 32
  for (int t = 0; t < a.tiles; ++t) {
    const uint32_t c = a.hist[static_cast<int64_t>(t) * kBins + d];
    before += t < static_cast<int>(blockIdx.x) ? c : 0u;
    all += c;
  }
  scan[d] = all;
  __syncthreads();
  for (int s = 1; s < kBins; s <<= 1) {
    const uint32_t v = d >= s ? scan[d - s] : 0u;
    __syncthreads();
    scan[d] += v;
    __syncthreads();
  }
  uint32_t at = scan[d] - all + before;
  for (int w = 0; w < kSortWaves; ++w) {
    const uint32_t c = cnt[w][d];
    cnt[w][d] = at;
    at += c;
  }
  __syncthreads();
  int64_t lo, hi;
  wave_range(a, wave, &lo, &hi);
  const uint32_t mask = (1u << a.bits) - 1;
  // The wave's own row of cnt is where its next key of each digit goes; lanes
  // hand it to one another between steps, so it is read and written as memory.
  volatile uint32_t* next = cnt[wave];
  for (int64_t base = lo; base < hi; base += 64) {
    const int64_t i = base + lane;
    const bool valid = i < hi;
    const uint32_t key = valid ? sort_key<kFirst>(a, i) : 0u;
    const uint32_t digit = (key >> a.shift) & mask;
    uint64_t same = __ballot(valid);
    for (int b = 0; b < a.bits; ++b) {
      const uint64_t set = __ballot((digit >> b) & 1u);
      same &= (digit >> b) & 1u ? set : ~set;
    }
    const uint32_t rank = __builtin_amdgcn_mbcnt_hi(
        static_cast<uint32_t>(same >> 32),
        __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(same), 0u));
    const uint32_t to = valid ? next[digit] + rank : 0u;
    __builtin_amdgcn_wave_barrier();
    if (valid) {
      if (rank == 0) next[digit] = to + static_cast<uint32_t>(__popcll(same));
      a.keys_out[to] = key;
      a.pos_out[to] = kFirst ? static_cast<uint32_t>(i) : a.pos[i];
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The whole sort in one workgroup, for lists of at most kSmallSort positions: a
// key and its position share 32 bits (position in the low bits), a thread holds
// up to 16 of them in registers, and each pass ranks them as above and scatters
// them through LDS. The counts and the list share the LDS: one is dead where the
// other is written. One launch where the passes above are four and more: 1024
// positions take 11 us in it, 16384 37 (those four as long, one after another), and
// the whole fill goes on beside it.
constexpr int kSmallBlock = 1024;
constexpr int kSmallWaves = kSmallBlock / 64;
constexpr int kSmallEach = 16;
constexpr int kSmallSort = kSmallBlock * kSmallEach;
constexpr int kSmallCounts = kSmallWaves * kBins * 2 + kBins * 4;  // bytes

struct SmallSortArgs {
  const int64_t* tokens;
  uint32_t* keys_out;
  uint32_t* pos_out;
  Fill fill;
  int64_t start, vocab;
  int n, pos_bits, passes, bits;
};

__global__ __launch_bounds__(kSmallBlock) void sort_small_kernel(SmallSortArgs a) {
  extern __shared__ __align__(16) char lds[];
  if (blockIdx.x > 0) {
    fill_zeros(a.fill, static_cast<int>(blockIdx.x) - 1);
    return;
  }
  uint32_t* list = reinterpret_cast<uint32_t*>(lds);
  uint16_t* counts = reinterpret_cast<uint16_t*>(lds);  // [kSmallWaves][kBins]
  uint32_t* scan = reinterpret_cast<uint32_t*>(lds + kSmallWaves * kBins * 2);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int rounds = (a.n + kSmallBlock - 1) / kSmallBlock;
  const int first = wave * rounds * 64 + lane;  // this thread's positions: every 64th
  uint32_t key[kSmallEach], to[kSmallEach];
#pragma unroll
  for (int i = 0; i < kSmallEach; ++i) {
    const int at = first + 64 * i;
    if (i < rounds && at < a.n)
      key[i] = local_row(a.tokens[at], a.start, a.vocab) << a.pos_bits | at;
  }
  const uint32_t mask = (1u << a.bits) - 1;
  for (int p = 0; p < a.passes; ++p) {
    const int shift = a.pos_bits + p * a.bits;
    if (p > 0) {
#pragma unroll
      for (int i = 0; i < kSmallEach; ++i)
        if (i < rounds && first + 64 * i < a.n) key[i] = list[first + 64 * i];
      __syncthreads();
    }
    for (int d = tid; d < kSmallWaves * kBins / 2; d += kSmallBlock)
      reinterpret_cast<uint32_t*>(counts)[d] = 0;
    __syncthreads();
    // Ranks within the wave; counts[wave][d] ends as its keys of digit d.
    volatile uint16_t* mine = counts + wave * kBins;
#pragma unroll
    for (int i = 0; i < kSmallEach; ++i) {
      if (i < rounds) {
        const bool valid = first + 64 * i < a.n;
        const uint32_t digit = (key[i] >> shift) & mask;
        uint64_t same = __ballot(valid);
        for (int b = 0; b < a.bits; ++b) {
          const uint64_t set = __ballot((digit >> b) & 1u);
          same &= (digit >> b) & 1u ? set : ~set;
        }
        const uint32_t rank = __builtin_amdgcn_mbcnt_hi(
            static_cast<uint32_t>(same >> 32),
            __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(same), 0u));
        const uint32_t before = valid ? mine[digit] : 0u;
        to[i] = before + rank;
        __builtin_amdgcn_wave_barrier();
        if (valid && rank == 0)
          mine[digit] = static_cast<uint16_t>(before + static_cast<uint32_t>(__popcll(same)));
        __builtin_amdgcn_wave_barrier();
      }
    }
    __syncthreads();
    // Where each wave's first key of each digit goes.
    uint32_t total = 0;
    if (tid < kBins) {
      for (int w = 0; w < kSmallWaves; ++w) total += counts[w * kBins + tid];
      scan[tid] = total;
    }
    __syncthreads();
    for (int s = 1; s < kBins; s <<= 1) {
      const uint32_t v = tid >= s && tid < kBins ? scan[tid - s] : 0u;
      __syncthreads();
      if (tid < kBins) scan[tid] += v;
      __syncthreads();
    }
    if (tid < kBins) {
      uint32_t at = scan[tid] - total;
      for (int w = 0; w < kSmallWaves; ++w) {
        const uint32_t c = counts[w * kBins + tid];
        counts[w * kBins + tid] = static_cast<uint16_t>(at);  // below kSmallSort
        at += c;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSmallEach; ++i)
      if (i < rounds && first + 64 * i < a.n)
        to[i] += counts[wave * kBins + ((key[i] >> shift) & mask)];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSmallEach; ++i)
      if (i < rounds && first + 64 * i < a.n) list[to[i]] = key[i];
    __syncthreads();
  }
  for (int i = tid; i < a.n; i += kSmallBlock) {
    a.keys_out[i] = list[i] >> a.pos_bits;
    a.pos_out[i] = list[i] & ((1u << a.pos_bits) - 1);
  }
}

// ---- dW ---------------------------------------------------------------------
__global__ __launch_bounds__(kBlock) void zero_kernel(Fill f) {
  fill_zeros(f, blockIdx.x);
}

struct SumArgs {
  const uint32_t* keys;  // sorted rows; `vocab` marks ids of other shards, at the end
  const uint32_t* pos;
  float* part;           // [chunks][2][h]: an id's sum that began in an earlier chunk, and
                         // one that goes on in the next
  int64_t n, vocab, h, ldy, chunks, slabs;
  int chunk;
  float scale;
};

// A wave adds one chunk's rows of dY over 512 columns, in the sorted order, eight
// rows' loads ahead of the eight being added, past the caches (131072 bf16 rows of
// 1024 67 us against 92 through them: 4.0 TB/s, rows of 1 KiB in any order).
template <typename G, typename W, bool kVec>
__global__ __launch_bounds__(kBlock) void embed_sum_kernel(const G* __restrict__ dy,
                                                           W* __restrict__ dw, SumArgs a) {
  constexpr int kAhead = 8;  // rows whose loads are in flight together
  const int lane = threadIdx.x & 63;
  const int64_t total = a.chunks * a.slabs;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kBlock / 64);
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * (kBlock / 64) +
                    __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
       id < total; id += step) {
    const int64_t c = id / a.slabs, slab = id - c * a.slabs;
    const int64_t first = c * a.chunk;
    const int64_t end = first + a.chunk < a.n ? first + a.chunk : a.n;
    // The keys around the chunk and its first 64 positions, asked for together.
    const uint32_t prev_key = c > 0 ? a.keys[first - 1] : 0u;
    const uint32_t next_key = a.keys[end < a.n ? end : a.n - 1];
    int count = static_cast<int>(end - first < 64 ? end - first : 64);
    uint32_t my_key = a.keys[first + (lane < count ? lane : 0)];
    uint32_t my_pos = a.pos[first + (lane < count ? lane : 0)];
    uint32_t cur = __builtin_amdgcn_readfirstlane(my_key);
    if (cur >= a.vocab) continue;  // so are all behind it
    bool from_before = c > 0 && prev_key == cur;
    float sum[kPerLane] = {};
    // The current id's sum is complete unless it began before this chunk.
    auto finish = [&](bool goes_on) {
      if (from_before || goes_on) {
        store_row<float, kVec>(a.part + (2 * c + (from_before ? 0 : 1)) * a.h, slab, lane, a.h,
                               sum);
      } else {
#pragma unroll
        for (int e = 0; e < kPerLane; ++e) sum[e] *= a.scale;
        store_row<W, kVec>(dw + cur * a.h, slab, lane, a.h, sum);
      }
      from_before = false;
    };
    bool others = false;  // the rest of the list is other shards'
    for (int64_t batch = first; batch < end && !others; batch += 64) {
      if (batch > first) {
        count = static_cast<int>(end - batch < 64 ? end - batch : 64);
        my_key = a.keys[batch + (lane < count ? lane : 0)];
        my_pos = a.pos[batch + (lane < count ? lane : 0)];
      }
      // Rows past the count repeat the last one: loads without branches.
      auto load = [&](Row<G, kVec, true>* rows, int j0) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const int at = j0 + j < count ? j0 + j : count - 1;
          const uint32_t p = __builtin_amdgcn_readlane(my_pos, at);
          rows[j].load(dy + p * a.ldy, slab, lane, a.h);
        }
      };
      auto add = [&](const Row<G, kVec, true>* rows, int j0) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          if (j0 + j >= count || others) continue;
          const uint32_t key = __builtin_amdgcn_readlane(my_key, j0 + j);
          if (key != cur) {
            finish(false);
            cur = key;
#pragma unroll
            for (int e = 0; e < kPerLane; ++e) sum[e] = 0.0f;
            if (key >= a.vocab) {
              others = true;
              continue;
            }
          }
          float f[kPerLane];
          rows[j].get(f);
#pragma unroll
          for (int e = 0; e < kPerLane; ++e) sum[e] += f[e];
        }
      };
      Row<G, kVec, true> r0[kAhead], r1[kAhead];
      load(r0, 0);
      for (int j0 = 0; j0 < count && !others; j0 += 2 * kAhead) {
        if (j0 + kAhead < count) load(r1, j0 + kAhead);
        add(r0, j0);
        if (j0 + 2 * kAhead < count) load(r0, j0 + 2 * kAhead);
        add(r1, j0 + kAhead);
      }
    }
    if (!others) finish(end < a.n && next_key == cur);
  }
}

// The sums that cross chunks: the workgroup of the chunk in which one begins
// (its second partial) adds the first partials of the chunks it goes on in, a
// quarter of them a wave, then the waves' sums in order.
template <typename W, bool kVec>
__global__ __launch_bounds__(kBlock) void embed_join_kernel(W* __restrict__ dw, SumArgs a) {
  constexpr int kWaves = kBlock / 64;
  __shared__ float part[kWaves][kPerLane][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t total = a.chunks * a.slabs;
  for (int64_t id = blockIdx.x; id < total; id += gridDim.x) {
    const int64_t c = id / a.slabs, slab = id - c * a.slabs;
    const int64_t first = c * a.chunk, next = first + a.chunk;
    if (next >= a.n) continue;
    const uint32_t key = a.keys[next], in_last = a.keys[next - 1], in_first = a.keys[first];
    const uint32_t before = c > 0 ? a.keys[first - 1] : key;
    if (key >= a.vocab || in_last != key) continue;             // nothing goes on
    if (c > 0 && in_first == key && before == key) continue;    // it began earlier
    // The last chunk that begins with the id, 64 chunks looked at together.
    int64_t last = c + 1;
    for (;; last += 64) {
      const int64_t at = (last + lane) * a.chunk;
      const uint64_t same = __ballot(at < a.n && a.keys[at < a.n ? at : next] == key);
      if (~same) {
        last += __builtin_ctzll(~same) - 1;
        break;
      }
    }
    const int64_t parts = last - c + 1, share = (parts + kWaves - 1) / kWaves;
    const int64_t from = wave * share;
    const int64_t to = from + share < parts ? from + share : parts;
    float sum[kPerLane] = {};
    constexpr int kAhead = 8;  // partials whose loads are in flight together
    for (int64_t p0 = from; p0 < to; p0 += kAhead) {
      Row<float, kVec> row[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int64_t p = p0 + j < to ? p0 + j : to - 1;
        row[j].load(a.part + (p == 0 ? 2 * c + 1 : 2 * (c + p)) * a.h, slab, lane, a.h);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (p0 + j >= to) continue;
        float f[kPerLane];
        row[j].get(f);
#pragma unroll
        for (int e = 0; e < kPerLane; ++e) sum[e] += f[e];
      }
    }
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) part[wave][e][lane] = sum[e];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int e = 0; e < kPerLane; ++e) {
        float s = part[0][e][lane];
        for (int w = 1; w < kWaves; ++w) s += part[w][e][lane];
        sum[e] = s * a.scale;
      }
      store_row<W, kVec>(dw + key * a.h, slab, lane, a.h, sum);
    }
    __syncthreads();
  }
}

// ---- host -------------------------------------------------------------------
inline int64_t slabs_of(int64_t h) { return (h + kSlab - 1) / kSlab; }

inline unsigned blocks_for(int64_t blocks) {
  return static_cast<unsigned>(blocks < kMaxBlocks ? blocks : kMaxBlocks);
}

// Workgroups that fill `bytes`.
inline int64_t fill_blocks(int64_t bytes, int threads) {
  const int64_t most = kMaxFillThreads / threads, want = bytes / 16 / threads + 1;
  return want < most ? want : most;
}

// Sorted positions per chunk: a power of two that leaves about 4096 waves (16
// for each compute unit's four SIMDs to switch between), at least 8, so that a
// wave has rows to keep in flight, and at most 256. (For twice or four times the
// waves 16384 x 4096 takes 266 and 279 us in all, against 262.)
inline int chunk_of(int64_t n, int64_t h) {
  int c = 8;
  while (c < 256 && n * slabs_of(h) / (2 * c) >= 4096) c *= 2;
  return c;
}

struct BwdLayout {
  int64_t tile, hist, keys[2], pos[2], part, total;
  int tiles, passes, bits, chunk, key_bits;
};

BwdLayout embed_layout(int64_t n, int64_t vocab, int64_t h) {
  BwdLayout L{};
  int key_bits = 1;  // rows 0 .. vocab
  while ((vocab >> key_bits) != 0) ++key_bits;
  L.key_bits = key_bits;
  L.passes = (key_bits + kMaxDigit - 1) / kMaxDigit;
  L.bits = (key_bits + L.passes - 1) / L.passes;
  L.tile = round_up(n > kMaxTiles ? (n + kMaxTiles - 1) / kMaxTiles : 1, kMinTile);
  L.tiles = static_cast<int>((n + L.tile - 1) / L.tile);
  L.chunk = chunk_of(n, h);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += align256(bytes);
    return o;
  };
  L.hist = take(static_cast<int64_t>(kMaxTiles) * kBins * 4);
  for (int i = 0; i < 2; ++i) {
    L.keys[i] = take(n * 4);
    L.pos[i] = take(n * 4);
  }
  L.part = take((n + L.chunk - 1) / L.chunk * 2 * h * 4);
  L.total = at;
  return L;
}

inline bool dtype_ok(int d) { return d == NMCE_F32 || d == NMCE_BF16; }
inline int64_t size_of(int d) { return d == NMCE_F32 ? 4 : 2; }

// Whole 16-byte vectors at every row's start.
inline bool rows_aligned(const void* p, int dtype, int64_t ld) {
  return aligned16(p) && (ld * size_of(dtype)) % 16 == 0;
}

int check_sizes(int64_t n, int64_t vocab, int64_t h) {
  // Rows and positions are held in 32 bits.
  const int64_t most = (int64_t{1} << 31) - 1;
  if (n < 0 || n > most || vocab < 1 || vocab > most || h < 1 || h > kMaxHidden)
    return NMCE_EINVAL_SHAPE;
  return NMCE_OK;
}

template <typename W, typename O, bool kVec, int kRows>
int launch_fwd_rows(const int64_t* tokens, int64_t n, const void* weight, int64_t vocab, int64_t h,
                    int64_t ldw, int64_t start, float scale, void* out, int64_t ldo,
                    hipStream_t s) {
  const int64_t slabs = slabs_of(h), per = (kBlock / 64) * kRows;
  const int64_t want = (n + per - 1) / per, most = (int64_t{1} << 22) / slabs + 1;
  const dim3 grid(static_cast<unsigned>(want < most ? want : most), static_cast<unsigned>(slabs));
  hipLaunchKernelGGL((embed_fwd_kernel<W, O, kVec, kRows>), grid, dim3(kBlock), 0, s, tokens, n,
                     static_cast<const W*>(weight), vocab, h, ldw, start, scale,
                     static_cast<O*>(out), ldo);
  return launch_status();
}

template <typename W, typename O>
int launch_fwd(const int64_t* tokens, int64_t n, const void* weight, int64_t vocab, int64_t h,
               int64_t ldw, int64_t start, float scale, void* out, int64_t ldo, bool vec,
               hipStream_t s) {
  // Eight rows a wave where they still make eight waves for every SIMD, of which a
  // compute unit has four.
  const bool many = n * slabs_of(h) >= int64_t{8} * 8 * 4 * device_cus();
#define NMCE_FWD(VEC, ROWS)                                                                      \
  launch_fwd_rows<W, O, VEC, ROWS>(tokens, n, weight, vocab, h, ldw, start, scale, out, ldo, s)
  if (vec) return many ? NMCE_FWD(true, 8) : NMCE_FWD(true, 1);
  return many ? NMCE_FWD(false, 8) : NMCE_FWD(false, 1);
#undef NMCE_FWD
}

// The sort in passes over tiles, with the fill spread over its launches; the
// last pass writes list (passes - 1) & 1.
int launch_sort(const int64_t* tokens, int64_t n, int64_t vocab, int64_t start, const BwdLayout& L,
                char* ws, const Fill& fill, hipStream_t s) {
  SortArgs a{};
  a.tokens = tokens;
  a.hist = reinterpret_cast<uint32_t*>(ws + L.hist);
  a.n = n;
  a.start = start;
  a.vocab = vocab;
  a.tile = L.tile;
  a.tiles = L.tiles;
  a.bits = L.bits;
  // Each of the sort's launches takes an equal share of the fill.
  const int64_t share = round_up((fill.bytes + 2 * L.passes - 1) / (2 * L.passes), 16);
  int64_t done = 0;
  auto next_fill = [&] {
    a.fill = Fill{fill.to + done, fill.bytes - done < share ? fill.bytes - done : share};
    done += a.fill.bytes;
    return dim3(static_cast<unsigned>(L.tiles + fill_blocks(a.fill.bytes, kSortBlock)));
  };
  for (int p = 0; p < L.passes; ++p) {
    a.shift = p * L.bits;
    a.keys = reinterpret_cast<const uint32_t*>(ws + L.keys[(p + 1) & 1]);
    a.pos = reinterpret_cast<const uint32_t*>(ws + L.pos[(p + 1) & 1]);
    a.keys_out = reinterpret_cast<uint32_t*>(ws + L.keys[p & 1]);
    a.pos_out = reinterpret_cast<uint32_t*>(ws + L.pos[p & 1]);
    const dim3 block(kSortBlock);
    dim3 grid = next_fill();
    if (p == 0) {
      hipLaunchKernelGGL(sort_count_kernel<true>, grid, block, 0, s, a);
      if (const int st = launch_status()) return st;
      grid = next_fill();
      hipLaunchKernelGGL(sort_move_kernel<true>, grid, block, 0, s, a);
    } else {
      hipLaunchKernelGGL(sort_count_kernel<false>, grid, block, 0, s, a);
      if (const int st = launch_status()) return st;
      grid = next_fill();
      hipLaunchKernelGGL(sort_move_kernel<false>, grid, block, 0, s, a);
    }
    if (const int st = launch_status()) return st;
  }
  return NMCE_OK;
}

// sort_small_kernel's list and the fill of the whole of dW.
int launch_small_sort(SmallSortArgs a, hipStream_t s) {
  static std::atomic<bool> lds_set{false};
  if (const int rc = allow_lds(reinterpret_cast<const void*>(&sort_small_kernel),
                               kSmallSort * 4, lds_set))
    return rc;
  const int list = a.n * 4, lds = list > kSmallCounts ? list : kSmallCounts;
  const dim3 grid(static_cast<unsigned>(1 + fill_blocks(a.fill.bytes, kSmallBlock)));
  hipLaunchKernelGGL(sort_small_kernel, grid, dim3(kSmallBlock), lds, s, a);
  return launch_status();
}

template <typename G, typename W, bool kVec>
int launch_sums(const void* dy, void* dw, const SumArgs& a, hipStream_t s) {
  const dim3 block(kBlock);
  hipLaunchKernelGGL((embed_sum_kernel<G, W, kVec>), dim3(blocks_for((a.chunks * a.slabs + 3) / 4)),
                     block, 0, s, static_cast<const G*>(dy), static_cast<W*>(dw), a);
  if (const int st = launch_status()) return st;
  hipLaunchKernelGGL((embed_join_kernel<W, kVec>), dim3(blocks_for(a.chunks * a.slabs)), block, 0,
                     s, static_cast<W*>(dw), a);
  return launch_status();
}

}  // namespace
}  // namespace nmce

using namespace nmce;

extern "C" {

int nmce_embedding_fwd(const int64_t* tokens, int64_t n_tokens, const void* weight,
                       int weight_dtype, int64_t vocab_local, int64_t hidden, int64_t ldw,
                       int64_t vocab_start, float scale, void* out, int out_dtype, int64_t ldo,
                       void* stream) {
  if (!dtype_ok(weight_dtype) || !dtype_ok(out_dtype)) return NMCE_EINVAL_DTYPE;
  if (const int st = check_sizes(n_tokens, vocab_local, hidden)) return st;
  if (ldw < hidden || ldo < hidden) return NMCE_EINVAL_SHAPE;
  if (n_tokens == 0) return NMCE_OK;
  if (!tokens || !weight || !out) return NMCE_EINVAL_PTR;
  if (reinterpret_cast<uintptr_t>(tokens) % 8 ||
      reinterpret_cast<uintptr_t>(weight) % size_of(weight_dtype) ||
      reinterpret_cast<uintptr_t>(out) % size_of(out_dtype))
    return NMCE_EINVAL_ALIGN;
  const bool vec = rows_aligned(weight, weight_dtype, ldw) && rows_aligned(out, out_dtype, ldo);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (weight_dtype == NMCE_F32)
    return out_dtype == NMCE_F32
               ? launch_fwd<float, float>(tokens, n_tokens, weight, vocab_local, hidden, ldw,
                                          vocab_start, scale, out, ldo, vec, s)
               : launch_fwd<float, uint16_t>(tokens, n_tokens, weight, vocab_local, hidden, ldw,
                                             vocab_start, scale, out, ldo, vec, s);
  return out_dtype == NMCE_F32
             ? launch_fwd<uint16_t, float>(tokens, n_tokens, weight, vocab_local, hidden, ldw,
                                           vocab_start, scale, out, ldo, vec, s)
             : launch_fwd<uint16_t, uint16_t>(tokens, n_tokens, weight, vocab_local, hidden, ldw,
                                              vocab_start, scale, out, ldo, vec, s);
}

int64_t nmce_embedding_bwd_workspace_bytes(int64_t n_tokens, int64_t vocab_local, int64_t hidden) {
  if (check_sizes(n_tokens, vocab_local, hidden)) return -1;
  return embed_layout(n_tokens, vocab_local, hidden).total;
}

int nmce_embedding_bwd(const int64_t* tokens, int64_t n_tokens, const void* grad_out,
                       int grad_dtype, int64_t ldg, int64_t vocab_local, int64_t hidden,
                       int64_t vocab_start, float scale, void* grad_weight, int weight_dtype,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  if (!dtype_ok(grad_dtype) || !dtype_ok(weight_dtype)) return NMCE_EINVAL_DTYPE;
  if (const int st = check_sizes(n_tokens, vocab_local, hidden)) return st;
  if (ldg < hidden) return NMCE_EINVAL_SHAPE;
  if (!grad_weight || (n_tokens > 0 && (!tokens || !grad_out))) return NMCE_EINVAL_PTR;
  if (reinterpret_cast<uintptr_t>(tokens) % 8 ||
      reinterpret_cast<uintptr_t>(grad_out) % size_of(grad_dtype) || !aligned16(grad_weight))
    return NMCE_EINVAL_ALIGN;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const BwdLayout L = embed_layout(n_tokens, vocab_local, hidden);
  char* ws = static_cast<char*>(workspace);
  if (n_tokens > 0 && (!ws || workspace_bytes < L.total || !aligned16(ws)))
    return NMCE_EINVAL_WORKSPACE;

  const int64_t bytes = vocab_local * hidden * size_of(weight_dtype);
  char* dw = static_cast<char*>(grad_weight);
  if (n_tokens == 0) {
    const dim3 grid(static_cast<unsigned>(fill_blocks(bytes, kBlock)));
    hipLaunchKernelGGL(zero_kernel, grid, dim3(kBlock), 0, s,
                       Fill{dw, bytes});
    return launch_status();
  }

  int pos_bits = 0;
  while (((n_tokens - 1) >> pos_bits) != 0) ++pos_bits;
  int sorted = 0;  // which of the two lists holds the result
  if (n_tokens <= kSmallSort && L.key_bits + pos_bits <= 32) {
    SmallSortArgs a{};
    a.tokens = tokens;
    a.keys_out = reinterpret_cast<uint32_t*>(ws + L.keys[0]);
    a.pos_out = reinterpret_cast<uint32_t*>(ws + L.pos[0]);
    a.fill = Fill{dw, bytes};
    a.start = vocab_start;
    a.vocab = vocab_local;
    a.n = static_cast<int>(n_tokens);
    a.pos_bits = pos_bits;
    a.passes = L.passes;
    a.bits = L.bits;
    if (const int st = launch_small_sort(a, s)) return st;
  } else {
    if (const int st = launch_sort(tokens, n_tokens, vocab_local, vocab_start, L, ws,
                                   Fill{dw, bytes}, s))
      return st;
    sorted = (L.passes - 1) & 1;
  }

  SumArgs m{};
  m.keys = reinterpret_cast<const uint32_t*>(ws + L.keys[sorted]);
  m.pos = reinterpret_cast<const uint32_t*>(ws + L.pos[sorted]);
  m.part = reinterpret_cast<float*>(ws + L.part);
  m.n = n_tokens;
  m.vocab = vocab_local;
  m.h = hidden;
  m.ldy = ldg;
  m.chunk = L.chunk;
  m.chunks = (n_tokens + L.chunk - 1) / L.chunk;
  m.slabs = slabs_of(hidden);
  m.scale = scale;
  // The partials' rows and dW's lie whole vectors apart where hidden does.
  const bool vec = rows_aligned(grad_out, grad_dtype, ldg) && hidden % 8 == 0;
#define NMCE_SUMS(G, W) \
  return vec ? launch_sums<G, W, true>(grad_out, grad_weight, m, s) \
             : launch_sums<G, W, false>(grad_out, grad_weight, m, s)
  if (grad_dtype == NMCE_F32) {
    if (weight_dtype == NMCE_F32) NMCE_SUMS(float, float);
    NMCE_SUMS(float, uint16_t);
  }
  if (weight_dtype == NMCE_F32) NMCE_SUMS(uint16_t, float);
  NMCE_SUMS(uint16_t, uint16_t);
#undef NMCE_SUMS
}

}  // extern "C"
