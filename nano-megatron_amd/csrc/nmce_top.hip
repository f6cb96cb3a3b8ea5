// The k largest logits of every row of a vocabulary shard, in order, with their ids
// (of equal logits the lowest id first), and the row's log-normaliser
// log sum exp(x / T), for gfx950.
//
// One pass over the row by one workgroup (or by several, a slab each, where the rows are
// few). The first chunk is held in registers; of two maxima a thread, the k-th largest
// is a floor under the row's k-th largest logit, since k of the row's elements reach it.
// Elements that reach the floor are noted as keys (value, id) in LDS, k and a few from
// the first chunk and as many again from each like stretch after it; when the notes
// fill up, all but the k largest go and the floor rises to the k-th. Keys are unique, so
// the order in which the lanes note them does not matter: the result is the same at
// every run. A chunk of which more reach the floor than fit (a row of equal logits) is
// first cut to its k largest keys by bisection.
//
// The exponentials' sum rides along. 4096 x 128256 bf16, k 64: 204 us (5.2 TB/s; the VALU is
// busy for 0.86 of it, 12 instructions an element, half of them the exponentials' sum; up to 260
// from the 2nd to the 9th millisecond of such work after idling, with or without a profiler).
// 777 x 100277 fp32, k 500: 103 (3.0 TB/s): the cuts take half of the instructions, and some
// compute units have four rows where the mean is 3.04. A few rows take the latency of their
// steps: read, floor, notes, order, and the merge's: one of 50257, k 20: 8 and 5 us.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "nmce.h"
#include "nmce_device.h"

namespace nmce {
namespace {

constexpr int kMaxK = NMCE_TOP_MAX_K;
constexpr int kVecs = 4;  // 16-byte vectors of a thread's chunk
constexpr int kLeast = 4096;

// A workgroup's shape: threads, the wanted logits it is for, places for notes (past half of
// them they are cut) and for those a cut leaves, maxima a thread gives to the floor. At k 128
// Few takes 28 us for 64 rows of 128256 bf16, Many 32; 85 and 95 for 4096 of 32000; 58 and 52
// for 512 of 128256. At k 20, 64 rows of 128256: 17 and 21; one of 50257 fp32: 12 and 14.
struct Few {
  static constexpr int kBlock = 256, kMost = 128, kNotes = 1024, kRoom = 160, kTops = 1;
};
struct Many {
  static constexpr int kBlock = 512, kMost = kMaxK, kNotes = 2048, kRoom = kMaxK, kTops = 2;
};

// A cut looks for a key that k or somewhat more reach: the last steps of a bisection would
// only tell neighbours apart, which putting them in order does anyway.
__host__ __device__ constexpr int enough(int k, int room) {
  return k + k / 8 + 8 < room ? k + k / 8 + 8 : room;
}
static_assert(enough(Few::kMost, 1 << 20) <= Few::kRoom, "");
constexpr float kInf = __builtin_huge_valf();

// An order of the logits as integers: NaN (any) above +inf, -0 as 0. bf16 takes 16 bits.
template <typename T>
struct Rank {
  static constexpr int kShift = sizeof(T) == 2 ? 16 : 0;
  __device__ static __forceinline__ uint32_t of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    const uint32_t r = static_cast<int32_t>(u) < 0 ? ~u : u | 0x80000000u;
    return (x != x ? 0xffffffffu : r) >> kShift;
  }
  __device__ static __forceinline__ float value(uint32_t rank) {
    const uint32_t r = rank << kShift;
    const uint32_t u = r & 0x80000000u ? r & 0x7fffffffu : ~r >> kShift << kShift;
    return __uint_as_float(u);
  }
  // A float below value(rank) and not below the next lower value (whose rank is one
  // less; -0, below 0, is no value).
  __device__ static __forceinline__ float below(uint32_t rank) {
    const uint32_t r = (rank << kShift) - 1;
    return Rank<float>::value(r == 0x7fffffffu ? r - 1 : r);
  }
};

// A list entry, as it leaves a shard: the fp32 value's order, then the id from the top
// down. 0 is no entry.
__device__ __forceinline__ uint64_t entry_of(float value, int64_t id) {
  return static_cast<uint64_t>(Rank<float>::of(value)) << 32 |
         (0xffffffffu - static_cast<uint32_t>(id));
}

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
  for (int s = 32; s > 0; s >>= 1) {
    const uint64_t o = __shfl_xor(static_cast<unsigned long long>(v), s);
    v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ uint64_t wave_min_u64(uint64_t v) { return ~wave_max_u64(~v); }

// One wave: a rank that k or somewhat more of the maxima reach; 0 if fewer are there.
template <int kMaxima>
__device__ uint32_t floor_rank(const uint32_t* maxima, int k) {
  const int lane = threadIdx.x & 63;
  uint32_t r[kMaxima / 64];
  uint32_t lo = 0xffffffffu, hi = 0;
  int here = 0;
#pragma unroll
  for (int i = 0; i < kMaxima / 64; ++i) {
    r[i] = maxima[i * 64 + lane];
    here += __popcll(__ballot(r[i] != 0));
    if (r[i] != 0) lo = r[i] < lo ? r[i] : lo;
    hi = r[i] > hi ? r[i] : hi;
  }
  if (here < k) return 0;
  for (int s = 32; s > 0; s >>= 1) {
    const uint32_t a = __shfl_xor(lo, s), b = __shfl_xor(hi, s);
    lo = a < lo ? a : lo;
    hi = b > hi ? b : hi;
  }
  const int enough = k + k / 8;
  while (hi - lo > 1) {  // here >= k reach lo
    const uint32_t mid = lo + (hi - lo) / 2;
    int c = 0;
#pragma unroll
    for (int i = 0; i < kMaxima / 64; ++i) c += __popcll(__ballot(r[i] >= mid));
    if (c >= k) {
      lo = mid;
      if (c <= enough) break;
    } else {
      hi = mid;
    }
  }
  return lo;
}

// 16 bytes at any element's alignment (rows of odd widths start anywhere), streamed: 4096 x
// 128256 bf16 241 -> 215 us.
__device__ __forceinline__ u32x4 load16(const void* p) {
  typedef u32x4 anywhere __attribute__((aligned(2)));
  return __builtin_nontemporal_load(static_cast<const anywhere*>(p));
}

template <typename Shape>
struct Shared {
  uint64_t notes[Shape::kNotes];
  __align__(16) uint64_t kept[Shape::kRoom];
  uint64_t wave_lo[Shape::kBlock / 64], wave_hi[Shape::kBlock / 64];
  uint32_t floor;  // of the first chunk
  float first;     // the largest logit
  int n, n_kept, counts[3];
  float wave_m[Shape::kBlock / 64];
  double wave_s[Shape::kBlock / 64];
};

// One wave: a key that k to `most` of n keys reach, by bisection over eight of them a lane in
// registers, and what there is beyond 512 from LDS. The keys are unique but for zeros, which
// are none and reach nothing; of the others there are k at least, and more than `most` if n is.
__device__ uint64_t kth_key(const uint64_t* list, int n, int k, int most) {
  constexpr int kHeld = 8;
  const int lane = threadIdx.x & 63;
  uint64_t held[kHeld];
  uint64_t lo = ~uint64_t{0}, hi = 0;
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const int i = j * 64 + lane;
    held[j] = i < n ? list[i] : 0;
    if (i < n) {
      lo = held[j] < lo ? held[j] : lo;
      hi = held[j] > hi ? held[j] : hi;
    }
  }
  for (int i = kHeld * 64 + lane; i < n; i += 64) {
    lo = list[i] < lo ? list[i] : lo;
    hi = list[i] > hi ? list[i] : hi;
  }
  // Above 0: past the largest entry there can be (a NaN's at id 0, all ones) hi is 2^64, held
  // as 0, and hi - lo is right only where lo is not 0 too.
  lo = wave_min_u64(lo);
  lo = lo > 0 ? lo : 1;
  hi = wave_max_u64(hi) + 1;
  while (n > most && hi - lo > 1) {  // more than `most` reach lo, fewer than k reach hi
    const uint64_t mid = lo + (hi - lo) / 2;  // (above lo, so a 0 does not reach it)
    int c = 0;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) c += __popcll(__ballot(held[j] >= mid));
    for (int i = kHeld * 64; i < n; i += 64)
      c += __popcll(__ballot(i + lane < n && list[i + lane] >= mid));
    if (c >= k) lo = mid;
    if (c >= k && c <= most) break;
    if (c < k) hi = mid;
  }
  return lo;
}

// The k largest of the n notes (k <= n, unique keys), and a few more, into kept; the key
// that they reach is returned. Every thread calls it, behind a barrier. Few notes are one
// wave's work while the others wait (and other workgroups read): 4096 x 128256 bf16, k 64:
// 207 us, by all waves 220. More are held by all threads, four a thread, a barrier a step:
// 777 x 100277 fp32, k 500: 112 us, by one wave from LDS 137.
template <typename Shape>
__device__ uint64_t cut_notes(Shared<Shape>& sh, int n, int k) {
  constexpr int kEach = Shape::kNotes / Shape::kBlock, kWaves = Shape::kBlock / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int most = enough(k, Shape::kRoom);
  if (Shape::kNotes <= 1024 || n <= 512) {
    if (wave == 0) {
      const uint64_t key = kth_key(sh.notes, n, k, most);
      if (lane == 0) {
        sh.wave_lo[0] = key;
        sh.n_kept = 0;
      }
    }
    __syncthreads();
    const uint64_t key = sh.wave_lo[0];
    for (int i = tid; i < n; i += Shape::kBlock)
      if (sh.notes[i] >= key) sh.kept[atomicAdd(&sh.n_kept, 1)] = sh.notes[i];
    __syncthreads();
    return key;
  }
  uint64_t held[kEach];
  uint64_t lo = ~uint64_t{0}, hi = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = j * Shape::kBlock + tid;
    held[j] = i < n ? sh.notes[i] : 0;
    if (i < n) {
      lo = held[j] < lo ? held[j] : lo;
      hi = held[j] > hi ? held[j] : hi;
    }
  }
  lo = wave_min_u64(lo);
  hi = wave_max_u64(hi);
  if (lane == 0) {
    sh.wave_lo[wave] = lo;
    sh.wave_hi[wave] = hi;
  }
  if (tid == 0) sh.counts[0] = sh.counts[1] = sh.counts[2] = sh.n_kept = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    lo = sh.wave_lo[w] < lo ? sh.wave_lo[w] : lo;
    hi = sh.wave_hi[w] > hi ? sh.wave_hi[w] : hi;
  }
  ++hi;
  // More than `most` reach lo, fewer than k reach hi.
  for (int turn = 0; n > most && hi - lo > 1; turn = turn == 2 ? 0 : turn + 1) {
    const uint64_t mid = lo + (hi - lo) / 2;  // (above lo, so a 0 does not reach it)
    int c = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) c += __popcll(__ballot(held[j] >= mid));
    if (lane == 0) atomicAdd(&sh.counts[turn], c);
    __syncthreads();
    c = sh.counts[turn];
    if (tid == 0) sh.counts[turn == 0 ? 2 : turn - 1] = 0;  // read by all before this barrier
    if (c >= k) lo = mid;
    if (c >= k && c <= most) break;
    if (c < k) hi = mid;
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (j * Shape::kBlock + tid < n && held[j] >= lo)
      sh.kept[atomicAdd(&sh.n_kept, 1)] = held[j];
  __syncthreads();
  return lo;
}

// The n <= kRoom keys in falling order, put(place, key) each. Every thread calls it, behind a
// barrier. Few are counted among one another (8 cycles of LDS for two keys and a wave);
// 256 and more are sorted, in pairs of growing distance: 500 keys 2 us, counted 7.
template <int kThreads, int kRoom, typename Put>
__device__ void in_order(uint64_t* keys, int n, Put&& put) {
  const int tid = threadIdx.x;
  if (kRoom <= 256 || n <= 160) {
    const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(keys);
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t key = keys[i];
      int place = 0;
#pragma unroll 4
      for (int j = 0; j < n / 2; ++j) {
        const ulonglong2 two = pairs[j];
        place += (two.x > key) + (two.y > key);
      }
      if (n & 1) place += keys[n - 1] > key;
      put(place, key);
    }
    return;
  }
  int all = 256;
  while (all < n) all *= 2;
  for (int i = n + tid; i < all; i += kThreads) keys[i] = 0;
  for (int size = 2; size <= all; size *= 2) {
    for (int apart = size / 2; apart > 0; apart /= 2) {
      __syncthreads();
      for (int t = tid; t < all / 2; t += kThreads) {
        const int i = 2 * t - (t & (apart - 1)), j = i + apart;
        const uint64_t a = keys[i], b = keys[j];
        if ((a < b) == ((i & size) == 0)) {
          keys[i] = b;
          keys[j] = a;
        }
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) put(i, keys[i]);
}

// The results of whole rows; norm null: lists are wanted.
template <typename T>
struct Out {
  T* values;
  int64_t* ids;
  float* norm;
};

// log sum exp(x / T) from the maximum m, the sum over exp((x - m) / T) and the first of
// the top logits, which is NaN where any is. +inf beside numbers is the sum.
__device__ __forceinline__ float log_norm(float m, double s, float first, double c) {
  return first != first ? first
         : m == kInf    ? kInf
                        : static_cast<float>(static_cast<double>(m) * c + log(s));
}

// Row blockIdx.x / slabs, columns [slab * width, + width) of it. lists[row][slab] gets k
// entries in order and the pair (maximum, sum of exp((x - maximum) / T)); or, of whole
// rows, `out` the results.
// 64 registers: four workgroups share a compute unit, and while one looks for its floor or
// its k-th key (a wave's work, the others wait) the rest read.
template <typename T, typename Shape>
__global__ __launch_bounds__(Shape::kBlock, 8) void top_kernel(const T* __restrict__ x, int64_t ld,
                                                        int64_t v, int64_t vocab_start,
                                                        int64_t slabs, int64_t width, int k,
                                                        int id_bits, float c, double c64,
                                                        uint64_t* __restrict__ lists,
                                                        Out<T> results) {
  using E = Elem<T>;
  constexpr int EPV = E::kPerVec;
  constexpr int kBlock = Shape::kBlock, kNotes = Shape::kNotes, kWaves = kBlock / 64;
  static_assert(2 * Shape::kMost <= kNotes && Shape::kMost <= Shape::kTops * kBlock &&
                Shape::kTops * kBlock * 4 <= kNotes * 8, "");
  __shared__ Shared<Shape> sh;
  constexpr uint32_t kChunk = kBlock * kVecs * EPV;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / slabs, slab = blockIdx.x - row * slabs;
  // Columns below are of the slab, from 0.
  const int64_t from = slab * width;
  const uint32_t end = static_cast<uint32_t>(v - from < width ? v - from : width);
  const T* xr = x + row * ld + from;
  const uint64_t last_id = (uint64_t{1} << id_bits) - 1 - static_cast<uint64_t>(from);
  const uint64_t id_mask = (uint64_t{1} << id_bits) - 1;
  auto key_of = [&](float f, uint32_t column) {
    return static_cast<uint64_t>(Rank<T>::of(f)) << id_bits | (last_id - column);
  };
  // The first column of the thread's vector i. (Opaque to the compiler, which would keep
  // what it can compute from each of them in registers through the loop.)
  auto column_of = [&](uint32_t base, int i) {
    uint32_t t = base + static_cast<uint32_t>(tid * EPV);
    asm volatile("" : "+v"(t));
    return t + i * kBlock * EPV;
  };
  // Vectors i and i + 1 of the chunk from `base`: the one that the row ends in by its
  // elements, -inf behind it.
  auto load_pair = [&](uint32_t base, int i, u32x4& w0, u32x4& w1) {
    constexpr uint32_t kNone = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;  // -inf
    const uint32_t col = column_of(base, i);
    if (base + (i + 2) * kBlock * EPV <= end) {  // (the same for all threads)
      w0 = load16(xr + col);
      w1 = load16(xr + col + kBlock * EPV);
      return;
    }
    w0 = w1 = u32x4{kNone, kNone, kNone, kNone};
    auto last = [&](uint32_t c0, u32x4& w) {
      if (c0 + EPV <= end) {
        w = load16(xr + c0);
      } else if (c0 < end) {
        float f[EPV];
#pragma unroll
        for (int e = 0; e < EPV; ++e) f[e] = c0 + e < end ? E::load1(xr + c0 + e) : -kInf;
        w = E::pack(f);
      }
    };
    last(col, w0);
    last(col + kBlock * EPV, w1);
  };
  // The next free note. (The address is opaque: known to be the same for all lanes, the
  // compiler would count the lanes first, for 15 instructions more.)
  auto take_place = [&]() {
    auto* p = (__attribute__((address_space(3))) int*)&sh.n;
    asm volatile("" : "+v"(p));
    return __hip_atomic_fetch_add(p, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  if (tid == 0) sh.n = 0;
  u32x4 cur[kVecs];
  float m = kNegHuge, s = 0.0f;
  float floor = 0.0f;
  int n = 0;     // notes,
  int keys = 0;  // the first of them as keys; the others as (value, column), in fewer steps
  auto to_keys = [&](int first, int last) {
    for (int i = first + tid; i < last; i += kBlock) {
      const uint64_t note = sh.notes[i];
      sh.notes[i] = key_of(__uint_as_float(static_cast<uint32_t>(note >> 32)),
                           static_cast<uint32_t>(note));
    }
    __syncthreads();
  };
#pragma unroll
  for (int i = 0; i < kVecs; i += 2) load_pair(0, i, cur[i], cur[i + 1]);
  for (uint32_t base = 0; base < end; base += kChunk) {
    if (base == 0) {
      // The floor: from the maxima of a thread's even and odd vectors.
      uint32_t* maxima = reinterpret_cast<uint32_t*>(sh.notes);
#pragma unroll
      for (int h = 0; h < Shape::kTops; ++h) {
        uint32_t top = 0;
#pragma unroll
        for (int i = h; i < kVecs; i += Shape::kTops) {
          if (column_of(base, i) < end) {
            float f[EPV];
            E::unpack(cur[i], f);
            float q = -kInf;
#pragma unroll
            for (int e = 0; e < EPV; ++e) q = fmaxf(q, f[e]);
            const uint32_t r = Rank<T>::of(q);
            top = r > top ? r : top;
          }
        }
        maxima[h * kBlock + tid] = top;
      }
      __syncthreads();
      if (wave == 0) {
        const uint32_t r = floor_rank<Shape::kTops * kBlock>(maxima, k);
        if (lane == 0) sh.floor = r;
      }
      __syncthreads();
      // What reaches the floor: above the next lower value (NaN: everything does).
      const uint32_t r = sh.floor;
      floor = r > Rank<T>::of(-kInf) ? Rank<T>::below(r) : __builtin_nanf("");
    }
    const int before = n;
    if (base != 0) __syncthreads();  // every thread has read the last chunk's count
#pragma unroll
    for (int i = 0; i < kVecs; i += 2) {
      if (base + i * kBlock * EPV >= end) break;  // (the same for all threads)
      float q, sum;
      {
        float f[2 * EPV];
        E::unpack(cur[i], f);
        E::unpack(cur[i + 1], f + EPV);
        q = f[0];
#pragma unroll
        for (int j = 1; j < 2 * EPV; ++j) q = fmaxf(q, f[j]);
        const float nm = fmaxf(m, q);
#pragma unroll
        for (int j = 0; j < 2 * EPV; ++j) f[j] = exp2_hw((f[j] - nm) * c);
#pragma unroll
        for (int w = 1; w < 2 * EPV; w *= 2) {
#pragma unroll
          for (int j = 0; j + w < 2 * EPV; j += 2 * w) f[j] += f[j + w];
        }
        sum = f[0];
        s = fmaf(s, exp2_hw((m - nm) * c), sum);
        m = nm;
      }
      // (A NaN among them shows in their sum.) Few lanes have anything to note, and
      // those one element mostly: each notes its own.
      if (!(q <= floor) || sum != sum) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t col = column_of(base, i + h);
          u32x4 w = cur[i + h];
          asm volatile("" : "+v"(w));  // unpack again: the exponentials took the registers
          float f[EPV];
          E::unpack(w, f);
#pragma unroll
          for (int j = 0; j < EPV; ++j) {
            if (!(f[j] <= floor) && col + j < end) {
              const int at = take_place();
              if (at < kNotes)
                sh.notes[at] = static_cast<uint64_t>(__float_as_uint(f[j])) << 32 | (col + j);
            }
          }
        }
      }
      // The next chunk's take their place, under way across the barriers.
      if (base + kChunk < end) load_pair(base + kChunk, i, cur[i], cur[i + 1]);
    }
    __syncthreads();
    n = sh.n;
    if (n > kNotes) {
      // More reach the floor than fit: the chunk's k largest keys alone, by bisection
      // over its elements, read again. (The notes from before are whole.)
      auto each_key = [&](auto&& use) {
#pragma unroll 1
        for (int i = 0; i < kVecs; ++i) {
          const uint32_t col = column_of(base, i);
          if (col + EPV <= end) {
            float f[EPV];
            E::unpack(load16(xr + col), f);
#pragma unroll
            for (int j = 0; j < EPV; ++j) use(key_of(f[j], col + j));
          } else {
            for (uint32_t c = col; c < end; ++c) use(key_of(E::load1(xr + c), c));
          }
        }
      };
      uint64_t lo = 0, hi = uint64_t{1} << (32 - Rank<T>::kShift + id_bits);
      if (tid == 0) sh.counts[0] = sh.counts[1] = 0;
      __syncthreads();
      for (int turn = 0; hi - lo > 1; turn ^= 1) {
        const uint64_t mid = lo + (hi - lo) / 2;
        int count = 0;
        each_key([&](uint64_t key) { count += key >= mid; });
        for (int d = 32; d > 0; d >>= 1) count += __shfl_xor(count, d);
        if (lane == 0) atomicAdd(&sh.counts[turn], count);
        __syncthreads();
        const int all = sh.counts[turn];
        if (tid == 0) sh.counts[turn ^ 1] = 0;
        __syncthreads();
        if (all == k) {
          lo = mid;
          break;
        }
        if (all > k) lo = mid;
        else hi = mid;
      }
      if (tid == 0) sh.n = before;
      __syncthreads();
      each_key([&](uint64_t key) {
        if (key >= lo) sh.notes[atomicAdd(&sh.n, 1)] = key;
      });
      __syncthreads();
      n = sh.n;
      to_keys(keys, before);
      keys = n;
    }
    if (base == 0 && sh.floor != 0) floor = Rank<T>::value(sh.floor);
    if (n > kNotes / 2) {
      to_keys(keys, n);
      const uint64_t key = cut_notes(sh, n, k);
      n = keys = sh.n_kept;
      for (int i = tid; i < n; i += kBlock) sh.notes[i] = sh.kept[i];
      if (tid == 0) sh.n = n;
      // Later columns of the same value come behind: only what is above it counts.
      floor = Rank<T>::value(static_cast<uint32_t>(key >> id_bits));
      __syncthreads();
    }
  }

  // The sum over the workgroup, in 64 bits.
  float wm = wave_max(m);
  if (lane == 0) sh.wave_m[wave] = wm;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) wm = fmaxf(wm, sh.wave_m[w]);
  double total = static_cast<double>(s) * static_cast<double>(exp2_hw((m - wm) * c));
  for (int d = 32; d > 0; d >>= 1) total += __shfl_xor(total, d);
  if (lane == 0) sh.wave_s[wave] = total;
  to_keys(keys, n);
  if (n > k) {
    cut_notes(sh, n, k);
    n = sh.n_kept;
  } else {
    for (int i = tid; i < n; i += kBlock) sh.kept[i] = sh.notes[i];
    __syncthreads();
  }
  uint64_t* out = lists + blockIdx.x * static_cast<int64_t>(k + 1);
  in_order<kBlock, Shape::kRoom>(sh.kept, n, [&](int place, uint64_t key) {
    if (place >= k) return;
    const int64_t id = vocab_start + static_cast<int64_t>(id_mask - (key & id_mask));
    const float f = Rank<T>::value(static_cast<uint32_t>(key >> id_bits));
    if (results.norm) {
      E::store1(results.values + row * k + place, f);
      results.ids[row * k + place] = id;
    } else {
      out[place] = entry_of(f, id);
    }
    if (place == 0) sh.first = f;
  });
  if (!results.norm)
    for (int i = n + tid; i < k; i += kBlock) out[i] = 0;
  __syncthreads();
  if (tid == 0) {
    total = 0.0;
    for (int w = 0; w < kWaves; ++w) total += sh.wave_s[w];
    if (results.norm) {
      results.norm[row] = log_norm(wm, total, sh.first, c64);
      return;
    }
    out[k] = static_cast<uint64_t>(__float_as_uint(wm)) << 32 |
             __float_as_uint(static_cast<float>(total));
  }
}

constexpr int kMergeBlock = 512;
constexpr int kStaged = 7168;  // entries that a workgroup holds in LDS

// One row's lists (entries of list l at lists + l * list_stride + row * row_stride, in
// order) as one, either a list again (merged) or the results. Staged in LDS, one wave finds
// the k-th entry, then those that reach it are put in order. Up to 1024 are held by the wave
// (16 lists of 20: 5.9 us; as below 7.6). Of more, a lane counts a list's entries that reach a
// key, a search between those of the last two keys (16 rows of 14 lists of 500: 25 us; counted
// by all waves among all entries 54). The last wave takes the normaliser meanwhile. Of more
// lists, or than LDS holds, an entry's place is how many are above it, its own list's by its
// index and the others' by bisection, from memory.
template <typename T>
__global__ __launch_bounds__(kMergeBlock) void top_merge_kernel(
    const uint64_t* __restrict__ lists, int64_t list_stride, int64_t row_stride, int n_lists,
    int k, double c, uint64_t* __restrict__ merged, T* __restrict__ values,
    int64_t* __restrict__ ids, float* __restrict__ norm) {
  extern __shared__ __align__(16) uint64_t stage[];  // n_lists * k entries, or none
  __shared__ __align__(16) uint64_t kept[kMaxK];
  __shared__ uint64_t reached;
  __shared__ int n_kept, n_have;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint64_t* in = lists + row * row_stride;
  const int total = n_lists * k;
  const int most = enough(k, kMaxK);
  if (tid == 0) n_kept = n_have = 0;
  auto put = [&](int rank, uint64_t key) {
    if (rank >= k) return;
    if (merged) {
      merged[row * (k + 1) + rank] = key;
      return;
    }
    Elem<T>::store1(values + row * k + rank,
                    Rank<float>::value(static_cast<uint32_t>(key >> 32)));
    ids[row * k + rank] = 0xffffffffu - static_cast<uint32_t>(key);
  };
  // (maximum, sum) over the lists and the largest entry, a lane each: the last wave's.
  auto normaliser = [&]() {
    uint64_t pair = lane < n_lists ? in[lane * list_stride + k] : 0;
    uint64_t head = lane < n_lists ? in[lane * list_stride] : 0;
    float m = lane < n_lists ? __uint_as_float(static_cast<uint32_t>(pair >> 32)) : kNegHuge;
    for (int l = lane + 64; l < n_lists; l += 64) {
      m = fmaxf(m, __uint_as_float(static_cast<uint32_t>(in[l * list_stride + k] >> 32)));
      head = in[l * list_stride] > head ? in[l * list_stride] : head;
    }
    m = wave_max(m);
    head = wave_max_u64(head);
    double s = 0.0;
    for (int l = lane; l < n_lists; l += 64) {
      if (l > lane) pair = in[l * list_stride + k];
      const double lm = __uint_as_float(static_cast<uint32_t>(pair >> 32));
      s += static_cast<double>(__uint_as_float(static_cast<uint32_t>(pair))) *
           exp2_64((lm - static_cast<double>(m)) * (c * kLog2e64));
    }
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if (lane != 0) return;
    if (merged)
      merged[row * (k + 1) + k] = static_cast<uint64_t>(__float_as_uint(m)) << 32 |
                                  __float_as_uint(static_cast<float>(s));
    else
      norm[row] = log_norm(m, s, Rank<float>::value(static_cast<uint32_t>(head >> 32)), c);
  };
  if (total <= kStaged && n_lists <= 64) {
    constexpr int kAhead = 4;
    for (int i0 = tid; i0 < total; i0 += kAhead * kMergeBlock) {
      uint64_t e[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int i = i0 + a * kMergeBlock < total ? i0 + a * kMergeBlock : total - 1;
        const int l = i / k;
        e[a] = in[l * list_stride + (i - l * k)];
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
        if (i0 + a * kMergeBlock < total) stage[i0 + a * kMergeBlock] = e[a];
    }
    __syncthreads();
    if (wave == 0) {
      const uint64_t* own = stage + (lane < n_lists ? lane : 0) * k;
      // How many of the list's entries, of which `a` do and those from b on do not, reach key.
      auto reach = [&](uint64_t key, int a, int b) {
        while (a < b) {
          const int i = (a + b) / 2;
          if (own[i] >= key) a = i + 1;
          else b = i;
        }
        return a;
      };
      auto over_lists = [&](int v) {  // (of numbers up to kMaxK, a ballot a bit)
        int n = 0;
#pragma unroll
        for (int bit = 0; kMaxK >> bit; ++bit) n += __popcll(__ballot(v >> bit & 1)) << bit;
        return n;
      };
      // The k of some list reach lo (or, of short lists, all that there are).
      uint64_t lo = wave_max_u64(lane < n_lists ? own[k - 1] : 0);
      lo = lo > 0 ? lo : 1;
      int a = 0, b = lane < n_lists ? reach(lo, 0, k) : 0;
      const int all = over_lists(b);
      // More than `most` reach lo, fewer than k some higher key: the middle one of the entries
      // between in the list that has most of them is the next to count.
      const bool small = total <= 1024;
      if (small && all > most) lo = kth_key(stage, total, k, most);
      for (int n = all; !small && n > most;) {
        const uint64_t middle = a < b ? own[(a + b - 1) / 2] : 0;
        const float widest =
            wave_max(middle > lo ? static_cast<float>((b - a) * 64 + lane) : -1.0f);
        if (widest < 0.0f) break;  // (of lists that are not of different ids)
        const int from = __builtin_amdgcn_readfirstlane(static_cast<int>(widest)) & 63;
        const uint64_t key =
            static_cast<uint64_t>(static_cast<uint32_t>(
                __builtin_amdgcn_readlane(static_cast<int>(middle >> 32), from)))
                << 32 |
            static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(middle), from));
        const int at = reach(key, a, b);
        const int count = over_lists(at);
        if (count >= k) {
          lo = key;
          b = at;
          n = count;
        } else {
          a = at;
        }
      }
      if (lane == 0) {
        reached = lo;
        n_have = all;
      }
    } else if (wave == kMergeBlock / 64 - 1) {
      normaliser();
    }
    __syncthreads();
    const uint64_t lo = reached;
    for (int i = tid; i < total; i += kMergeBlock) {
      if (stage[i] < lo) continue;
      const int at = atomicAdd(&n_kept, 1);
      if (at < kMaxK) kept[at] = stage[i];  // (more: of lists that are not of different ids)
    }
    __syncthreads();
    in_order<kMergeBlock, kMaxK>(kept, n_kept < kMaxK ? n_kept : kMaxK, put);
  } else {
    __syncthreads();
    for (int i = tid; i < total; i += kMergeBlock) {
      const int l = i / k, j = i - l * k;
      const uint64_t key = in[l * list_stride + j];
      if (key == 0) continue;
      atomicAdd(&n_have, 1);
      int rank = j;
      for (int o = 0; o < n_lists && rank < k; ++o) {
        if (o == l) continue;
        const uint64_t* p = in + o * list_stride;
        int lo = 0, hi = k;  // entries before lo are above key, from hi on are not
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (p[mid] > key) lo = mid + 1;
          else hi = mid;
        }
        rank += lo;
      }
      put(rank, key);
    }
    if (wave == kMergeBlock / 64 - 1) normaliser();
    __syncthreads();
  }
  for (int i = n_have + tid; i < k; i += kMergeBlock) {  // (more wanted than there are)
    if (merged) {
      merged[row * (k + 1) + i] = 0;
    } else {
      Elem<T>::store1(values + row * k + i, -kInf);
      ids[row * k + i] = -1;
    }
  }
}

int id_bits_of(int64_t v) {
  int bits = 1;
  while ((int64_t{1} << bits) < v) ++bits;
  return bits;
}

// Columns of a slab: the whole row, or, where the rows do not fill the card, as few as
// give a workgroup's place to every slab (64 rows of 128256 bf16, k 20: 17.0 us a call; half
// the places 19.0, twice 20.4), but no fewer than kLeast (a workgroup's own steps take as long
// as reading these: one row of 50257 fp32, k 20: 11.9; of 8192 columns 13.6, of 2048 12.7; eight
// of 100277: 13.6, 15.2 and 18.5; bf16, whose chunk is 8192, would have a little of the wider
// ones: 16 of 128256 16.1, 14.5 and 20.8, 64 of them 17.0, 16.6 and 16.9) and 16 a wanted logit
// (so that the floor holds).
int64_t width_of(int64_t n_rows, int64_t v, int k) {
  const int64_t places = 4 * static_cast<int64_t>(device_cus());
  const int64_t slabs = n_rows > 0 ? places / n_rows : 1;
  if (slabs <= 1) return v;
  const int64_t merged = kStaged / k < 64 ? kStaged / k : 64;  // (from LDS)
  const int64_t most = slabs < merged ? slabs : merged;
  int64_t width = round_up((v + most - 1) / most, 8);
  width = width > kLeast ? width : kLeast;
  return width > 16 * k ? width : 16 * k;
}

int check_rows(int dtype, int64_t n_rows, int64_t v, int k, double temperature) {
  if (dtype != NMCE_F32 && dtype != NMCE_BF16) return NMCE_EINVAL_DTYPE;
  if (n_rows < 0 || n_rows > (int64_t{1} << 22) || v < 1 || v >= (int64_t{1} << 31) || k < 1 ||
      k > kMaxK || !(temperature >= 1e-30 && temperature <= 1e30))  // (its inverse in fp32)
    return NMCE_EINVAL_SHAPE;
  return NMCE_OK;
}

int merge(const uint64_t* lists, int64_t list_stride, int64_t row_stride, int n_lists, int dtype,
          int64_t n_rows, int k, double c, uint64_t* merged, void* values, int64_t* ids,
          float* norm, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(n_rows)), block(kMergeBlock);
  const int64_t total = static_cast<int64_t>(n_lists) * k;
  const unsigned lds = total <= kStaged && n_lists <= 64 ? static_cast<unsigned>(total * 8) : 0;
  if (dtype == NMCE_F32)
    hipLaunchKernelGGL(top_merge_kernel<float>, grid, block, lds, s, lists, list_stride,
                       row_stride, n_lists, k, c, merged, static_cast<float*>(values), ids, norm);
  else
    hipLaunchKernelGGL(top_merge_kernel<uint16_t>, grid, block, lds, s, lists, list_stride,
                       row_stride, n_lists, k, c, merged, static_cast<uint16_t*>(values), ids,
                       norm);
  return launch_status();
}

}  // namespace
}  // namespace nmce

using namespace nmce;

extern "C" {

int64_t nmce_top_workspace_bytes(int64_t n_rows, int64_t vocab_local, int k) {
  if (n_rows < 0 || n_rows > (int64_t{1} << 22) || vocab_local < 1 ||
      vocab_local >= (int64_t{1} << 31) || k < 1 || k > kMaxK)
    return -1;
  const int64_t width = width_of(n_rows, vocab_local, k);
  const int64_t slabs = (vocab_local + width - 1) / width;
  return align256(n_rows * slabs * (k + 1) * 8);
}

int nmce_top_logits(const void* logits, int dtype, int64_t n_rows, int64_t vocab_local, int64_t ld,
                    int64_t vocab_start, int k, double temperature, int64_t* list, void* values,
                    int64_t* ids, float* log_normalizer, void* workspace, int64_t workspace_bytes,
                    void* stream) {
  if (const int st = check_rows(dtype, n_rows, vocab_local, k, temperature)) return st;
  if (ld < vocab_local || vocab_start < 0 || vocab_start >= (int64_t{1} << 31) - vocab_local ||
      (!list && k > vocab_local))
    return NMCE_EINVAL_SHAPE;
  if (n_rows == 0) return NMCE_OK;
  if (!logits || (!list && (!values || !ids || !log_normalizer))) return NMCE_EINVAL_PTR;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == NMCE_F32 ? 4 : 2)) return NMCE_EINVAL_ALIGN;
  if (!workspace || !aligned16(workspace) ||
      workspace_bytes < nmce_top_workspace_bytes(n_rows, vocab_local, k))
    return NMCE_EINVAL_WORKSPACE;
  const int64_t width = width_of(n_rows, vocab_local, k);
  const int64_t slabs = (vocab_local + width - 1) / width;
  const dim3 grid(static_cast<unsigned>(n_rows * slabs));
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint64_t* lists = static_cast<uint64_t*>(workspace);
  const double c = 1.0 / temperature;
  const float c2 = static_cast<float>(1.4426950408889634 * c);
  const int bits = id_bits_of(vocab_local);
  const bool whole = slabs == 1 && !list;
  uint64_t* part = list && slabs == 1 ? reinterpret_cast<uint64_t*>(list) : lists;
  auto run = [&](auto element, auto shape) {
    using T = decltype(element);
    using Shape = decltype(shape);
    hipLaunchKernelGGL((top_kernel<T, Shape>), grid, dim3(Shape::kBlock), 0, s,
                       static_cast<const T*>(logits), ld, vocab_local, vocab_start, slabs, width, k,
                       bits, c2, c, part,
                       Out<T>{static_cast<T*>(values), ids, whole ? log_normalizer : nullptr});
  };
  const bool few = k <= Few::kMost;
  if (dtype == NMCE_F32)
    few ? run(float{}, Few{}) : run(float{}, Many{});
  else
    few ? run(uint16_t{}, Few{}) : run(uint16_t{}, Many{});
  if (const int st = launch_status()) return st;
  if (slabs == 1) return NMCE_OK;
  return merge(lists, k + 1, slabs * (k + 1), static_cast<int>(slabs), dtype, n_rows, k, c,
               reinterpret_cast<uint64_t*>(list), values, ids, log_normalizer, s);
}

int nmce_top_merge(const int64_t* lists, int ranks, int dtype, int64_t n_rows, int k,
                   double temperature, void* values, int64_t* ids, float* log_normalizer,
                   void* stream) {
  if (const int st = check_rows(dtype, n_rows, 1, k, temperature)) return st;
  if (ranks < 1 || ranks > (1 << 20)) return NMCE_EINVAL_TP;
  if (n_rows == 0) return NMCE_OK;
  if (!lists || !values || !ids || !log_normalizer) return NMCE_EINVAL_PTR;
  return merge(reinterpret_cast<const uint64_t*>(lists), n_rows * (k + 1), k + 1, ranks, dtype,
               n_rows, k, 1.0 / temperature, nullptr, values, ids, log_normalizer,
               static_cast<hipStream_t>(stream));
}

}  // extern "C"
