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
// The exponentials' sum rides along; a batch is bounded by the read of the logits.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "nmce.h"
#include "nmce_device.h"

namespace nmce {
namespace {

constexpr int kBlock = 512;
constexpr int kWaves = kBlock / 64;
constexpr int kVecs = 4;      // 16-byte vectors of a thread's chunk
constexpr int kNotes = 2048;  // keys noted at most; cut to k past half of them
constexpr int kLeast = 4096;
constexpr int kFew = 64;
constexpr int kMaxK = NMCE_TOP_MAX_K;
static_assert(2 * kMaxK <= kNotes && kMaxK <= kBlock && kMaxK <= 2 * kBlock, "");
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

// One wave: a key that exactly k of n unique keys (n >= k) reach. Up to 512 are held in
// registers: 14 cycles a key and step, where LDS would answer each in a hundred.
__device__ uint64_t kth_key(const uint64_t* list, int n, int k) {
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
  lo = wave_min_u64(lo);
  hi = wave_max_u64(hi) + 1;
  if (n == k) return lo;
  while (hi - lo > 1) {  // all reach lo, more than k of them; fewer reach hi
    const uint64_t mid = lo + (hi - lo) / 2;  // (above lo, so a 0 does not reach it)
    int c = 0;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) c += __popcll(__ballot(held[j] >= mid));
    for (int i = kHeld * 64; i < n; i += 64)
      c += __popcll(__ballot(i + lane < n && list[i + lane] >= mid));
    if (c == k) return mid;
    if (c > k) lo = mid;
    else hi = mid;
  }
  return lo;
}

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

// 16 bytes at any element's alignment (rows of odd widths start anywhere).
__device__ __forceinline__ u32x4 load16(const void* p) {
  u32x4 v;
  memcpy(&v, p, 16);
  return v;
}

struct Shared {
  uint64_t notes[kNotes];
  uint64_t kept[kMaxK];
  uint64_t key;    // what the k largest reach
  uint32_t floor;  // of the first chunk
  float first;     // the largest logit
  int n, n_kept, counts[2];
  float wave_m[kWaves];
  double wave_s[kWaves];
};

// All but the k largest notes go (k <= n); every thread calls it, behind a barrier.
__device__ void cut_notes(Shared& sh, int n, int k) {
  if (threadIdx.x < 64) {
    const uint64_t key = kth_key(sh.notes, n, k);
    if (threadIdx.x == 0) {
      sh.key = key;
      sh.n_kept = 0;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kBlock)
    if (sh.notes[i] >= sh.key) sh.kept[atomicAdd(&sh.n_kept, 1)] = sh.notes[i];
  __syncthreads();
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
template <typename T>
__global__ __launch_bounds__(kBlock, 8) void top_kernel(const T* __restrict__ x, int64_t ld,
                                                        int64_t v, int64_t vocab_start,
                                                        int64_t slabs, int64_t width, int k,
                                                        int id_bits, float c, double c64,
                                                        uint64_t* __restrict__ lists,
                                                        Out<T> results) {
  using E = Elem<T>;
  constexpr int EPV = E::kPerVec;
  constexpr uint32_t kChunk = kBlock * kVecs * EPV;
  __shared__ Shared sh;
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
  auto load_chunk = [&](uint32_t base, u32x4 (&w)[kVecs]) {
    const uint32_t col = column_of(base, 0);
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      if (col + i * kBlock * EPV + EPV <= end) w[i] = load16(xr + col + i * kBlock * EPV);
    if (base + kChunk <= end) return;
    // The vector that the row ends in, and none behind it.
    constexpr uint32_t kNone = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;  // -inf
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const uint32_t c0 = col + i * kBlock * EPV;
      if (c0 + EPV > end) {
        w[i] = u32x4{kNone, kNone, kNone, kNone};
        if (c0 < end) {
          float f[EPV];
#pragma unroll
          for (int e = 0; e < EPV; ++e) f[e] = c0 + e < end ? E::load1(xr + c0 + e) : -kInf;
          w[i] = E::pack(f);
        }
      }
    }
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
  for (uint32_t base = 0; base < end; base += kChunk) {
    load_chunk(base, cur);
    if (base == 0) {
      // The floor: from the maxima of a thread's even and odd vectors.
      uint32_t* maxima = reinterpret_cast<uint32_t*>(sh.notes);
      uint32_t tops[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t top = 0;
#pragma unroll
        for (int i = h; i < kVecs; i += 2) {
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
        tops[h] = top;
      }
      // One maximum a thread does for few.
      const bool two = k > kFew;
      maxima[tid] = two || tops[0] > tops[1] ? tops[0] : tops[1];
      if (two) maxima[kBlock + tid] = tops[1];
      __syncthreads();
      if (wave == 0) {
        const uint32_t r = two ? floor_rank<2 * kBlock>(maxima, k) : floor_rank<kBlock>(maxima, k);
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
      cut_notes(sh, n, k);
      for (int i = tid; i < k; i += kBlock) sh.notes[i] = sh.kept[i];
      if (tid == 0) sh.n = k;
      n = keys = k;
      // Later columns of the same value come behind: only what is above it counts.
      floor = Rank<T>::value(static_cast<uint32_t>(sh.key >> id_bits));
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
  const int have = n < k ? n : k;
  to_keys(keys, n);
  if (n > k) {
    cut_notes(sh, n, k);
  } else {
    for (int i = tid; i < n; i += kBlock) sh.kept[i] = sh.notes[i];
    __syncthreads();
  }
  uint64_t* out = lists + blockIdx.x * static_cast<int64_t>(k + 1);
  if (tid < have) {
    const uint64_t key = sh.kept[tid];
    int rank = 0;
    for (int i = 0; i < have; ++i) rank += sh.kept[i] > key;
    const int64_t id = vocab_start + static_cast<int64_t>(id_mask - (key & id_mask));
    const float f = Rank<T>::value(static_cast<uint32_t>(key >> id_bits));
    if (results.norm) {
      E::store1(results.values + row * k + rank, f);
      results.ids[row * k + rank] = id;
    } else {
      out[rank] = entry_of(f, id);
    }
    if (rank == 0) sh.first = f;
  } else if (tid < k) {
    out[tid] = 0;
  }
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
constexpr int kCounted = 1024;  // entries up to which a place is found by counting
constexpr int kStageBytes = 64 * 1024;

// One row's lists (entries of list l at lists + l * list_stride + row * row_stride), each
// in order, as one: an entry's place is how many are above it, its own list's by its index
// and the others' by bisection. Either the list again (merged) or the results.
template <typename T>
__global__ __launch_bounds__(kMergeBlock) void top_merge_kernel(
    const uint64_t* __restrict__ lists, int64_t list_stride, int64_t row_stride, int n_lists,
    int k, bool staged, double c, uint64_t* __restrict__ merged, T* __restrict__ values,
    int64_t* __restrict__ ids, float* __restrict__ norm) {
  extern __shared__ uint64_t stage[];
  const int64_t row = blockIdx.x;
  const uint64_t* in = lists + row * row_stride;
  const int total = n_lists * k;
  if (staged) {
    for (int i = threadIdx.x; i < n_lists * (k + 1); i += kMergeBlock) {
      const int l = i / (k + 1);
      stage[i] = in[l * list_stride + (i - l * (k + 1))];
    }
    __syncthreads();
    in = stage;
    list_stride = k + 1;
  }
  for (int i = threadIdx.x; i < total; i += kMergeBlock) {
    const int l = i / k, j = i - l * k;
    const uint64_t key = in[l * list_stride + j];
    int rank = j;
    if (key == 0) continue;  // (fewer entries than k: the places behind are filled below)
    if (staged && total <= kCounted) {
      // Few entries are counted one by one: no read waits for another.
      rank = 0;
      for (int o = 0; o < n_lists * (k + 1); o += k + 1)
#pragma unroll 4
        for (int e = 0; e < k; ++e) rank += stage[o + e] > key;
    } else for (int o = 0; o < n_lists && rank < k; ++o) {
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
    if (rank < k) {
      if (merged) {
        merged[row * (k + 1) + rank] = key;
      } else {
        const float f = Rank<float>::value(static_cast<uint32_t>(key >> 32));
        Elem<T>::store1(values + row * k + rank, f);
        ids[row * k + rank] = 0xffffffffu - static_cast<uint32_t>(key);
      }
    }
  }
  if (threadIdx.x < 64) {
    // (maximum, sum) over the lists, a lane each.
    float m = kNegHuge;
    int have = 0;
    for (int l = threadIdx.x; l < n_lists; l += 64) {
      m = fmaxf(m, __uint_as_float(static_cast<uint32_t>(in[l * list_stride + k] >> 32)));
      for (int j = k; j > 0; --j)
        if (in[l * list_stride + j - 1] != 0) {
          have += j;
          break;
        }
    }
    m = wave_max(m);
    double s = 0.0;
    for (int l = threadIdx.x; l < n_lists; l += 64) {
      const uint64_t pair = in[l * list_stride + k];
      const double lm = __uint_as_float(static_cast<uint32_t>(pair >> 32));
      s += static_cast<double>(__uint_as_float(static_cast<uint32_t>(pair))) *
           (lm == m ? 1.0 : exp((lm - static_cast<double>(m)) * c));
    }
    for (int d = 32; d > 0; d >>= 1) {
      s += __shfl_xor(s, d);
      have += __shfl_xor(have, d);
    }
    uint64_t first = 0;
    for (int l = threadIdx.x; l < n_lists; l += 64)
      first = in[l * list_stride] > first ? in[l * list_stride] : first;
    first = wave_max_u64(first);
    if (merged) {
      for (int i = have + threadIdx.x; i < k; i += 64) merged[row * (k + 1) + i] = 0;
      if (threadIdx.x == 0)
        merged[row * (k + 1) + k] = static_cast<uint64_t>(__float_as_uint(m)) << 32 |
                                    __float_as_uint(static_cast<float>(s));
    } else {
      for (int i = have + threadIdx.x; i < k; i += 64) {  // (more wanted than there are)
        Elem<T>::store1(values + row * k + i, -kInf);
        ids[row * k + i] = -1;
      }
    }
    if (!merged && threadIdx.x == 0)
      norm[row] = log_norm(m, s, Rank<float>::value(static_cast<uint32_t>(first >> 32)), c);
  }
}

// (A temperature past these is merely very high or very low.)
double inverse(double temperature) { return fmin(fmax(1.0 / temperature, 1e-30), 1e30); }

int id_bits_of(int64_t v) {
  int bits = 1;
  while ((int64_t{1} << bits) < v) ++bits;
  return bits;
}

// Columns of a slab: the whole row, or, where the rows do not fill the card, as few as
// give a workgroup's place to every slab, but no fewer than kLeast (a workgroup's own
// steps take as long as reading these) and 16 a wanted logit (so that the floor holds).
int64_t width_of(int64_t n_rows, int64_t v, int k) {
  const int64_t places = 4 * static_cast<int64_t>(device_cus());
  const int64_t slabs = n_rows > 0 ? places / n_rows : 1;
  if (slabs <= 1) return v;
  int64_t width = round_up((v + slabs - 1) / slabs, 8);
  width = width > kLeast ? width : kLeast;
  return width > 16 * k ? width : 16 * k;
}

int check_rows(int dtype, int64_t n_rows, int64_t v, int k, double temperature) {
  if (dtype != NMCE_F32 && dtype != NMCE_BF16) return NMCE_EINVAL_DTYPE;
  if (n_rows < 0 || n_rows > (int64_t{1} << 22) || v < 1 || v >= (int64_t{1} << 31) || k < 1 ||
      k > kMaxK || !(temperature > 0.0 && temperature < HUGE_VAL))
    return NMCE_EINVAL_SHAPE;
  return NMCE_OK;
}

int merge(const uint64_t* lists, int64_t list_stride, int64_t row_stride, int n_lists, int dtype,
          int64_t n_rows, int k, double c, uint64_t* merged, void* values, int64_t* ids,
          float* norm, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(n_rows)), block(kMergeBlock);
  const int64_t bytes = static_cast<int64_t>(n_lists) * (k + 1) * 8;
  const bool staged = bytes <= kStageBytes;
  const unsigned lds = staged ? static_cast<unsigned>(bytes) : 0;
  if (dtype == NMCE_F32)
    hipLaunchKernelGGL(top_merge_kernel<float>, grid, block, lds, s, lists, list_stride,
                       row_stride, n_lists, k, staged, c, merged, static_cast<float*>(values), ids,
                       norm);
  else
    hipLaunchKernelGGL(top_merge_kernel<uint16_t>, grid, block, lds, s, lists, list_stride,
                       row_stride, n_lists, k, staged, c, merged, static_cast<uint16_t*>(values),
                       ids, norm);
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
  const dim3 grid(static_cast<unsigned>(n_rows * slabs)), block(kBlock);
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint64_t* lists = static_cast<uint64_t*>(workspace);
  const double c = inverse(temperature);
  const float c2 = static_cast<float>(1.4426950408889634 * c);
  const int bits = id_bits_of(vocab_local);
  const bool whole = slabs == 1 && !list;
  uint64_t* part = list && slabs == 1 ? reinterpret_cast<uint64_t*>(list) : lists;
  if (dtype == NMCE_F32)
    hipLaunchKernelGGL(top_kernel<float>, grid, block, 0, s, static_cast<const float*>(logits), ld,
                       vocab_local, vocab_start, slabs, width, k, bits, c2, c, part,
                       Out<float>{static_cast<float*>(values), ids, whole ? log_normalizer : nullptr});
  else
    hipLaunchKernelGGL(top_kernel<uint16_t>, grid, block, 0, s,
                       static_cast<const uint16_t*>(logits), ld, vocab_local, vocab_start, slabs,
                       width, k, bits, c2, c, part,
                       Out<uint16_t>{static_cast<uint16_t*>(values), ids,
                                     whole ? log_normalizer : nullptr});
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
               n_rows, k, inverse(temperature), nullptr, values, ids, log_normalizer,
               static_cast<hipStream_t>(stream));
}

}  // extern "C"
