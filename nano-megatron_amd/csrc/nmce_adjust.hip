// Penalties for repeated tokens, biases of single ids and masks of allowed ids, on
// the logits of a vocabulary shard, for gfx950. For row i of a sequence (its next
// token's logits, and those after its first i drafted tokens), with count = how
// often an id is among the sequence's output tokens and its first i drafts:
//
//   id in the prompt or count > 0:   x <- x / r where x > 0, else x r
//   count > 0:                       x <- x - f count - p
//   then x + the id's biases (in their order), and -inf where it is not allowed.
//
// A workgroup holds one sequence's counts of a slab of the vocabulary in LDS, so a list is
// read once by every slab (from the L2 after the first) and nothing of the vocabulary's size
// is kept in memory; the counts are integers, whose order does not matter. Then the rows go
// by, 16 bytes a load and under their mask; the few elements with a count are formed in 64
// bits and rounded once, in the registers, before the store. What bounds a batch is one
// read and one write of the logits; in place only vectors with something to change move.
// 24 x 9 rows of 151936 bf16, 1250 listed ids, masked: 29 us (4.7 TB/s with the masks; the
// counts, before the first store, are what is left to 21), in place 26; 64 x 1 of 128256: 16,
// in place 16; one of 50257 fp32: 6, a launch and three dependent reads; 8 of 100277 fp32 with
// 139264 ids and 300 biases each: 24, in place 25, of which the lists take 12 (a compute unit's
// 64 bytes a cycle from its L2: 7) and the biases 8.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <type_traits>

#include "nmce.h"
#include "nmce_device.h"

namespace nmce {
namespace {

constexpr int kSlab = 8192;               // ids of a workgroup
constexpr int kBiases = 512;              // biases of a slab that are summed by id in LDS
constexpr float kInf = __builtin_huge_valf();

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

// A slab's counts in LDS, of 32 bits or, where the lists are shorter than 2^14, of 16 (twice
// the workgroups fit a compute unit: 24 x 9 rows of 151936 bf16, then 38 -> 33 us). The upper two
// bits tell that the id is in the prompt and that it has a bias.
template <bool kNarrow>
struct Counts {
  static constexpr int kBits = kNarrow ? 16 : 32, kPer = 32 / kBits;
  static constexpr uint32_t kPrompt = 1u << (kBits - 1), kBiased = 1u << (kBits - 2),
                            kTimes = kBiased - 1;
  static constexpr int kWords = kSlab / kPer;
  uint32_t* words;
  __device__ __forceinline__ static int shift(int s) { return kNarrow ? (s & 1) * 16 : 0; }
  // (A plain store, before any count: many lanes name an id at once.)
  __device__ __forceinline__ void in_prompt(int s) {
    if constexpr (kNarrow) reinterpret_cast<uint16_t*>(words)[s] = kPrompt;
    else words[s] = kPrompt;
  }
  __device__ __forceinline__ void once_more(int s) { atomicAdd(words + s / kPer, 1u << shift(s)); }
  // Whether it had one before.
  __device__ __forceinline__ bool with_bias(int s) {
    return atomicOr(words + s / kPer, kBiased << shift(s)) >> shift(s) & kBiased;
  }
  __device__ __forceinline__ uint32_t at(int s) const {
    return kNarrow ? words[s / kPer] >> shift(s) & 0xffffu : words[s];
  }
  // Of kVec places from s on (a multiple), those with a count, the first in bit 0.
  template <int kVec>
  __device__ __forceinline__ uint32_t some(int s) const {
    constexpr uint32_t kAny = kPrompt | kTimes;
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < kVec; e += 4) {
      if constexpr (kNarrow) {
        const uint2 w = *reinterpret_cast<const uint2*>(words + (s + e) / 2);
        bits |= (w.x & kAny ? 1u << e : 0u) | (w.x & kAny << 16 ? 2u << e : 0u) |
                (w.y & kAny ? 4u << e : 0u) | (w.y & kAny << 16 ? 8u << e : 0u);
      } else {
        const u32x4 w = *reinterpret_cast<const u32x4*>(words + s + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) bits |= w[i] & kAny ? 1u << (e + i) : 0u;
      }
    }
    return bits;
  }
};

struct Penalties {
  double r, f, p, inv;  // inv: 1 / r
  __device__ __forceinline__ bool none() const { return r == 1.0 && f == 0.0 && p == 0.0; }
  // x / r, x > 0, by the reciprocal and one correction (an infinite quotient, of an infinite x
  // or of an r whose reciprocal or quotient passes 64 bits, has none to take).
  __device__ __forceinline__ double quotient(double x) const {
    const double q = x * inv, e = fma(-q, r, x);
    return fabs(e) < static_cast<double>(kInf) ? fma(e, inv, q) : q;
  }
  template <typename Count>
  __device__ __forceinline__ double on(double x, uint32_t word, const Count&) const {
    const uint32_t times = word & Count::kTimes;
    if ((word & (Count::kPrompt | Count::kTimes)) && r != 1.0) x = x > 0.0 ? quotient(x) : x * r;
    if (times) x = x - f * static_cast<double>(times) - p;
    return x;
  }
};

__device__ __forceinline__ double of_sequence(const float* each, double all, int64_t b) {
  return each ? static_cast<double>(each[b]) : all;
}

// 16 bytes at any element's alignment, streamed.
typedef u32x4 anywhere __attribute__((aligned(2)));
__device__ __forceinline__ u32x4 load16(const void* p) {
  return __builtin_nontemporal_load(static_cast<const anywhere*>(p));
}
__device__ __forceinline__ void store16(void* p, const u32x4& v) {
  __builtin_nontemporal_store(v, static_cast<anywhere*>(p));
}

// Element e of a vector, by its bits.
template <typename T>
__device__ __forceinline__ uint32_t element(const u32x4& v, int e) {
  constexpr int kPer = 4 / sizeof(T);
  const int d = e / kPer;
  const uint32_t w = d < 2 ? (d == 0 ? v[0] : v[1]) : (d == 2 ? v[2] : v[3]);
  return kPer == 1 ? w : w >> (e % kPer * 16) & 0xffffu;
}
template <typename T>
__device__ __forceinline__ void set_element(u32x4& v, int e, uint32_t bits) {
  constexpr int kPer = 4 / sizeof(T);
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const uint32_t keep = kPer == 1 ? 0u : e % kPer ? 0x0000ffffu : 0xffff0000u;
    if (e / kPer == d) v[d] = (v[d] & keep) | bits << (kPer == 1 ? 0 : e % kPer * 16);
  }
}

// -inf for the elements that have no bit (the first's is bit 0). The others keep their bits,
// which a signalling NaN does not in a conversion.
template <typename T>
__device__ __forceinline__ void mask_out(u32x4& v, uint32_t bits) {
  // All ones where bit i is set.
  auto spread = [&](int i) {
    return static_cast<uint32_t>(static_cast<int32_t>(bits << (31 - i)) >> 31);
  };
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const uint32_t keep = sizeof(T) == 4 ? spread(d)
                                         : (spread(2 * d) & 0xffffu) |
                                               (spread(2 * d + 1) & 0xffff0000u);
    v[d] = (v[d] & keep) | ((sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u) & ~keep);
  }
}

// Row `row` of sequence b, slab `slab` of the vocabulary.
template <typename T, int kBlock, bool kInPlace, bool kNarrow>
__global__ __launch_bounds__(kBlock, kNarrow && sizeof(T) == 2 ? 6 : 4) void adjust_kernel(
    nmce_adjust_batch a, int64_t slabs) {
  using E = Elem<T>;
  constexpr int kVec = E::kPerVec;
  constexpr int kEach = kSlab / kBlock / kVec;  // vectors of a thread
  constexpr uint32_t kAll = (1u << kVec) - 1;
  static_assert(kEach >= 1, "");
  using Count = Counts<kNarrow>;
  __shared__ __align__(16) uint32_t count_words[Count::kWords];
  Count count{count_words};
  // The slab's biases; where an id comes twice, its sum at the first place, kSlab at others.
  __shared__ __align__(16) uint16_t bias_place[kBiases];
  __shared__ double bias_sum[kBiases];
  __shared__ int repeated, wave_n[kBlock / 64];
  const int tid = threadIdx.x;
  // Neighbours in this order, which read the same lists, share an XCD and its L2 (workgroups go
  // to the eight in turn): 8 rows with 139264 ids each 28 -> 25 us.
  const uint32_t xcd = blockIdx.x % 8, eighth = gridDim.x / 8, over = gridDim.x % 8;
  const int64_t turn = xcd * eighth + (xcd < over ? xcd : over) + blockIdx.x / 8;
  const int64_t br = turn / slabs, slab = turn - br * slabs;
  const int64_t b = br / a.rows, row = br - b * a.rows;
  const int64_t c0 = slab * kSlab;
  const int64_t left = a.vocab_local - c0;
  const int width = static_cast<int>(left < kSlab ? left : kSlab);
  const int64_t g0 = a.vocab_start + c0;  // the slab's first global id
  const T* x = static_cast<const T*>(a.logits) + b * a.logits_batch_stride +
               row * a.logits_row_stride + c0;
  T* y = static_cast<T*>(a.out) + b * a.out_batch_stride + row * a.out_row_stride + c0;
  const uint32_t* words =
      a.allowed ? a.allowed + b * a.allowed_batch_stride + row * a.allowed_row_stride : nullptr;
  // The first column of the thread's vector k. (Opaque to the compiler, which would keep
  // what it can compute from each of them in registers through the rows.)
  auto column_of = [&](int k) {
    int t = tid * kVec;
    asm volatile("" : "+v"(t));
    return t + k * kBlock * kVec;
  };

  // The vectors and their masks are on their way while the lists are counted.
  u32x4 v[kEach];
  uint32_t lo[kEach], hi[kEach];  // the words with the vectors' mask bits
  if (words) {
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      // (Past the vocabulary its last word again: no load waits for a condition.)
      const int64_t g = g0 + column_of(k), end = a.vocab_total - 1;
      lo[k] = words[(g < end ? g : end) >> 5];
      hi[k] = words[(g + kVec - 1 < end ? g + kVec - 1 : end) >> 5];
    }
  }
  if (!kInPlace && width == kSlab) {
#pragma unroll
    for (int k = 0; k < kEach; ++k) v[k] = load16(x + column_of(k));
  } else if (!kInPlace) {
#pragma unroll
    for (int k = 0; k < kEach; ++k)
      if (column_of(k) + kVec <= width) v[k] = load16(x + column_of(k));
  }

  const int64_t* bias_ids = a.bias_ids + b * a.bias_ids_stride;
  const float* bias = a.bias + b * a.bias_stride;
  int64_t first_id = -1;
  float first_bias = 0.0f;
  if (a.n_bias > 0) {
    const int64_t j = tid < a.n_bias ? tid : a.n_bias - 1;
    first_id = bias_ids[j];
    first_bias = bias[j];
  }

  for (int i = tid * 4; i < Count::kWords; i += kBlock * 4)
    *reinterpret_cast<u32x4*>(count_words + i) = u32x4{0u, 0u, 0u, 0u};
  if (tid == 0) repeated = 0;
  __syncthreads();

  Penalties pen;
  pen.r = of_sequence(a.repetition, a.repetition_all, b);
  pen.f = of_sequence(a.frequency, a.frequency_all, b);
  pen.p = of_sequence(a.presence, a.presence_all, b);
  if (!(pen.r > 0.0 && pen.r < static_cast<double>(kInf))) pen.r = 1.0;
  pen.inv = 1.0 / pen.r;
  const bool counted = !pen.none();
  // An id's place in the slab, or kSlab and above.
  auto place = [&](int64_t id) {
    const uint32_t s = static_cast<uint32_t>(id) - static_cast<uint32_t>(g0);
    return id >> 32 == 0 && s < static_cast<uint32_t>(width) ? static_cast<int>(s) : kSlab;
  };
  // Two ids a load and kAhead loads of a thread on their way at once (the lists come from the
  // L2, a microsecond away): 8 rows of 100277 fp32, 139264 ids each, 36 us with one id a load,
  // 28 with two and the prompt stored plainly.
  auto count_list = [&](const int64_t* __restrict__ list, int64_t n, auto prompt) {
    typedef uint64_t two_ids __attribute__((ext_vector_type(2), aligned(8)));
    constexpr int kAhead = kBlock == 1024 ? 4 : 2;
    const two_ids* ids = reinterpret_cast<const two_ids*>(list);
    auto take = [&](uint64_t id) {
      const uint64_t s = id - static_cast<uint64_t>(g0);
      if (s >= static_cast<uint64_t>(width)) return;
      if constexpr (decltype(prompt)::value) count.in_prompt(static_cast<int>(s));
      else count.once_more(static_cast<int>(s));
    };
    const int64_t pairs = n / 2;
    int64_t j0 = tid;
    for (; j0 + (kAhead - 1) * kBlock < pairs; j0 += kBlock * kAhead) {
      two_ids id[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) id[i] = ids[j0 + i * kBlock];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        take(id[i][0]);
        take(id[i][1]);
      }
    }
    if (j0 < pairs) {
      two_ids id[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        // (The last ones again past the end: a load under a condition would be waited for
        // before the next.)
        const int64_t j = j0 + i * kBlock;
        id[i] = ids[j < pairs ? j : pairs - 1];
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (j0 + i * kBlock >= pairs) break;
        take(id[i][0]);
        take(id[i][1]);
      }
    }
    if ((n & 1) && tid == kBlock - 1) take(static_cast<uint64_t>(list[n - 1]));
  };
  if (counted) {
    if (pen.r != 1.0 && a.n_prompt > 0) {
      count_list(a.prompt + b * a.prompt_stride, a.n_prompt, std::true_type{});
      __syncthreads();
    }
    count_list(a.output + b * a.output_stride, a.n_output, std::false_type{});
    count_list(a.drafts + b * a.drafts_stride, row, std::false_type{});
  }
  // The slab's biases in their order (the first of them were asked for at the start).
  int n_here = 0;
  for (int64_t j0 = 0; j0 < a.n_bias; j0 += kBlock) {
    const int64_t j = j0 + tid;
    if (j0 > 0 && j < a.n_bias) {
      first_id = bias_ids[j];
      first_bias = bias[j];
    }
    const int s = j < a.n_bias ? place(first_id) : kSlab;
    if (s < kSlab && count.with_bias(s)) repeated = 1;
    const uint64_t here = __ballot(s < kSlab);
    if ((tid & 63) == 0) wave_n[tid >> 6] = __popcll(here);
    __syncthreads();
    int at = n_here + __popcll(here & ((uint64_t{1} << (tid & 63)) - 1));
    for (int w = 0; w < kBlock / 64; ++w) {
      if (w < tid >> 6) at += wave_n[w];
      n_here += wave_n[w];
    }
    if (tid < 8 && n_here + tid < kBiases) bias_place[n_here + tid] = kSlab;
    if (s < kSlab && at < kBiases) {
      bias_place[at] = static_cast<uint16_t>(s);
      bias_sum[at] = first_bias;
    }
    __syncthreads();
  }
  __syncthreads();
  const bool in_lds = n_here <= kBiases;  // (more than that: from memory again)
  const bool apart = repeated != 0;
  if (in_lds && apart) {
    // All biases of an id at the first of its entries: 300 with a few ids twice, over 100277
    // fp32, 65 -> 36 us.
    double sum[(kBiases + kBlock - 1) / kBlock];
    bool mine[(kBiases + kBlock - 1) / kBlock];
#pragma unroll
    for (int r = 0; r < (kBiases + kBlock - 1) / kBlock; ++r) {
      const int t = r * kBlock + tid;
      mine[r] = t < n_here;
      sum[r] = 0.0;
      if (!mine[r]) continue;
      const uint32_t s = bias_place[t];
      for (int i = 0; i < n_here && mine[r]; i += 8) {  // (what lies behind them is kSlab)
        const u32x4 w = *reinterpret_cast<const u32x4*>(bias_place + i);
        uint32_t same = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          same |= (w[e / 2] >> (e % 2 * 16) & 0xffffu) == s ? 1u << e : 0u;
        if (i < t && (same & ((1u << (t - i < 8 ? t - i : 8)) - 1))) mine[r] = false;
        for (; same; same &= same - 1) sum[r] += bias_sum[i + __builtin_ctz(same)];
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < (kBiases + kBlock - 1) / kBlock; ++r) {
      const int t = r * kBlock + tid;
      if (t < n_here) {
        if (!mine[r]) bias_place[t] = kSlab;
        bias_sum[t] = sum[r];
      }
    }
    __syncthreads();
  }

  auto allowed = [&](int s) {
    return !words || (words[(g0 + s) >> 5] >> ((g0 + s) & 31) & 1u);
  };
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int c = column_of(k);
    if (c + kVec > width) break;
    // The vector's allowed ids, the first in bit 0.
    const uint64_t both = static_cast<uint64_t>(hi[k]) << 32 | lo[k];
    const uint32_t bits =
        words ? static_cast<uint32_t>(both >> ((g0 + c) & 31)) & kAll : kAll;
    // Those with a count, and allowed.
    uint32_t touched = counted ? count.template some<kVec>(c) & bits : 0u;
    if (kInPlace) {
      if (bits == kAll && touched == 0) continue;  // nothing to write
      if (bits != 0) v[k] = load16(x + c);
    }
    for (; touched; touched &= touched - 1) {  // (with a bias: formed by that, below)
      const int e = __builtin_ctz(touched);
      const uint32_t was = element<T>(v[k], e);
      const float f = sizeof(T) == 4 ? __uint_as_float(was)
                                     : bf16_to_f32(static_cast<uint16_t>(was));
      T to;
      const uint32_t word = count.at(c + e);
      if (word & Count::kBiased) continue;
      store_rounded(&to, pen.on(static_cast<double>(f), word, count));
      uint32_t is;
      if constexpr (sizeof(T) == 4) is = __float_as_uint(to);
      else is = to;
      set_element<T>(v[k], e, is);
    }
    if (bits != kAll) mask_out<T>(v[k], bits);
    store16(y + c, v[k]);
  }
  // The shard's last elements, of no whole vector.
  const int c = width / kVec * kVec + tid;
  if (c < width) {
    const uint32_t word = count.at(c);
    if (!allowed(c)) E::store1(y + c, -kInf);
    else if (!(word & Count::kBiased) && word)
      store_rounded(y + c, pen.on(static_cast<double>(E::load1(x + c)), word, count));
    else if (!kInPlace) y[c] = x[c];
  }
  if (n_here > 0) {
    // The stores have reached the memory before any thread of the workgroup
    // stores an element over them.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    auto put = [&](int s, double add) {
      if (s < kSlab && allowed(s))
        store_rounded(y + s, pen.on(static_cast<double>(E::load1(x + s)), count.at(s), count) +
                                  add);
    };
    if (in_lds) {
      for (int t = tid; t < n_here; t += kBlock) put(bias_place[t], bias_sum[t]);
    } else {
      for (int64_t j = tid; j < a.n_bias; j += kBlock) {
        const int64_t id = bias_ids[j];
        const int s = place(id);
        if (s >= kSlab) continue;
        double add = bias[j];
        if (apart) {
          // The first entry of an id adds all of them, in their order. (The whole list from
          // memory for each entry: milliseconds, where one id of so many comes again.)
          bool mine = true;
          for (int64_t i = 0; i < j && mine; ++i) mine = bias_ids[i] != id;
          if (!mine) continue;
          for (int64_t i = j + 1; i < a.n_bias; ++i)
            if (bias_ids[i] == id) add += static_cast<double>(bias[i]);
        }
        put(s, add);
      }
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
  if (a->batch > (int64_t{1} << 23) || a->batch * a->rows > (int64_t{1} << 23) ||
      a->batch * a->rows * slabs > (int64_t{1} << 23))
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
  // A workgroup for a slab of every row, drafts' too, which counts the lists again (24 x 9 rows
  // of 151936 bf16: with 1250 ids 29 us, by nine rows each 62; with 64250 82 and 134).
  const dim3 grid(static_cast<unsigned>(a->batch * a->rows * slabs));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto run = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, g, slabs);
  };
  // Where there is no workgroup for every compute unit, 1024 threads share a slab (8 rows with
  // 139264 ids each: 25 us, by 256 threads 54; 64 rows of 128256, enough workgroups: 24 and 16);
  // with lists longer than a slab, two (30 rows of 128256, 30250 ids: 17 us and 23; 450: 11
  // and 10).
  const int64_t lists = a->n_prompt + a->n_output;
  const bool few = static_cast<int64_t>(grid.x) <= (lists > kSlab ? 2 : 1) * device_cus();
  const bool narrow = a->n_output + a->rows <= static_cast<int64_t>(Counts<true>::kTimes);
  auto pick = [&](auto element, auto in_place_, auto narrow_) {
    using T = decltype(element);
    constexpr bool kInPlace = decltype(in_place_)::value, kNarrow = decltype(narrow_)::value;
    few ? run(adjust_kernel<T, 1024, kInPlace, kNarrow>, 1024)
        : run(adjust_kernel<T, 256, kInPlace, kNarrow>, 256);
  };
  auto pick_counts = [&](auto element, auto in_place_) {
    narrow ? pick(element, in_place_, std::true_type{}) : pick(element, in_place_, std::false_type{});
  };
  auto pick_place = [&](auto element) {
    in_place ? pick_counts(element, std::true_type{}) : pick_counts(element, std::false_type{});
  };
  a->dtype == NMCE_F32 ? pick_place(float{}) : pick_place(uint16_t{});
  return launch_status();
}

}  // extern "C"
