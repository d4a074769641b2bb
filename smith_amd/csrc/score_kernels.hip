// score_kernels.hip -- gfx950 kernels of smith_logprobs (smith_score.hsaco): log
// probabilities of given tokens, entropy and top alternatives of rows of logits.
//
// Of a row x with m = max x, d = x - m, l = sum e^d and s = sum e^d d:
//   log p(t) = d_t - log l,   entropy = -sum p log p = log l - s / l,
// in one pass: a thread keeps (m, l, s) of what it has seen, and when m grows to M
//   l' = e^(m - M) l,   s' = e^(m - M) (s + (m - M) l).
//
// The top k are found in the same pass.  An element is a 64-bit key: its value,
// ordered as a whole number, above the complement of its place, so that keys are
// all different and the larger one is the larger value or, of equal ones, the
// lower place.  A wave keeps the 64 best of its elements sorted over its lanes;
// an element goes in if it is above the k-th of each of the workgroup's waves, which
// after a few thousand elements is rare, so that the pass costs a comparison with
// the maximum of 16.  Lists are
// joined by bitonic merges: the result does not depend on who comes first.
//
// Bound by memory where few are wanted of long f32 rows: 900 of 131072, 472 MB, 83 us
// without top ones (5.7 TB/s; a large copy: 5.2), 90 with 8, 138 with 64; of bf16 logits
// by the operations, 48, 70 and 136.  Short rows by the first lists and their merges: one
// row of 32000 4.8 us without top ones, 8.6 with 8, 12.8 with 64.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lanes.h"
#include "paged.h"
#include "paged_dev.h"

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_2 __attribute__((ext_vector_type(4), aligned(2)));

#define LOG2E 1.44269504088896341f
#define THREADS SCORE_THREADS
#define WAVES (SCORE_THREADS / 64)
// Lanes whose elements go into a list together, sorted first (900 rows of 131072 f32, top
// 64, 138 us, 150 with 6, 138 with 24; 256 rows of 32000, top 20, 22.1, 22.5 and 22.6)
#define MANY 12
// Top ones for which one sorted round is enough, the rest of a chunk going in one by one (57
// rows of 50003, top 20: 14.2 us, 15.1 with rounds while they are many; top 64: 23 and 18)
#define FEW 24
#define PER 16                    // elements of a thread to a chunk
#define CHUNK SCORE_WAVE_CHUNK    // of a wave

struct LogitsF32 {
  typedef float T;
  static constexpr uint32_t WIDTH = 4;  // elements to a 16-byte load
  static __device__ __forceinline__ void load(const T* p, float* x) {
    const f32x4_any v = *(const f32x4_any*)p;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = v[i];
  }
  static __device__ __forceinline__ float up(T v) { return v; }
};
template <class T_>
struct Logits16 {
  typedef T_ T;
  static constexpr uint32_t WIDTH = 8;
  static __device__ __forceinline__ void load(const T* p, float* x) {
    const u32x4_2 v = *(const u32x4_2*)p;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = (float)__builtin_bit_cast(T, (uint16_t)v[i]);
      x[2 * i + 1] = (float)__builtin_bit_cast(T, (uint16_t)(v[i] >> 16));
    }
  }
  static __device__ __forceinline__ float up(T v) { return (float)v; }
};

// ---- keys ----
__device__ __forceinline__ uint64_t key_of(float x, uint32_t place) {
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 is 0
  return ((uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32) | ~place;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
// lane ^ D's, without an LDS round trip: DPP within 16 lanes, swaps of rows and halves
template <int D>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  if constexpr (D == 1) return dpp_u32<0xB1>(v);
  if constexpr (D == 2) return dpp_u32<0x4E>(v);
  if constexpr (D == 3) return dpp_u32<0x1B>(v);
  if constexpr (D == 7) return dpp_u32<0x141>(v);   // half-row mirror
  if constexpr (D == 15) return dpp_u32<0x140>(v);  // row mirror
  if constexpr (D == 4) {  // lane + 4 to the lower half of 8, lane - 4 to the upper
    const int lower = __builtin_amdgcn_update_dpp((int)v, (int)v, 0x104, 0xF, 0x5, false);
    return (uint32_t)__builtin_amdgcn_update_dpp(lower, (int)v, 0x114, 0xF, 0xA, false);
  }
  if constexpr (D == 8) return dpp_u32<0x128>(v);  // rotated within 16
  if constexpr (D == 16) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? p[0] : p[1];
  }
  if constexpr (D == 32) {
    const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? p[0] : p[1];
  }
  if constexpr (D == 31) return lane_xor<16>(lane_xor<15>(v));
  if constexpr (D == 63) return lane_xor<32>(lane_xor<16>(lane_xor<15>(v)));
}
template <int D>
__device__ __forceinline__ uint64_t lane_xor64(uint64_t k) {
  return ((uint64_t)lane_xor<D>((uint32_t)(k >> 32)) << 32) | lane_xor<D>((uint32_t)k);
}
__device__ __forceinline__ uint64_t readlane64(uint64_t k, uint32_t lane) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), (int)lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)k, (int)lane);
}
// the larger of a lane's key and its partner's where lane & HALF is 0, the smaller elsewhere
template <int PARTNER, int HALF>
__device__ __forceinline__ uint64_t exchange(uint64_t k) {
  constexpr uint64_t upper = HALF == 1 ? 0xAAAAAAAAAAAAAAAA : HALF == 2 ? 0xCCCCCCCCCCCCCCCC : HALF == 4 ? 0xF0F0F0F0F0F0F0F0
                             : HALF == 8 ? 0xFF00FF00FF00FF00 : HALF == 16 ? 0xFFFF0000FFFF0000 : 0xFFFFFFFF00000000;
  const uint64_t o = lane_xor64<PARTNER>(k);
  return __builtin_amdgcn_inverse_ballot_w64(__builtin_amdgcn_ballot_w64(o > k) ^ upper) ? o : k;
}
// bitonic sequences of 2 D lanes each, sorted, the largest first
template <int D>
__device__ __forceinline__ uint64_t sort_bitonic(uint64_t k) {
  k = exchange<D, D>(k);
  if constexpr (D > 1) k = sort_bitonic<D / 2>(k);
  return k;
}
// two sorted sequences of D lanes each into one: after an exchange with the mirror lane
// both halves are bitonic
template <int D>
__device__ __forceinline__ uint64_t sort_halves(uint64_t k) {
  k = exchange<2 * D - 1, D>(k);
  if constexpr (D > 1) k = sort_bitonic<D / 2>(k);
  return k;
}
__device__ __forceinline__ uint64_t sort64(uint64_t k) {
  k = sort_halves<1>(k);
  k = sort_halves<2>(k);
  k = sort_halves<4>(k);
  k = sort_halves<8>(k);
  k = sort_halves<16>(k);
  return sort_halves<32>(k);
}
// the 64 largest of two sorted lists, sorted
__device__ __forceinline__ uint64_t merge64(uint64_t a, uint64_t b) {
  const uint64_t o = lane_xor64<63>(b);
  return sort_bitonic<32>(a > o ? a : o);
}
// key c (the same in all lanes) into a sorted list
__device__ __forceinline__ uint64_t insert(uint64_t list, uint64_t c, uint32_t lane) {
  const uint32_t at = (uint32_t)__popcll(__ballot(list > c));
  const uint64_t up = ((uint64_t)dpp_u32<0x138>((uint32_t)(list >> 32)) << 32) | dpp_u32<0x138>((uint32_t)list);  // lane - 1's
  return lane < at ? list : lane == at ? c : up;
}

// ---- (m, l, s) ----
struct Sums {
  float m, l, s;
};
__device__ __forceinline__ Sums moved(Sums a, float M) {  // to a maximum that is no lower
  const bool some = a.m != -__builtin_inff();
  const float d = a.m - M, f = some ? __builtin_amdgcn_exp2f(d * LOG2E) : 0.f;
  return {M, f * a.l, some ? f * (f == 0.f ? 0.f : __builtin_fmaf(d, a.l, a.s)) : 0.f};
}
__device__ __forceinline__ Sums over_lanes(Sums a) {
  float M = max16_lanes(a.m);
  M = fmaxf(M, __uint_as_float(lane_xor<16>(__float_as_uint(M))));
  M = fmaxf(M, __uint_as_float(lane_xor<32>(__float_as_uint(M))));
  a = moved(a, M);
  return {M, sum64_lanes(a.l), sum64_lanes(a.s)};
}

// a partial's words cross from one XCD's L2 to another's
__device__ __forceinline__ void put64(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t get64(uint64_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t two(float a, float b) {
  return ((uint64_t)__float_as_uint(b) << 32) | __float_as_uint(a);
}

template <class L>
__device__ __forceinline__ void logprobs_body(const ScoreArgs& a) {
  typedef typename L::T T;
  constexpr uint32_t LOADS = PER / L::WIDTH;
  __shared__ uint64_t s_list[WAVES][64];
  __shared__ Sums s_sums[WAVES];
  __shared__ uint32_t s_last;
  __shared__ uint64_t s_least;  // the highest of the waves' k-th: no lower element is one of the row's k
  const uint32_t tid = threadIdx.x, lane = tid & 63, w = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t row = a.row0 + blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const T* x = (const T*)a.logits + (size_t)row * a.ld;
  // this split's chunks, to the waves in turn
  const uint32_t begin = split * a.per_split, end = a.vocab - begin < a.per_split ? a.vocab : begin + a.per_split;

  // the first 64 given tokens and their logits, on their way while the row is read
  int32_t token = -1;
  float given = 0.f;
  if (w == 0 && lane < a.given) {
    token = a.tokens[(size_t)row * a.given + lane];
    if ((uint32_t)token < a.vocab) given = L::up(x[token]);
  }
  if (tid == 0) s_least = 0;
  if (a.top) __syncthreads();
  Sums sum = {-__builtin_inff(), 0.f, 0.f};
  uint64_t list = 0, least = 0;  // sorted over the lanes; the highest k-th that the wave knows of
  float least_value = -__builtin_inff();
  auto place = [&](uint32_t at, uint32_t i) { return at + i / L::WIDTH * 64 * L::WIDTH + lane * L::WIDTH + i % L::WIDTH; };
  auto load = [&](uint32_t at, float (&v)[PER]) {
    if (at + CHUNK <= end) {
#pragma unroll
      for (uint32_t k = 0; k < LOADS; k++) L::load(x + at + k * 64 * L::WIDTH + lane * L::WIDTH, v + k * L::WIDTH);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < PER; i++)
        v[i] = place(at, i) < end ? L::up(x[place(at, i)]) : -__builtin_inff();  // weighs nothing
    }
  };
  // The chunk's elements above the k-th of any of the waves' lists.  While many lanes
  // have some, the best of each lane goes in, sorted first; the others one by one, slot
  // by slot (an element of each lane).
  auto pick = [&](uint32_t at, const float (&v)[PER], bool many) {
    uint64_t below = ~0ull;  // the lane's elements from this key on are through
    auto key = [&](uint32_t i) {  // 0: none, or no number
      // (worked out anew for each use: kept, the 16 keys cost half of the waves)
      float x = v[i];
      asm volatile("" : "+v"(x));
      const uint64_t k = key_of(x, place(at, i));
      return x == x && k < below && k > least ? k : 0ull;
    };
    auto raise = [&] {
      const uint64_t k = readlane64(list, a.top - 1);
      least = k > least ? k : least;
      least_value = least ? value_of(least) : -__builtin_inff();
    };
    while (many) {
      uint64_t best = 0;
#pragma unroll
      for (uint32_t i = 0; i < PER; i++) {
        const uint64_t k = key(i);
        best = k > best ? k : best;
      }
      many = __popcll(__ballot(best != 0)) > MANY;
      if (!many) break;
      const uint64_t sorted = sort64(best);
      list = readlane64(list, 0) ? merge64(list, sorted) : sorted;
      raise();
      below = best;
      if (a.top <= FEW) break;
    }
#pragma unroll
    for (uint32_t i = 0; i < PER; i++) {
      if (!__any(v[i] >= least_value)) continue;
      const uint64_t k = key(i);
      uint64_t there = __ballot(k != 0);
      while (there) {
        const uint64_t c = readlane64(k, (uint32_t)__ffsll((unsigned long long)there) - 1);
        there &= there - 1;
        if (c > least) {
          list = insert(list, c, lane);
          raise();
        }
      }
    }
    if (lane == 0) __hip_atomic_fetch_max(&s_least, least, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  float v[PER], next[PER];
  uint32_t at = begin + w * CHUNK;
  if (at < end) load(at, v);
  for (; at < end; at += WAVES * CHUNK) {
    const bool more = at + WAVES * CHUNK < end;
    if (more) load(at + WAVES * CHUNK, next);
    float mx = v[0];
#pragma unroll
    for (uint32_t i = 1; i < PER; i++) mx = fmaxf(mx, v[i]);
    if (__any(mx > sum.m)) sum = moved(sum, fmaxf(mx, sum.m));
    const float m = sum.m == -__builtin_inff() ? 0.f : sum.m;
#pragma unroll
    for (uint32_t i = 0; i < PER; i++) {
      const float d = v[i] - m, e = __builtin_amdgcn_exp2f(d * LOG2E);
      sum.l += e;
      sum.s = __builtin_fmaf(e, fmaxf(d, -1000.f), sum.s);  // 0 of -inf
    }
    if (a.top && __any(mx >= least_value || !least)) {
      const uint64_t others = __hip_atomic_load(&s_least, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      const uint64_t known = readlane64(others, 0);
      if (known > least) {
        least = known;
        least_value = value_of(least);
      }
      const uint64_t some = __ballot(mx >= least_value || !least);
      if (some) {
        if (at + CHUNK > end)
#pragma unroll
          for (uint32_t i = 0; i < PER; i++)
            if (place(at, i) >= end) v[i] = __builtin_nanf("");  // no element
        pick(at, v, __popcll(some) > MANY);
      }
    }
    if (more)
#pragma unroll
      for (uint32_t i = 0; i < PER; i++) v[i] = next[i];
  }

  // ---- the waves', then the splits' ----
  sum = over_lanes(sum);
  s_list[w][lane] = list;
  if (lane == 0) s_sums[w] = sum;
  __syncthreads();
  auto join = [&](Sums b) {
    const float M = fmaxf(sum.m, b.m);
    const Sums p = moved(sum, M), q = moved(b, M);
    sum = {M, p.l + q.l, p.s + q.s};
  };
  // lists of the waves into wave 0's
  auto gather = [&] {
    static_assert(WAVES == 4, "two levels");
    if (!(w & 1)) list = merge64(list, s_list[w + 1][lane]);
    if (w == 2) s_list[2][lane] = list;
    __syncthreads();
    if (w == 0) list = merge64(list, s_list[2][lane]);
  };
  if (a.top) gather();
  if (w == 0)
    for (uint32_t k = 1; k < WAVES; k++) join(s_sums[k]);
  if (a.splits > 1) {
    // per split: (m, l), (s, -), the keys
    const size_t stride = a.top + 2;
    uint64_t* all = a.parts + (size_t)(row - a.row0) * a.splits * stride;
    if (w == 0) {
      uint64_t* mine = all + split * stride;
      if (lane < a.top) put64(mine + 2 + lane, list);
      if (lane == 0) {
        put64(mine, two(sum.m, sum.l));
        put64(mine + 1, two(sum.s, 0.f));
      }
    }
    stores_done();
    __syncthreads();
    if (tid == 0) {
      uint32_t* done = a.counters + (row - a.row0);
      s_last = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.splits - 1;
      if (s_last) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!s_last) return;
    list = 0;
    if (a.top) {
      constexpr uint32_t BATCH = 8;  // loads under way
      for (uint32_t k0 = w; k0 < a.splits; k0 += WAVES * BATCH) {
        uint64_t x[BATCH];
#pragma unroll
        for (uint32_t j = 0; j < BATCH; j++)
          x[j] = lane < a.top && k0 + j * WAVES < a.splits ? get64(all + (k0 + j * WAVES) * stride + 2 + lane) : 0ull;
        if (k0 == w) list = x[0];
#pragma unroll
        for (uint32_t j = 0; j < BATCH; j++)
          if (k0 + j * WAVES < a.splits && (j || k0 != w)) list = merge64(list, x[j]);
      }
      s_list[w][lane] = list;
    }
    sum = {-__builtin_inff(), 0.f, 0.f};
    if (lane < a.splits) {  // at most 64
      const uint64_t ml = get64(all + lane * stride), s = get64(all + lane * stride + 1);
      sum = {__uint_as_float((uint32_t)ml), __uint_as_float((uint32_t)(ml >> 32)), __uint_as_float((uint32_t)s)};
    }
    sum = over_lanes(sum);
    __syncthreads();
    if (a.top) gather();
  }
  if (w) return;
  // a row without a finite maximum has no distribution
  const float nan = __builtin_nanf("");
  const bool fine = fabsf(sum.m) < __builtin_inff();
  const float log_l = fine ? logf(sum.l) : nan;
  if (a.entropy && lane == 0) a.entropy[row] = log_l - sum.s / sum.l;
  if (lane < a.top) {
    const size_t to = (size_t)row * a.top + lane;
    a.top_ids[to] = list ? (int32_t)~(uint32_t)list : -1;
    a.top_logprobs[to] = list ? value_of(list) - sum.m - log_l : nan;
  }
  for (uint32_t k = lane; k < a.given; k += 64) {
    const size_t to = (size_t)row * a.given + k;
    if (k >= 64) {
      token = a.tokens[to];
      if ((uint32_t)token < a.vocab) given = L::up(x[token]);
    }
    float p = 0.f;
    if (token != -1) {
      const bool in = (uint32_t)token < a.vocab;
      if (!in) paged_err(a.err, PAGED_ERR_SCORE_TOKEN, row);
      p = in ? given - sum.m - log_l : nan;
    }
    a.logprobs[to] = p;
  }
}

#define DEF_LOGPROBS(TYPE, L)                                                                          \
  extern "C" __global__ __launch_bounds__(THREADS) void smith_logprobs_##TYPE(ScoreArgs a) { \
    logprobs_body<L>(a);                                                                               \
  }
DEF_LOGPROBS(f32, LogitsF32)
DEF_LOGPROBS(f16, Logits16<_Float16>)
DEF_LOGPROBS(bf16, Logits16<__bf16>)
