// paged_kernels.hip -- gfx950 kernels of the paged key-value cache: several
// requests share one pool of pages per layer (smith_paged.hsaco).
//
// Pools are [n_pages][n_kv_heads][page_size][head_dim], one for keys and one
// for values, of f32, f16 or bf16; page_size is a power of two.  Request b's
// key t lies in page tables[b][t / page_size] at t % page_size; the slot of a
// key is page * page_size + t % page_size.  Everything a kernel reads out of
// device memory to index with (lengths, slots, positions, pages) is checked
// there before it is used; what fails is left out and recorded for the next
// synchronising call (paged_err).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lanes.h"
#include "paged.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
// rows and tables of the caller need start on no more than 4 bytes; the
// hardware's 16-byte accesses want no more either
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4_8 __attribute__((ext_vector_type(4), aligned(8)));
__device__ __forceinline__ f32x4 load8(const float* p) { return *(const f32x4_8*)p; }
__device__ __forceinline__ f32x4 load4(const float* p) { return *(const f32x4_any*)p; }
__device__ __forceinline__ void store4(float* p, f32x4 v) { *(f32x4_any*)p = v; }

// One 64-bit word of host-mapped memory: (code, argument), the first one kept.
__device__ __forceinline__ void paged_err(uint64_t* __restrict__ err, uint32_t code, uint32_t arg) {
  if (__hip_atomic_load(err, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM) == 0u)
    __hip_atomic_store(err, ((uint64_t)arg << 32) | code, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

template <class T>
__device__ __forceinline__ T max64_lanes(T v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  return v;
}
// sum over the lanes up to this one: within rows of 16, then across them
__device__ __forceinline__ uint32_t scan64_lanes(uint32_t v) {
#define SCAN_DPP(CTRL, ROWS) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false)
  SCAN_DPP(0x111, 0xF);  // row_shr 1, 2, 4, 8
  SCAN_DPP(0x112, 0xF);
  SCAN_DPP(0x114, 0xF);
  SCAN_DPP(0x118, 0xF);
  SCAN_DPP(0x142, 0xA);  // row_bcast 15 into rows 1 and 3, 31 into 2 and 3
  SCAN_DPP(0x143, 0xC);
#undef SCAN_DPP
  return v;
}

// A page's values in f32, and f32 rounded to nearest even into a page.
struct KvF32 {
  typedef float T;
  static __device__ __forceinline__ float up(T v) { return v; }
  static __device__ __forceinline__ T down(float v) { return v; }
};
struct KvF16 {
  typedef _Float16 T;
  static __device__ __forceinline__ float up(T v) { return (float)v; }
  static __device__ __forceinline__ T down(float v) { return (T)v; }
};
struct KvBf16 {
  typedef __bf16 T;
  static __device__ __forceinline__ float up(T v) { return (float)v; }
  static __device__ __forceinline__ T down(float v) { return (T)v; }
};

// ---------------------------------------------------------------------------
// Plan of a step.  Request b has c = cached[b] keys and brings a = added[b]
// rows; with P keys to a page it owns old = ceil(c/P) pages and needs new =
// ceil((c+a)/P).  R_b = sum of a, F_b = sum of (new - old) over the requests
// before b; new page j comes off the end of the free list,
//   tables[b][j] = free[n - 1 - F_b - (j - old)],  old <= j < new,
// and row R_b + i is position c + i in slot tables[b][(c+i)/P]*P + (c+i)%P.
//
// Latency is all of it (a few bytes a row): one launch, no exchange between
// workgroups.  Each of them forms both prefix sums of all the requests by
// itself (they are a few KB, in L2) and then serves its PLAN_THREADS rows: a
// row's request by bisection, its page from the table or, if it is a new one,
// from the free list; the row that opens a page writes the table entry.  24
// requests, 20 rows: 3.2 us; 700 requests, 9631 rows: 4.8 us.
// ---------------------------------------------------------------------------
#define PLAN_THREADS 256

extern "C" __global__ __launch_bounds__(PLAN_THREADS) void smith_paged_plan(
    const int32_t* __restrict__ cached, const int32_t* __restrict__ added, uint32_t n_req,
    const int32_t* __restrict__ free_pages, const int32_t* __restrict__ free_count, uint32_t n_list, uint32_t n_pages,
    uint32_t shift, uint32_t max_pages, uint32_t max_rows, int32_t* __restrict__ tables, int32_t* __restrict__ row_start,
    int32_t* __restrict__ lens, int32_t* __restrict__ slots, int32_t* __restrict__ positions,
    int32_t* __restrict__ free_left, uint64_t* __restrict__ err) {
  __shared__ uint32_t s_row[PAGED_MAX_REQ + 1], s_page[PAGED_MAX_REQ], s_had[PAGED_MAX_REQ];
  __shared__ uint64_t s_wr[PLAN_THREADS / 64], s_wp[PLAN_THREADS / 64];
  __shared__ uint32_t s_bad[PLAN_THREADS / 64];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t P = 1u << shift;
  const uint64_t cap = (uint64_t)max_pages << shift;
  const uint32_t per = (n_req + PLAN_THREADS - 1) / PLAN_THREADS;
  const int64_t have = free_count[0];
  // f(request, its keys, its rows) of this thread's requests, four loaded at once
  auto each = [&](auto f) {
    for (uint32_t k0 = 0; k0 < per; k0 += 4) {
      int32_t c[4], a[4];
#pragma unroll
      for (uint32_t k = 0; k < 4; k++) {
        const uint32_t b = tid * per + k0 + k, at = b < n_req ? b : n_req - 1;
        c[k] = cached[at];
        a[k] = added[at];
      }
#pragma unroll
      for (uint32_t k = 0; k < 4; k++) {
        const uint32_t b = tid * per + k0 + k;
        if (k0 + k < per && b < n_req) f(b, c[k], a[k]);
      }
    }
  };
  auto new_pages = [&](int32_t c, int32_t a) {
    return (uint32_t)(((uint64_t)((int64_t)c + a + P - 1) >> shift) - ((uint64_t)((int64_t)c + P - 1) >> shift));
  };
  uint64_t rows = 0, pages = 0;
  uint32_t bad = 0;  // 1 + the first request whose lengths do not fit
  each([&](uint32_t b, int32_t c, int32_t a) {
    if ((c < 0 || a < 0 || (uint64_t)((int64_t)c + a) > cap) && !bad) bad = b + 1;
    if (bad) return;
    rows += (uint32_t)a;
    pages += new_pages(c, a);
  });
  // sums over the wave up to this thread, of less than 2^35 each, in two halves of 24 bits
  auto scan = [](uint64_t v) {
    return ((uint64_t)scan64_lanes((uint32_t)(v >> 24)) << 24) + scan64_lanes((uint32_t)v & 0xFFFFFFu);
  };
  const uint64_t ir = scan(rows), ip = scan(pages);
  const uint64_t bads = __ballot(bad != 0);
  const uint32_t first_bad = bads ? (uint32_t)__shfl((int)bad, __ffsll((unsigned long long)bads) - 1) : 0u;
  if (lane == 63) {
    s_wr[wave] = ir;
    s_wp[wave] = ip;
    s_bad[wave] = first_bad;
  }
  __syncthreads();
  uint64_t tr = 0, tp = 0, br = 0, bp = 0;
  uint32_t bad_req = 0;
#pragma unroll
  for (uint32_t w = 0; w < PLAN_THREADS / 64; w++) {
    if (w < wave) {
      br += s_wr[w];
      bp += s_wp[w];
    }
    tr += s_wr[w];
    tp += s_wp[w];
    if (!bad_req) bad_req = s_bad[w];
  }
  // the same in every workgroup
  const uint32_t code = bad_req             ? PAGED_ERR_PLAN_LENGTH
                        : tr > max_rows     ? PAGED_ERR_PLAN_ROWS
                        : have < 0 || have > (int64_t)n_list || tp > (uint64_t)have ? PAGED_ERR_PLAN_PAGES
                                            : 0u;
  if (code && blockIdx.x == 0 && tid == 0) paged_err(err, code, bad_req ? bad_req - 1 : code == PAGED_ERR_PLAN_ROWS ? max_rows : (uint32_t)have);
  uint32_t at_row = (uint32_t)(br + ir - rows), at_page = (uint32_t)(bp + ip - pages);
  each([&](uint32_t b, int32_t c, int32_t a) {
    if (code) a = 0;
    s_row[b] = at_row;
    s_page[b] = at_page;
    s_had[b] = (uint32_t)c;
    if (blockIdx.x == 0) {
      row_start[b] = code ? 0 : (int32_t)at_row;
      lens[b] = (int32_t)((uint32_t)c + (uint32_t)a);
    }
    at_row += (uint32_t)a;
    if (!code) at_page += new_pages(c, a);
  });
  const uint32_t total = code ? 0u : (uint32_t)tr;
  if (tid == 0) {
    s_row[n_req] = total;
    if (blockIdx.x == 0) {
      row_start[n_req] = (int32_t)total;
      free_left[0] = code ? (int32_t)have : (int32_t)(have - (int64_t)tp);
    }
  }
  __syncthreads();
  const uint32_t r = blockIdx.x * PLAN_THREADS + tid;
  if (r >= max_rows) return;
  int32_t slot = -1, pos = -1;
  if (r < total) {
    // the last request that starts at or before r (those without rows start there too)
    uint32_t lo = 0, hi = n_req;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) >> 1;
      if (s_row[mid] <= r) lo = mid;
      else hi = mid;
    }
    const uint32_t c = s_had[lo], p = c + (r - s_row[lo]);
    const uint32_t j = p >> shift, old = (c + P - 1) >> shift;
    const int32_t page = j < old ? tables[(size_t)lo * max_pages + j]
                                 : free_pages[(uint32_t)have - 1 - (s_page[lo] + (j - old))];
    if (j >= old && (p & (P - 1)) == 0) tables[(size_t)lo * max_pages + j] = page;
    pos = (int32_t)p;
    if ((uint32_t)page < n_pages) slot = (int32_t)(((uint32_t)page << shift) + (p & (P - 1)));
    else paged_err(err, PAGED_ERR_PLAN_PAGE, lo);
  }
  slots[r] = slot;
  positions[r] = pos;
}

// ---------------------------------------------------------------------------
// Append: q and k of every row rotated by the angles of its position, k and v
// rounded into the row's slot.  A pair (x0, x1) = (x[i], x[i + H]) becomes
// (x0 cos - x1 sin, x0 sin + x1 cos) with table entry pos * H + i; H is half
// the row's width (q's and k's own: the whole-row indexing of smith_attention)
// or half the head.  Bound by memory: a thread takes four neighbouring pairs
// (two 16-byte loads of x, one each of cos and sin), or eight elements of v.  6001
// rows of 32 + 2 x 8 heads of 128 into bf16 pages, 273 MB: 49 us, 5.5 TB/s (a
// large copy: 4.8); 57 of them into f16 pages 3.0 us.
// ---------------------------------------------------------------------------
template <class KV>
__device__ __forceinline__ void put4(typename KV::T* p, f32x4 v) {
  typedef typename KV::T T4 __attribute__((ext_vector_type(4)));
  T4 t;
#pragma unroll
  for (int i = 0; i < 4; i++) t[i] = KV::down(v[i]);
  *(T4*)p = t;
}

template <class KV>
__device__ __forceinline__ void append_body(const float* qkv, uint32_t ld, const int32_t* __restrict__ slots,
                                            const int32_t* __restrict__ positions, uint32_t nH, uint32_t nKV,
                                            uint32_t hd, uint32_t rope, const float* __restrict__ cosT,
                                            const float* __restrict__ sinT, uint32_t rope_len,
                                            typename KV::T* __restrict__ kpages, typename KV::T* __restrict__ vpages,
                                            uint32_t n_slots, uint32_t shift, float* q_out, uint32_t ld_q,
                                            uint32_t row0, uint64_t* __restrict__ err) {
  const uint32_t r = row0 + blockIdx.y, item = blockIdx.x * 256 + threadIdx.x;
  const int32_t slot = slots[r], pos = positions[r];
  if (slot == -1) return;  // padding
  const bool lead = item == 0;
  if ((uint32_t)slot >= n_slots) {
    if (lead) paged_err(err, PAGED_ERR_APPEND_SLOT, r);
    return;
  }
  const uint32_t Wq = nH * hd, Wk = nKV * hd;
  if (rope && (pos < 0 || ((uint64_t)(uint32_t)pos + 1) * ((rope == PAGED_ROPE_ROW ? Wq : hd) / 2) > rope_len)) {
    if (lead) paged_err(err, PAGED_ERR_APPEND_POS, r);
    return;
  }
  const uint32_t nq = Wq / 8, nk = Wk / 8;
  const float* row = qkv + (size_t)r * ld;
  const uint32_t P = 1u << shift, page = (uint32_t)slot >> shift, off = (uint32_t)slot & (P - 1);
  // element e of the row's keys or values in its page
  auto at = [&](uint32_t e) {
    return (((size_t)page * nKV + e / hd) * P + off) * hd + e % hd;
  };
  if (item < nq + nk) {
    const bool isq = item < nq;
    if (isq && !q_out) return;
    const uint32_t W = isq ? Wq : Wk, i4 = 4 * (isq ? item : item - nq);
    const float* x = row + (isq ? 0 : Wq);
    uint32_t e0, half, t;  // first element of the pairs, distance to the second, table entry
    if (rope == PAGED_ROPE_ROW) {
      half = W / 2;
      e0 = t = i4;
    } else {
      half = hd / 2;
      t = i4 % half;
      e0 = i4 / half * hd + t;
    }
    f32x4 x0 = load4(x + e0), x1 = load4(x + e0 + half);
    if (rope) {
      const size_t a = (size_t)(uint32_t)pos * half + t;
      const f32x4 c = load4(cosT + a), s = load4(sinT + a);
      const f32x4 y0 = x0 * c - x1 * s;
      x1 = x0 * s + x1 * c;
      x0 = y0;
    }
    if (isq) {
      store4(q_out + (size_t)r * ld_q + e0, x0);
      store4(q_out + (size_t)r * ld_q + e0 + half, x1);
    } else {
      put4<KV>(kpages + at(e0), x0);
      put4<KV>(kpages + at(e0 + half), x1);
    }
  } else if (item < nq + 2 * nk) {
    const uint32_t e = 8 * (item - nq - nk);
    const float* x = row + Wq + Wk + e;
    put4<KV>(vpages + at(e), load4(x));
    put4<KV>(vpages + at(e) + 4, load4(x + 4));
  }
}

#define DEF_APPEND(NAME, KV)                                                                                        \
  extern "C" __global__ __launch_bounds__(256) void NAME(                                                          \
      const float* qkv, uint32_t ld, const int32_t* __restrict__ slots, const int32_t* __restrict__ positions,      \
      uint32_t nH, uint32_t nKV, uint32_t hd, uint32_t rope, const float* __restrict__ cosT,                        \
      const float* __restrict__ sinT, uint32_t rope_len, KV::T* __restrict__ kpages, KV::T* __restrict__ vpages,    \
      uint32_t n_slots, uint32_t shift, float* q_out, uint32_t ld_q, uint32_t row0, uint64_t* __restrict__ err) {   \
    append_body<KV>(qkv, ld, slots, positions, nH, nKV, hd, rope, cosT, sinT, rope_len, kpages, vpages, n_slots,    \
                    shift, q_out, ld_q, row0, err);                                                                 \
  }
DEF_APPEND(smith_paged_append_f32, KvF32)
DEF_APPEND(smith_paged_append_f16, KvF16)
DEF_APPEND(smith_paged_append_bf16, KvBf16)

// ---------------------------------------------------------------------------
// Attention over the pages: row i of request b's n rows is position p = len -
// n + i and sees its keys 0 .. p; head h reads KV head h / G, G = nH / nKV:
//   s_t = scale q.k_t,  out = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m).
// A row without keys gives zeros.
//
// The (row, head) pairs that read one KV head are the columns of a product:
// S^T = K Q^T and O^T = V^T P^T on the matrix cores, 16 columns to a tile, in one
// pass over the keys with each column's running maximum m, sum l and O^T.  In this
// form nothing moves between lanes: a lane's four (or eight) scores of S^T are one
// column's, so they become the P operand where they are, and m, l and the
// rescaling of O^T are the lane's own.
//   MFMA 16x16: lane (n = lane % 16, g = lane / 16) holds row n of A and column n
//   of B at the k's of group g, and rows 4g .. 4g+3 of column n of D.
//   K: A rows are keys, lane n its key's dims.  V: lane n holds dims n*DPL ..
//   +DPL-1 of the keys 4g .. 4g+3 (of each 16), row n of the d-th A operand being
//   dim n*DPL + d; so D's row 4g+i is dim (4g+i)*DPL + d.
//
// f16 and bf16 pages are exact in the matrix cores' operands; q and P are split
// into parts of the pages' type that add up to 22 (two f16) or 24 (three bf16)
// bits, the products are exact and summed in f32.  For f16, q and P are brought far
// up by a power of two first, since small parts round at f16's least step: 2^-38 of
// the largest.  f32 pages go through the f32 matrix cores.
//
// scale log2 e is a factor of q but for a power of two c, by which the sums are
// multiplied.  So a score in powers of two is exact from its sum, its difference
// from m is rounded once and is 0 for the largest, however far up the scores are: a
// weight never leaves its range.
//
// Work is cut on the device, where the lengths are: an item is (request, block
// of columns, KV head, split of the block's keys).  With W = sum over blocks of
// their request's length, a request of more than 5/4 C keys, C = max(split_min,
// W / target), has its keys cut into splits of at most that many, so that target
// items or so, two to a CU, fill the chip whatever the lengths are; requests of
// nearly one length (their longest within 5/4 of the mean) get one item to a
// workgroup and no more.  Every workgroup forms the prefix sums of the items by
// itself.  The last of a block's splits to finish (agent-scope counter) joins
// their partials in split order: the same sums whichever finishes last.  An item
// costs 5 us before its keys count (cycles at 2.4 GHz, one row of 32 heads of 128
// f16: lengths and cuts 1800, the item 2300, Q and the first page 4700, the waves'
// join 1800; of a split 900 to write it, 900 to count it, 4000 to join them),
// which is why twice or three times the items lose: one request of 20000 keys
// 22.8 us with 512 wanted, 30 with 768.
// ---------------------------------------------------------------------------
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// maximum over the lanes l, l ^ 16, l ^ 32, l ^ 48 (a number wins over a NaN)
__device__ __forceinline__ float max_xor16_32(float v) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
// Weights are P = 2^(score - m).  m is P_EXP (of the page type) under a column's
// maximum, and follows a new one only when that would have a weight above 2^P_TOP.
// Past FAR_SCORE f32 holds every second whole number and fewer: m is the maximum
// itself there, P_EXP below which would be rounded to something else.
#define FAR_SCORE 16777216.0f

// the parts of eight f32 values in the pages' type, and the product of parts
struct MmF16 {
  typedef _Float16 T;
  static constexpr int TERMS = 2;
  static constexpr uint32_t EXPONENT = 0x7C00u;
  // The largest weight is 2^13 to 2^15.9 of f16's 2^16: its second part rounds at
  // 2^-25, half of f16's least step, so beside 2^-22 of itself a weight loses up to
  // 2^-38 of the largest.  (2^6 to 2^14 would lose 2^-31, and be 1 % faster for rows: m
  // moves less often.  A prompt of 2000 rows, 32 heads on 8 of 128, 83.0 and 83.8 us;
  // 600 rows 31.1 and 31.7.)
  static constexpr float P_EXP = 13.0f, P_TOP = 15.9f;
  // by what power of two q of elements up to 2^e is multiplied: to [2^15, 2^16), far up
  // in f16 as well
  static __device__ __forceinline__ int q_shift(int e) { return 16 - e; }
  // word k of the parts, from values 2k and 2k + 1
  static __device__ __forceinline__ void split2(float x, float y, u32x4 (&t)[TERMS], int k) {
    // the rest in one mixed-precision operation each (without a factor that the
    // compiler does not know it makes a conversion and a subtraction)
    float minus = -1.f;
    asm("" : "+s"(minus));
    const f16x2 hi = __builtin_convertvector((f32x2){x, y}, f16x2);
    const f16x2 lo = (f16x2){(_Float16)__builtin_fmaf((float)hi[0], minus, x), (_Float16)__builtin_fmaf((float)hi[1], minus, y)};
    t[0][k] = __builtin_bit_cast(uint32_t, hi);
    t[1][k] = __builtin_bit_cast(uint32_t, lo);
  }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
struct MmBf16 {
  typedef __bf16 T;
  static constexpr int TERMS = 3;
  static constexpr uint32_t EXPONENT = 0x7F80u;
  // only what is far from 1 is moved, to where its parts and its sums of products with
  // keys of any size are inside f32 if they were
  static __device__ __forceinline__ int q_shift(int e) { return (e < -64 ? -64 : e > 64 ? 64 : e) - e; }
  static constexpr float P_EXP = -8.0f, P_TOP = 0.0f;  // no weight above 1: sums overflow where they would of weights of 1
  static __device__ __forceinline__ void split2(float x, float y, u32x4 (&t)[TERMS], int k) {
    f32x2 r = (f32x2){x, y};
#pragma unroll
    for (int p = 0; p < TERMS; p++) {
      t[p][k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
      r[0] -= __uint_as_float(t[p][k] << 16);
      r[1] -= __uint_as_float(t[p][k] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
  }
};

// The first of the DPL dims that lane n of 16 holds of a key: none past the head.
// Where DPL does not divide the head the last two lanes share some dims, whose
// sums are the same and go to the same place.
template <int DPL>
__device__ __forceinline__ uint32_t first_dim(uint32_t n, uint32_t hd) {
  return n * DPL < hd - DPL ? n * DPL : hd - DPL;
}
template <int N>
struct Words {
  uint32_t w[N];
};

// One wave's tile of 32 keys of f16 or bf16: K and V operands in registers.
template <class MM, int DPL>
struct Tile16 {
  typedef typename MM::T T;
  static constexpr int NJ = 2, KS = DPL / 2, TERMS = MM::TERMS, QREG = KS * TERMS;
  static constexpr float P_EXP = MM::P_EXP, P_TOP = MM::P_TOP;
  u32x4 K[NJ][KS];
  uint32_t V[8][DPL / 2];  // a key's dims of this lane
  // the lane's column of q: dims s*32 + 8g .. +7 (past the head others, then 0)
  static constexpr int QRAW = 2 * KS;
  static __device__ __forceinline__ void load_q(const float* q, uint32_t g, uint32_t hd, f32x4 (&x)[QRAW]) {
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const uint32_t e = s * 32 + 8 * g;
      const float* at = q + (e < hd ? e : hd - 8);
      x[2 * s] = load4(at);
      x[2 * s + 1] = load4(at + 4);
    }
  }
  // ... in parts, times `factor` (at least 0.36, less than 0.73, of either sign) and a
  // power of two (MM::q_shift); what is not finite stays as it is.  Register k of the
  // steps that do(s) says goes to put(k, parts).
  template <class DO, class PUT>
  static __device__ __forceinline__ void split_q(const f32x4 (&x)[QRAW], bool there, uint32_t g, uint32_t hd, float factor,
                                                 int& e2, DO todo, PUT put) {
    float big = 0.f;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int e = 0; e < 8; e++) big = fmaxf(big, fabsf(x[2 * s + e / 4][e % 4]));  // a repeated element is one of the row's
    big = max_xor16_32(big);
    e2 = there && big > 0.f && big < __builtin_inff() ? MM::q_shift(__builtin_amdgcn_frexp_expf(big)) : 0;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      if (!todo(s)) continue;
      float y[8];
      const bool in = there && s * 32 + 8 * g < hd;
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = in ? __builtin_amdgcn_ldexpf(x[2 * s + e / 4][e % 4], e2) * factor : 0.f;
      u32x4 t[TERMS];
#pragma unroll
      for (int k = 0; k < 4; k++) MM::split2(y[2 * k], y[2 * k + 1], t, k);
#pragma unroll
      for (int k = 0; k < TERMS; k++) put(s * TERMS + k, t[k]);
    }
  }
  // of the j-th 16 keys, lane n's: `off` values behind `key`
  __device__ __forceinline__ void load_k(int j, const T* key, uint32_t off, uint32_t g, uint32_t hd) {
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const uint32_t e = s * 32 + 8 * g;
      K[j][s] = *(const u32x4*)(key + (off + (e < hd ? e : hd - 8)));  // past the head: against zeros of Q
    }
  }
  // key 4g + i of the j-th 16
  __device__ __forceinline__ void load_v(int j, int i, const T* key, uint32_t off, uint32_t n, uint32_t hd) {
    uint32_t(&r)[DPL / 2] = V[4 * j + i];
    const Words<DPL / 2> v = *(const Words<DPL / 2>*)(key + (off + first_dim<DPL>(n, hd)));
#pragma unroll
    for (int k = 0; k < DPL / 2; k++) r[k] = v.w[k];
  }
  __device__ __forceinline__ void zero_v(int j, int i) {
#pragma unroll
    for (int k = 0; k < DPL / 2; k++) V[4 * j + i][k] = 0u;
  }
  // dim d of the lane's keys: word k holds keys 2k, 2k+1
  __device__ __forceinline__ u32x4 dim(int d) const {
    u32x4 a;
#pragma unroll
    for (int k = 0; k < 4; k++)
      a[k] = __builtin_amdgcn_perm(V[2 * k + 1][d / 2], V[2 * k][d / 2], d & 1 ? 0x07060302u : 0x05040100u);
    return a;
  }
  __device__ __forceinline__ bool finite_v(int j, int i) const {
    bool ok = true;
#pragma unroll
    for (int d = 0; d < DPL / 2; d++) {
      const uint32_t x = V[4 * j + i][d];
      ok = ok && (x & MM::EXPONENT) != MM::EXPONENT && (x & (MM::EXPONENT << 16)) != (MM::EXPONENT << 16);
    }
    return ok;
  }
  template <class QF>
  __device__ __forceinline__ void scores(QF q, f32x4 (&S)[NJ]) const {
    // products of one sum are four apart, which covers the first's latency
    f32x4 sum[2][NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) sum[0][j] = sum[1][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < KS * TERMS; i++) {
      const u32x4 x = q(i);
#pragma unroll
      for (int j = 0; j < NJ; j++) sum[i & 1][j] = MM::mfma(K[j][i / TERMS], x, sum[i & 1][j]);
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) S[j] = sum[0][j] + sum[1][j];
  }
  __device__ __forceinline__ void add_pv(const f32x4 (&S)[NJ], f32x4 (&O)[DPL]) const {
    u32x4 t[TERMS];
#pragma unroll
    for (int k = 0; k < 4; k++) MM::split2(S[k / 2][k % 2 * 2], S[k / 2][k % 2 * 2 + 1], t, k);
#pragma unroll
    for (int d = 0; d < DPL; d += 2) {
      const u32x4 v[2] = {dim(d), dim(d + 1)};
#pragma unroll
      for (int k = 0; k < TERMS; k++)
#pragma unroll
        for (int e = 0; e < 2; e++) O[d + e] = MM::mfma(v[e], t[k], O[d + e]);
    }
  }
};

// One wave's tile of 16 keys of f32.
template <int DPL>
struct Tile32 {
  typedef float T;
  static constexpr int NJ = 1, KS = DPL, QREG = KS;
  static constexpr float P_EXP = -8.0f, P_TOP = 0.0f;  // no weight above 1: sums overflow where they would of weights of 1
  f32x4 K[KS];  // dims s*16 + 4g .. +3
  float V[4][DPL];
  static constexpr int QRAW = KS;
  static __device__ __forceinline__ void load_q(const float* q, uint32_t g, uint32_t hd, f32x4 (&x)[QRAW]) {
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const uint32_t e = s * 16 + 4 * g;
      x[s] = load4(q + (e < hd ? e : hd - 4));
    }
  }
  template <class DO, class PUT>
  static __device__ __forceinline__ void split_q(const f32x4 (&x)[QRAW], bool there, uint32_t g, uint32_t hd, float factor,
                                                 int& e2, DO todo, PUT put) {
    e2 = 0;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      if (!todo(s)) continue;
      f32x4 y = x[s] * factor;
      if (!there || s * 16 + 4 * g >= hd) y = (f32x4){0.f, 0.f, 0.f, 0.f};
      put(s, __builtin_bit_cast(u32x4, y));
    }
  }
  __device__ __forceinline__ void load_k(int, const float* key, uint32_t off, uint32_t g, uint32_t hd) {
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const uint32_t e = s * 16 + 4 * g;
      K[s] = *(const f32x4*)(key + (off + (e < hd ? e : hd - 4)));
    }
  }
  __device__ __forceinline__ void load_v(int, int i, const float* key, uint32_t off, uint32_t n, uint32_t hd) {
    const Words<DPL> v = *(const Words<DPL>*)(key + (off + first_dim<DPL>(n, hd)));
#pragma unroll
    for (int k = 0; k < DPL; k++) V[i][k] = __uint_as_float(v.w[k]);
  }
  __device__ __forceinline__ void zero_v(int, int i) {
#pragma unroll
    for (int k = 0; k < DPL; k++) V[i][k] = 0.f;
  }
  __device__ __forceinline__ bool finite_v(int, int i) const {
    bool ok = true;
#pragma unroll
    for (int d = 0; d < DPL; d++) ok = ok && (__float_as_uint(V[i][d]) & 0x7F800000u) != 0x7F800000u;
    return ok;
  }
  template <class QF>
  __device__ __forceinline__ void scores(QF q, f32x4 (&S)[NJ]) const {
    // two independent chains, summed at the end
    f32x4 a = (f32x4){0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const f32x4 x = __builtin_bit_cast(f32x4, q(s));
      a = __builtin_amdgcn_mfma_f32_16x16x4f32(K[s][0], x[0], a, 0, 0, 0);
      b = __builtin_amdgcn_mfma_f32_16x16x4f32(K[s][1], x[1], b, 0, 0, 0);
      a = __builtin_amdgcn_mfma_f32_16x16x4f32(K[s][2], x[2], a, 0, 0, 0);
      b = __builtin_amdgcn_mfma_f32_16x16x4f32(K[s][3], x[3], b, 0, 0, 0);
    }
    S[0] = a + b;
  }
  __device__ __forceinline__ void add_pv(const f32x4 (&S)[NJ], f32x4 (&O)[DPL]) const {
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int d = 0; d < DPL; d++) O[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(V[i][d], S[0][i], O[d], 0, 0, 0);
  }
};

struct AttArgs {
  const float* q;
  const int32_t* row_start;
  const int32_t* lens;
  const int32_t* tables;
  const void* kpages;
  const void* vpages;
  float* out;
  float* parts;        // a split's partial: O [columns][head dim], then (m, l) of each column
  uint32_t* counters;  // splits of a block that are done, by the index of its first partial; zero between calls
  uint32_t* queue;     // items taken beyond each workgroup's first; zero between calls
  uint64_t* err;
  uint32_t ld_q, ld_out, max_rows, n_req, max_pages, nKV, G, hd, n_pages, shift;
  uint32_t rows_blk, heads_blk, groups;  // rows to a block of columns, heads of each, blocks to a row's heads
  float per_target;                     // KV heads / items wanted
  float split_min;                      // least C
  float q_factor;                       // scale log2 e = q_factor 2^c_exp, 0.36 < |q_factor| < 0.73
  int32_t c_exp;
};

// a / b of a < 2^20 by a reciprocal: (a + 1/2) / b is 1 / 2b away from the next
// whole number and off by less than a / b 2^-22
__device__ __forceinline__ uint32_t small_quotient(uint32_t a, uint32_t b) {
  return (uint32_t)(((float)a + 0.5f) * __builtin_amdgcn_rcpf((float)b));
}
__device__ __forceinline__ uint32_t quotient(uint32_t a, uint32_t b) { return a < 1u << 20 ? small_quotient(a, b) : a / b; }
__device__ __forceinline__ uint32_t div_up(uint32_t a, uint32_t b) { return quotient(a + b - 1, b); }
// of values that are the same in all lanes, in scalar registers
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
__device__ __forceinline__ uint32_t quotient_u(uint32_t a, uint32_t b) { return uniform(quotient(a, b)); }

// a partial's words cross from one XCD's L2 to another's: written and read
// through to the agent's coherence point
__device__ __forceinline__ void put2(float* p, float a, float b) {
  __hip_atomic_store((uint64_t*)p, ((uint64_t)__float_as_uint(b) << 32) | __float_as_uint(a), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float* p) {
  const uint64_t v = __hip_atomic_load((uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// Request b's first row, rows and length; no rows if they do not fit, or if
// row_start does not end in the rows there are.
__device__ __forceinline__ void request(const AttArgs& a, uint32_t b, bool tell, uint32_t& r0, uint32_t& n, uint32_t& len) {
  int32_t s = (int32_t)b, e = s + 1;
  if (a.row_start) {
    s = a.row_start[b];
    e = a.row_start[b + 1];
    const int32_t total = a.row_start[a.n_req];
    if (total < 0 || (uint32_t)total > a.max_rows) {
      if (tell && b == 0) paged_err(a.err, PAGED_ERR_ATT_ROWS, (uint32_t)total);
      tell = false;
      e = -1;
    }
  }
  const int32_t l = a.lens[b];
  r0 = (uint32_t)s;
  n = (uint32_t)(e - s);
  len = (uint32_t)l;
  const bool fits = s >= 0 && e >= s && (uint32_t)e <= a.max_rows &&
                    (s == e || (l >= 0 && (!a.row_start || len >= n) && (uint64_t)len <= ((uint64_t)a.max_pages << a.shift)));
  if (!fits) {
    if (tell) paged_err(a.err, PAGED_ERR_ATT_LENGTH, b);
    n = 0;
    len = 0;
  }
}

// The items of a call, from what each workgroup works out in LDS.  Which comes when
// matters where a workgroup gets two and where two share a CU (a grid of two to a
// CU puts workgroups i and i + CUS on one).  Blocks of many columns (SORT) of up to
// 64 requests, more than CUS of them and none cut: the longest first, and the
// second CUS in reverse.  4 prompts of 1000 rows, 16 heads of 128, microseconds by
// requests and so: f16 62, 56, bf16 81, 70, f32 194, 154; 8 of 16 heads of 64 on 4 KV
// heads 56, 46 | 70, 53 | 155, 132.  (To look an item up costs a microsecond more:
// one row a request loses 3 to 8 % by it, 20 mixed requests that are cut 5 % in f16.)
// Else by the request, those of the long ones (half of C keys and more) before the
// others.
#define CUS 256u
template <bool SORT>
struct Items {
  // [n_req + 1] of a request: its first item of its class (in the other class's
  // array the next request's), or its first level and its blocks of rows; its
  // first partial, its first row, its length
  uint32_t *longs, *shorts, *part, *row, *len;
  struct Head {
    uint32_t total_long;
    uint32_t levels;  // 0: not sorted
    float inv_c;
    uint32_t pad;
  }* head;  // of SORT, read where an item is looked up: registers for it cost the key loop spills
  uint32_t total, total_long;
  float inv_c;

  static __device__ __forceinline__ uint32_t splits(uint32_t keys, float inv_c) {  // of at most about 5/4 C keys
    const uint32_t s = (uint32_t)((float)keys * inv_c * 0.8f + 0.999f);
    return s < 1 ? 1u : s > PAGED_SPLIT_MAX ? PAGED_SPLIT_MAX : s;
  }
  static __device__ __forceinline__ bool is_long(uint32_t keys, float inv_c) { return (float)keys * inv_c >= 0.5f; }
};

template <bool SORT>
__device__ __forceinline__ void find_items(const AttArgs& a, uint32_t* lds, Items<SORT>& t) {
  t.head = (typename Items<SORT>::Head*)lds;
  t.longs = lds + sizeof(typename Items<SORT>::Head) / 4;
  t.shorts = t.longs + a.n_req + 1;
  t.part = t.shorts + a.n_req + 1;
  t.row = t.part + a.n_req + 1;
  t.len = t.row + a.n_req + 1;
  const uint32_t tid = threadIdx.x, lane = tid & 63, w = tid >> 6, RB = a.rows_blk, groups = a.groups;
  float inv_c = 0.f;
  uint32_t levels = 0, total_long = 0;
  auto set_work = [&](float work) { inv_c = 1.0f / fmaxf(work * a.per_target, a.split_min); };
  auto put_head = [&] {
    t.total_long = total_long;
    t.inv_c = inv_c;
    if (SORT) *t.head = typename Items<SORT>::Head{total_long, levels, inv_c, 0u};
  };
  if (a.n_req <= 64) {
    // every wave for itself, request to lane: no barriers (they all write the same)
    uint32_t r0 = 0, n = 0, len = 0;
    if (lane < a.n_req) request(a, lane, blockIdx.x == 0, r0, n, len);
    const uint32_t blocks = div_up(n, RB) * groups;
    set_work(sum64_lanes((float)blocks * (float)len));
    const uint32_t ns = t.splits(len, inv_c), it = blocks * a.nKV * ns;
    const bool lg = t.is_long(len, inv_c);
    const uint32_t il = scan64_lanes(lg ? it : 0u), is = scan64_lanes(lg ? 0u : it), ip = scan64_lanes(ns > 1 ? it : 0u);
    total_long = (uint32_t)__builtin_amdgcn_readlane((int)il, 63);
    t.total = total_long + (uint32_t)__builtin_amdgcn_readlane((int)is, 63);
    uint32_t first = il - (lg ? it : 0u), second = is - (lg ? 0u : it);
    if (SORT && t.total > CUS && !__builtin_amdgcn_readlane((int)ip, 63)) {
      // the level of a request's last rows: by how many blocks' rows it is shorter
      // than the longest
      const uint32_t keys = blocks ? len : 0u;
      first = (uint32_t)((float)(max64_lanes(keys) - keys) * __builtin_amdgcn_rcpf((float)RB));
      second = div_up(n, RB);
      levels = uniform(max64_lanes(blocks ? first + second : 0u));
    }
    put_head();
    if (lane < a.n_req) {
      t.longs[lane] = first;
      t.shorts[lane] = second;
      t.part[lane] = ip - (ns > 1 ? it : 0u);
      t.row[lane] = r0;
      t.len[lane] = len;
      if (lane + 1 == a.n_req) t.row[a.n_req] = r0 + n;
    }
    return;
  }
  __shared__ float s_sum[4];
  __shared__ uint32_t s_wave[4][3];
  const uint32_t per = (a.n_req + 255) / 256;
  float work = 0.f;  // only a measure of how much there is: the cuts hold for any
  for (uint32_t k = 0; k < per; k++) {
    const uint32_t b = tid * per + k;
    if (b >= a.n_req) break;
    uint32_t r0, n, len;
    request(a, b, blockIdx.x == 0, r0, n, len);
    t.row[b] = r0;
    t.len[b] = len;
    t.longs[b] = n;
    work = __builtin_fmaf((float)(div_up(n, RB) * groups), (float)len, work);
  }
  work = sum64_lanes(work);
  if (lane == 0) s_sum[w] = work;
  __syncthreads();
  set_work((s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]));
  uint32_t longs = 0, shorts = 0, parts = 0;
  for (uint32_t k = 0; k < per; k++) {
    const uint32_t b = tid * per + k;
    if (b >= a.n_req) break;
    const uint32_t ns = t.splits(t.len[b], inv_c), it = div_up(t.longs[b], RB) * groups * a.nKV * ns;
    (t.is_long(t.len[b], inv_c) ? longs : shorts) += it;
    parts += ns > 1 ? it : 0;
  }
  uint32_t il = scan64_lanes(longs), is = scan64_lanes(shorts), ip = scan64_lanes(parts);
  if (lane == 63) {
    s_wave[w][0] = il;
    s_wave[w][1] = is;
    s_wave[w][2] = ip;
  }
  __syncthreads();
  t.total = total_long = 0;
  il -= longs;
  is -= shorts;
  ip -= parts;
#pragma unroll
  for (uint32_t k = 0; k < 4; k++) {
    if (k < w) {
      il += s_wave[k][0];
      is += s_wave[k][1];
      ip += s_wave[k][2];
    }
    total_long += s_wave[k][0];
    t.total += s_wave[k][1];
  }
  t.total += total_long;
  put_head();
  if (blockIdx.x >= t.total) return;
  for (uint32_t k = 0; k < per; k++) {
    const uint32_t b = tid * per + k;
    if (b >= a.n_req) break;
    const uint32_t ns = t.splits(t.len[b], inv_c), n = t.longs[b], it = div_up(n, RB) * groups * a.nKV * ns;
    const bool lg = t.is_long(t.len[b], inv_c);
    t.longs[b] = il;
    t.shorts[b] = is;
    t.part[b] = ip;
    if (b + 1 == a.n_req) t.row[a.n_req] = t.row[b] + n;
    (lg ? il : is) += it;
    ip += ns > 1 ? it : 0;
  }
  __syncthreads();
}

// One item, the same in all lanes: columns (row, head) of a request, numbered
// row by row, and the keys k0 .. k1 - 1 of those that they see.
struct Item {
  uint32_t b, r0, n, len, kvh, split, ns, row0, rows, head0, heads, ncols;
  uint32_t keys, least;  // keys that the block's last and first row see
  uint32_t k0, k1;
  uint32_t part;  // of ns > 1: its partial; a block's next split has the one nKV further on

  template <bool SORT>
  __device__ __forceinline__ Item(const AttArgs& a, const Items<SORT>& t, uint32_t item, uint32_t CB, uint32_t unit) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t blk, rowblk;
    uint32_t levels = 0, total_long = t.total_long;
    float inv_c = t.inv_c;
    if (SORT) {
      levels = uniform(t.head->levels);
      total_long = uniform(t.head->total_long);
      inv_c = __uint_as_float(uniform(__float_as_uint(t.head->inv_c)));
    }
    if (SORT && levels) {
      // The request's keys fall by a block's rows from one level to the next, the
      // longest's last block being level 0: N(L) = sum over requests of the levels
      // that they have before L is the number of blocks before level L.
      const bool in = lane < a.n_req;
      const uint32_t from = in ? t.longs[lane] : 0u, deep = in ? t.shorts[lane] : 0u;
      const uint32_t rest = quotient_u(item, a.nKV);
      kvh = item - rest * a.nKV;
      uint32_t lo = 0, hi = levels, before = 0;  // N(lo) <= rest < N(hi)
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1, at = mid > from ? mid - from : 0u;
        const uint32_t N =
            (uint32_t)__builtin_amdgcn_readlane((int)scan64_lanes((at < deep ? at : deep) * a.groups), 63);
        if (N <= rest) {
          lo = mid;
          before = N;
        } else {
          hi = mid;
        }
      }
      const uint32_t here = lo >= from && lo - from < deep ? a.groups : 0u, upto = scan64_lanes(here), d = rest - before;
      b = (uint32_t)__popcll(__ballot(upto <= d));
      const uint32_t group = d - (uint32_t)__builtin_amdgcn_readlane((int)(upto - here), (int)b);
      r0 = uniform(t.row[b]);
      len = uniform(t.len[b]);
      n = a.row_start ? uniform(t.row[b + 1]) - r0 : 1u;
      ns = 1;
      split = 0;
      part = 0;
      rowblk = (uint32_t)__builtin_amdgcn_readlane((int)deep, (int)b) - 1 -
               (lo - (uint32_t)__builtin_amdgcn_readlane((int)from, (int)b));
      blk = rowblk * a.groups + group;
    } else {
      // the last request that starts at or before the item (those without items of
      // its class start there too)
      const uint32_t* from = item < total_long ? t.longs : t.shorts;
      if (item >= total_long) item -= total_long;
      uint32_t lo = 0;
      if (a.n_req > 64) {  // which 64 of them, then which one
        const uint32_t k = lane * 64;
        lo = 64 * (uint32_t)__popcll(__ballot(k < a.n_req && from[k < a.n_req ? k : 0] <= item)) - 64;
      }
      const uint32_t k = lo + lane;
      b = uniform(lo + (uint32_t)__popcll(__ballot(k < a.n_req && from[k < a.n_req ? k : 0] <= item)) - 1);
      r0 = uniform(t.row[b]);
      len = uniform(t.len[b]);
      const uint32_t local = item - uniform(from[b]);
      part = uniform(t.part[b]) + local;
      n = a.row_start ? uniform(t.row[b + 1]) - r0 : 1u;
      ns = uniform(t.splits(len, inv_c));
      // the KV head first (neighbouring blocks of a head meet in one XCD's L2 when
      // there are 8 of them), the blocks with the most keys before the others (a
      // request that is cut has no more items than there is room for partials)
      const uint32_t rest = quotient_u(local, a.nKV), later = ns > 1 ? uniform(small_quotient(rest, ns)) : rest;
      kvh = local - rest * a.nKV;
      split = rest - later * ns;
      blk = quotient_u(n + a.rows_blk - 1, a.rows_blk) * a.groups - 1 - later;
      rowblk = quotient_u(blk, a.groups);
    }
    head0 = (blk - rowblk * a.groups) * CB;
    heads = a.G - head0 < a.heads_blk ? a.G - head0 : a.heads_blk;
    head0 += kvh * a.G;
    row0 = rowblk * a.rows_blk;
    rows = n - row0 < a.rows_blk ? n - row0 : a.rows_blk;
    ncols = rows * heads;
    // row i of the request sees len - n + i + 1 keys (a lone row without keys none)
    keys = len - n + row0 + rows;
    least = len - n + row0 + 1;
    const uint32_t chunk = ns > 1 ? (quotient_u(keys + ns - 1, ns) + unit - 1) / unit * unit : keys;
    const uint64_t at = (uint64_t)split * chunk;
    k0 = at < keys ? (uint32_t)at : keys;
    k1 = keys - k0 < chunk ? keys : k0 + chunk;
  }
  __device__ __forceinline__ uint32_t row_of(uint32_t col) const { return small_quotient(col, heads); }
  // element 0 of a column in q or out
  __device__ __forceinline__ size_t at(uint32_t col, uint32_t ld, uint32_t hd) const {
    const uint32_t row = row_of(col);
    return (size_t)(r0 + row0 + row) * ld + (head0 + col - row * heads) * hd;
  }
};

// The workgroup's next item: its own number first, then whichever is next, so
// that workgroups with short items take more of them.  take() when an item's keys
// are through (thread 0's atomic is under way while the waves are joined; ahead of
// the keys every load would wait for it), next() by all at its end.  As many are
// taken as there are items; the last one taken clears the queue for the next call.
struct Turn {
  uint32_t item = blockIdx.x, taken = 0;
  bool more;
  __device__ __forceinline__ Turn(uint32_t total, bool sort) {
    if (!sort) return;
    const uint32_t first = total < gridDim.x ? total : gridDim.x;
    const uint32_t eights = first > CUS ? (first - CUS) / 8 : 0, j = item - CUS;
    if (item >= CUS && j / 8 < eights) item = uniform(CUS + (eights - 1 - j / 8) * 8 + j % 8);
    item = uniform(item);
  }
  __device__ __forceinline__ void take(const AttArgs& a, uint32_t total) {
    more = total > gridDim.x;
    if (more && threadIdx.x == 0) taken = __hip_atomic_fetch_add(a.queue, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __device__ __forceinline__ void next(const AttArgs& a, uint32_t total) {
    __shared__ uint32_t s_next;
    item = total;
    if (!more) return;
    if (threadIdx.x == 0) {
      s_next = taken + gridDim.x;
      if (taken == total - 1) __hip_atomic_store(a.queue, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    item = (uint32_t)__builtin_amdgcn_readfirstlane((int)s_next);
    __syncthreads();  // everybody's copy is taken (and LDS free for the next item)
  }
};

// A split is through: its partial [CB][hd] and (m, l) [CB] are written by all of
// the workgroup.  True in the last split of the block, which joins them.
__device__ __forceinline__ bool last_split(const AttArgs& a, const Item& I) {
  __shared__ uint32_t s_last;
  uint32_t* done = a.counters + (I.part - I.split * a.nKV);
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    s_last = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == I.ns - 1;
    if (s_last) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return s_last;
}

template <uint32_t N_>
struct Count {
  static constexpr uint32_t N = N_;
};

// A block of at most 16 columns.  s: LDS of PAGED_SPLIT_MAX * 16 + 128 floats that
// nobody uses any more.
__device__ __forceinline__ void join_16(const AttArgs& a, const Item& I, float* s) {
  constexpr uint32_t CB = 16;
  if (!last_split(a, I)) return;
  const uint32_t tid = threadIdx.x, lane = tid & 63, w = tid >> 6, ln = lane & 15, lg = lane >> 4;
  const uint32_t hd = a.hd, ns = I.ns, ncols = I.ncols, first = I.part - I.split * a.nKV;
  float *s_o = s, *s_ml = s + PAGED_SPLIT_MAX * 16;
  const float* all = a.parts + (size_t)first * CB * (hd + 2);
  const size_t stride = (size_t)a.nKV * CB * (hd + 2);
  // a thread's pair of dims over the splits, JOIN_BATCH loads in flight; behind
  // the last split it again, with a weight of 0.  The first loads and those of (m,
  // l) go out together.
  constexpr uint32_t JOIN_BATCH = 16;
  float2 x[JOIN_BATCH];
  auto load = [&](uint32_t e, uint32_t s0) {
    const float* src = all + (e < ncols * hd ? e : 0);
#pragma unroll
    for (uint32_t j = 0; j < JOIN_BATCH; j++) x[j] = get2(src + (s0 + j < ns ? s0 + j : ns - 1) * stride);
  };
  // weights 2^(m - max) of the splits, 16 threads to a column; 0 behind the last
  constexpr int PER = PAGED_SPLIT_MAX / 16;
  const uint32_t cc = ln < ncols ? ln : 0, sp0 = tid >> 4;
  const float* ml = all + CB * hd + cc * 2;
  float2 v[PER];
  float mx = -__builtin_inff(), sum = 0.f;
#pragma unroll
  for (int k = 0; k < PER; k++) v[k] = get2(ml + (sp0 + 16 * k < ns ? sp0 + 16 * k : 0u) * stride);
  load(2 * tid, 0);
#pragma unroll
  for (int k = 0; k < PER; k++) {
    if (sp0 + 16 * k >= ns) v[k] = make_float2(-__builtin_inff(), 0.f);
    mx = fmaxf(mx, v[k].x);
  }
  mx = max_xor16_32(mx);
  if (lg == 0) s_ml[w * 16 + ln] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(s_ml[ln], s_ml[16 + ln]), fmaxf(s_ml[32 + ln], s_ml[48 + ln]));
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const float f = v[k].x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(v[k].x - mx);
    s_o[(sp0 + 16 * k) * 16 + ln] = f;
    sum = __builtin_fmaf(f, v[k].y, sum);
  }
  sum = add_xor32(add_xor16(sum));
  if (lg == 0) s_ml[64 + w * 16 + ln] = sum;
  __syncthreads();
  for (uint32_t e = 2 * tid; e < ncols * hd; e += 512) {
    const uint32_t k = small_quotient(e, hd), d = e - k * hd;
    float2 o = make_float2(0.f, 0.f);
    if (e >= 512) load(e, 0);
    for (uint32_t s0 = 0;;) {
#pragma unroll
      for (uint32_t j = 0; j < JOIN_BATCH; j++) {
        const float f = s_o[(s0 + j) * 16 + k];
        o.x = __builtin_fmaf(f, x[j].x, o.x);
        o.y = __builtin_fmaf(f, x[j].y, o.y);
      }
      s0 += JOIN_BATCH;
      if (s0 >= ns) break;
      load(e, s0);
    }
    const float inv = 1.0f / (s_ml[64 + k] + s_ml[80 + k] + s_ml[96 + k] + s_ml[112 + k]);
    float* y = a.out + I.at(k, a.ld_out, hd) + d;
    y[0] = o.x * inv;
    y[1] = o.y * inv;
  }
}

// Blocks of more columns.  s: LDS of `room` floats, JOIN_ROOM at least, that
// nobody uses any more.
#define JOIN_ROOM (PAGED_SPLIT_MAX * 16 * 2 + 256)
__device__ __forceinline__ void join_many(const AttArgs& a, const Item& I, uint32_t CB, float* s, uint32_t room) {
  if (!last_split(a, I)) return;
  // O is read with ordinary loads, 16 bytes each: nothing of it may be left in the caches
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  const uint32_t tid = threadIdx.x, hd = a.hd, ns = I.ns, ncols = I.ncols, first = I.part - I.split * a.nKV;
  const float* all = a.parts + (size_t)first * CB * (hd + 2);
  const size_t stride = (size_t)a.nKV * CB * (hd + 2);
  // as many columns at once as (m, l) of their splits fit: 16, 32, .. 128
  uint32_t lw = 4;
  while (lw < 7 && (1u << lw) < ncols && (ns << (lw + 2)) + 256 <= room) lw++;
  const uint32_t width = 1u << lw, group = tid >> lw, groups = 256u >> lw;
  float *s_m = s + 256, *s_l = s_m + (ns << lw);  // [ns][width]; s: a number of each thread's
  for (uint32_t c0 = 0; c0 < ncols; c0 += width) {
    // weights 2^(m - max) of the splits: groups of threads, each some splits of all columns
    const uint32_t c = tid & (width - 1);
    const float* ml = all + CB * hd + (c0 + c < ncols ? c0 + c : 0) * 2;
    float mx = -__builtin_inff(), sum = 0.f;
    if (c0) __syncthreads();  // the columns before are through
#pragma unroll 8
    for (uint32_t k = group; k < ns; k += groups) {
      const float2 v = get2(ml + k * stride);
      s_m[(k << lw) + c] = v.x;
      s_l[(k << lw) + c] = v.y;
      mx = fmaxf(mx, v.x);
    }
    s[tid] = mx;
    __syncthreads();
    for (uint32_t k = 0; k < groups; k++) mx = fmaxf(mx, s[(k << lw) + c]);
    for (uint32_t k = group; k < ns; k += groups) {
      const float m = s_m[(k << lw) + c], f = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - mx);
      s_m[(k << lw) + c] = f;
      sum = __builtin_fmaf(f, s_l[(k << lw) + c], sum);
    }
    __syncthreads();
    s[tid] = sum;
    __syncthreads();
    const uint32_t nc = ncols - c0 < width ? ncols - c0 : width;
    auto put = [&](uint32_t e, f32x4 o) {
      const uint32_t k = small_quotient(e, hd);
      float tot = 0.f;
      for (uint32_t g = 0; g < groups; g++) tot += s[(g << lw) + k];
      store4(a.out + I.at(c0 + k, a.ld_out, hd) + (e - k * hd), o * (1.0f / tot));
    };
    // four dims at a time, all loads of 8 such in flight where there are few splits,
    // of 8 splits where there are many; what is behind the last split or dim is
    // loaded as that and weighs 0 or is not written
    const uint32_t quads = nc * hd / 4;
    const float* src = all + c0 * hd;
    auto few = [&](auto splits) {
      constexpr uint32_t NS = decltype(splits)::N;
      for (uint32_t e0 = tid; e0 < quads; e0 += 8 * 256) {
        f32x4 x[8][NS];
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
          for (uint32_t k = 0; k < NS; k++) x[j][k] = load8(src + k * stride + 4 * (e0 + 256 * j < quads ? e0 + 256 * j : quads - 1));
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const uint32_t e = 4 * (e0 + 256 * j);
          if (e >= 4 * quads) break;
          const float* f = s_m + small_quotient(e, hd);
          f32x4 o = x[j][0] * f[0];
#pragma unroll
          for (uint32_t k = 1; k < NS; k++) o += x[j][k] * f[k << lw];
          put(e, o);
        }
      }
    };
    if (ns == 2) {
      few(Count<2>());
    } else if (ns == 3) {
      few(Count<3>());
    } else if (ns == 4) {
      few(Count<4>());
    } else {
      constexpr uint32_t BATCH = 8;
      for (uint32_t e = 4 * tid; e < 4 * quads; e += 4 * 256) {
        const uint32_t k = small_quotient(e, hd);
        f32x4 o = (f32x4){0.f, 0.f, 0.f, 0.f};
        for (uint32_t s0 = 0; s0 < ns; s0 += BATCH) {
          f32x4 x[BATCH];
#pragma unroll
          for (uint32_t j = 0; j < BATCH; j++) x[j] = load8(src + (s0 + j < ns ? s0 + j : ns - 1) * stride + e);
#pragma unroll
          for (uint32_t j = 0; j < BATCH; j++) o += x[j] * (s0 + j < ns ? s_m[((s0 + j) << lw) + k] : 0.f);
        }
        put(e, o);
      }
    }
  }
}

#define MERGE_PAD 4  // floats between the columns of a wave's O in LDS

// 2^e, never 0 or infinite
__device__ __forceinline__ float score_factor(int e) {
  e = e < -126 ? -126 : e > 127 ? 127 : e;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Scores of one column (times c: in powers of two) become weights 2^(score - m):
// follow() moves the column's m, with its sum l (this lane's share) and O, and says
// what is added to a score; weight() is one of them.
template <class TILE, int NJ, int DPL>
__device__ __forceinline__ float follow(const f32x4 (&S)[NJ], float c, float& m, float& l, f32x4 (&O)[DPL]) {
  float x = -__builtin_inff();
#pragma unroll
  for (int j = 0; j < NJ; j++)
#pragma unroll
    for (int i = 0; i < 4; i++) x = fmaxf(x, S[j][i]);
  x = max_xor16_32(x) * c;
  if (__any(x - m > TILE::P_TOP)) {
    const float mn = fmaxf(x - (fabsf(x) > FAR_SCORE ? 0.f : TILE::P_EXP), m);
    const float f = mn == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= f;
#pragma unroll
    for (int d = 0; d < DPL; d++) O[d] *= f;
  }
  return m == -__builtin_inff() ? 0.f : -m;
}
__device__ __forceinline__ float weight(float s, float c, float shift, float& l) {
  const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s, c, shift));
  l += p;
  return p;
}
template <class TILE, int NJ, int DPL>
__device__ __forceinline__ void weigh(f32x4 (&S)[NJ], float c, float& m, float& l, f32x4 (&O)[DPL]) {
  const float shift = follow<TILE, NJ, DPL>(S, c, m, l, O);
#pragma unroll
  for (int j = 0; j < NJ; j++)
#pragma unroll
    for (int i = 0; i < 4; i++) S[j][i] = weight(S[j][i], c, shift, l);
}

// The kernel's arguments, read again: held over the key loops they take scalar
// registers and then lanes of vector registers (16 columns of f16, 128 dims: 230
// and 49 spilled scalars, so 203 and none; one row behind 1024 keys 10.3 and 9.7 us),
// or reloads in every stage behind the DMA (three-part weights of 128 dims).
__device__ __forceinline__ const AttArgs& again() {
  typedef const AttArgs __attribute__((address_space(4))) Kernarg;
  Kernarg* p = (Kernarg*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const AttArgs*)p;
}

// One tile of 16 columns to a workgroup.  Its four waves take the keys in turn, TK
// at a time, straight from the pages into the operands' registers, the next
// tile's while this one's are multiplied, and are joined through LDS at the end.
// For one row a request: bound by memory.  32 heads on 8 of 128 dims: 120 requests
// of 2800 to 4000 keys in bf16 (1.67 GB) 302 us, 5.5 TB/s; one of 131071 in f16 101
// us, 5.3 TB/s (a large copy: 4.8); 32 of 1 to 6000 31.1 us, 4.1 TB/s.  One of 517
// f32 keys, 16 heads of 64: 8.9 us, latency.  More waves to a CU (3 and 4
// workgroups by launch bounds) spill into scratch, whose loads wait for the
// keys': 64 requests of 4000 keys 178 us with 2, 193 with 3, 269 with 4.
template <class TILE, int DPL, bool SMALL>
__device__ __forceinline__ void attention_body(const AttArgs& args) {
  typedef typename TILE::T T;
  constexpr int NJ = TILE::NJ, QREG = TILE::QREG;
  constexpr uint32_t TK = 16 * NJ, HDP = 16 * DPL, CB = 16;
  constexpr uint32_t OS = HDP + MERGE_PAD;
  constexpr uint32_t OFLOATS = 4 * 16 * OS;
  static_assert(QREG * 64 * 4 <= OFLOATS && PAGED_SPLIT_MAX * 16 + 128 <= OFLOATS, "Q, and the weights of a join, fit where O does");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  u32x4* s_q = (u32x4*)lds;  // Q [QREG][64 lanes], until the keys are through; then
  float* s_o = (float*)lds;  // [4 waves][16 columns][OS]
  float* s_ml = s_o + OFLOATS;  // [4 waves][16 columns][m, l]
  const uint32_t tid = threadIdx.x, lane = tid & 63, w = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t ln = lane & 15, lg = lane >> 4;
  Items<false> items;
  find_items(args, (uint32_t*)(s_ml + 4 * 16 * 2), items);

  for (Turn turn(items.total, false); turn.item < items.total; turn.next(again(), items.total)) {
    const AttArgs& a = again();
    const uint32_t P = 1u << a.shift, hd = a.hd;
    const Item I(a, items, turn.item, CB, TK);
    const uint32_t k0 = I.k0, k1 = I.k1, kvh = I.kvh;
    f32x4 q_raw[TILE::QRAW];
    TILE::load_q(a.q + I.at(ln < I.ncols ? ln : 0, a.ld_q, hd), lg, hd, q_raw);

    // ---- this wave's keys, a tile's loads in flight before it is needed ----
    TILE tile;
    const int32_t* table = a.tables + (size_t)I.b * a.max_pages;
    const size_t head_len = (size_t)hd << a.shift;  // values of a page's KV head
    uint32_t bad = 0;
    auto page_of = [&](uint32_t t) {  // of key t < k1
      const uint32_t p = (uint32_t)table[t >> a.shift];
      bad |= (uint32_t)(p >= a.n_pages);
      return p < a.n_pages ? p : 0u;
    };
    auto address = [&](uint32_t page, uint32_t t) {
      return ((size_t)page * a.nKV + kvh) * head_len + (size_t)(t & (P - 1)) * hd;
    };
    // Keys from k1 on are loaded as others of their page, or as key k1 - 1.
    // Pages of 16 keys and more: 16 keys at a multiple of 16 lie in one, whose
    // address is the wave's; a lane holds the page of such 16 keys for the next
    // AHEAD tiles of the wave (lane NJ x + j: tile x, its j-th 16).  Smaller pages:
    // lane x holds key x's of the next tile.
    constexpr uint32_t AHEAD = SMALL ? 1 : 64 / NJ;
    uint32_t t0 = k0 + w * TK, pages = 0, tiles = 0;
    auto load_pages = [&](uint32_t t) {
      const uint32_t k = SMALL ? t + (lane & (TK - 1)) : t + lane / NJ * 4 * TK + lane % NJ * 16;
      pages = page_of(k < k1 ? k : k1 - 1);
    };
    auto load_k = [&](uint32_t t) {
#pragma unroll
      for (int j = 0; j < NJ; j++) {
        if constexpr (SMALL) {
          const uint32_t x = 16 * j + ln, k = t + x < k1 ? t + x : k1 - 1;
          tile.load_k(j, (const T*)a.kpages + address((uint32_t)__shfl((int)pages, (int)(k - t)), k), 0, lg, hd);
        } else {
          const uint32_t p = (uint32_t)__builtin_amdgcn_readlane((int)pages, (int)(tiles * NJ + j));
          tile.load_k(j, (const T*)a.kpages + address(p, t + 16 * j), ln * hd, lg, hd);
        }
      }
    };
    auto load_v = [&](uint32_t t) {
#pragma unroll
      for (int j = 0; j < NJ; j++) {
        if constexpr (SMALL) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t x = 16 * j + 4 * lg + i, k = t + x < k1 ? t + x : k1 - 1;
            tile.load_v(j, i, (const T*)a.vpages + address((uint32_t)__shfl((int)pages, (int)(k - t)), k), 0, ln, hd);
          }
        } else {
          const uint32_t p = (uint32_t)__builtin_amdgcn_readlane((int)pages, (int)(tiles * NJ + j));
#pragma unroll
          for (int i = 0; i < 4; i++) tile.load_v(j, i, (const T*)a.vpages + address(p, t + 16 * j), (4 * lg + i) * hd, ln, hd);
        }
      }
    };
    if (t0 < k1) {
      load_pages(t0);
      load_k(t0);
      load_v(t0);
    }

    float c;
    {
      // each wave splits the steps of its own number
      int e2;
      TILE::split_q(q_raw, ln < I.ncols, lg, hd, a.q_factor, e2,
                    [&](int s) { return (s & 3) == (int)w; }, [&](int k, u32x4 x) { s_q[k * 64 + lane] = x; });
      c = score_factor(a.c_exp - e2);
    }
    __syncthreads();
    const uint32_t limit = I.least + I.row_of(ln);
    f32x4 O[DPL];
    float m = -__builtin_inff(), l = 0.f;
#pragma unroll
    for (int d = 0; d < DPL; d++) O[d] = (f32x4){0.f, 0.f, 0.f, 0.f};

    for (; t0 < k1; t0 += 4 * TK) {
      const bool masked = t0 + TK > I.least || t0 + TK > k1, more = t0 + 4 * TK < k1;
      f32x4 S[NJ];
      asm volatile("" ::: "memory");  // Q is read from LDS here, not kept in registers over the keys
      tile.scores([&](int k) { return s_q[k * 64 + lane]; }, S);
      if (more) {
        if (++tiles == AHEAD) {
          tiles = 0;
          load_pages(t0 + 4 * TK);
        }
        load_k(t0 + 4 * TK);
      }
      if (masked) {
        // the lane's first hidden key behind t0 + 4 lg
        const int end = (int)((limit < k1 ? limit : k1) - t0 - 4 * lg);
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (16 * j + i >= end) S[j][i] = -__builtin_inff();
      }
      weigh<TILE, NJ, DPL>(S, c, m, l, O);
      if (masked) {
        // a weight of 0 does not hide a value that is not finite: values behind
        // the block's keys go to 0, and so do keys with such a value that only
        // some rows see; those rows' sums take it up instead
        uint32_t odd = 0;
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            bool hide = t0 + 16 * j + 4 * lg + i >= k1;
            if (I.rows > 1) {
              const bool some = (__ballot(!hide && !tile.finite_v(j, i)) >> (16 * lg)) & 0xFFFFu;
              odd |= (uint32_t)some << (4 * j + i);
              hide |= some;
            }
            if (hide) tile.zero_v(j, i);
          }
        if (__any(odd)) {
#pragma unroll
          for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              if ((odd >> (4 * j + i) & 1) && t0 + 16 * j + 4 * lg + i < limit) l = __builtin_nanf("");
        }
      }
      tile.add_pv(S, O);
      if (more) load_v(t0 + 4 * TK);
    }
    const AttArgs& z = again();
    if (bad) paged_err(z.err, PAGED_ERR_ATT_PAGE, I.b);
    turn.take(z, items.total);

    // ---- join the waves ----
    l = add_xor32(add_xor16(l));
    __syncthreads();  // s_q and s_ml are free
    if (lg == 0) {
      s_ml[(w * 16 + ln) * 2] = m;
      s_ml[(w * 16 + ln) * 2 + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int d = 0; d < DPL; d++) s_o[(w * 16 + ln) * OS + (4 * lg + i) * DPL + d] = O[d][i];
    __syncthreads();
    const uint32_t col = tid >> 4, at = (tid & 15) * DPL;
    float mx = s_ml[col * 2];
#pragma unroll
    for (int k = 1; k < 4; k++) mx = fmaxf(mx, s_ml[(k * 16 + col) * 2]);
    float sum = 0.f, o[DPL];
#pragma unroll
    for (int d = 0; d < DPL; d++) o[d] = 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float mk = s_ml[(k * 16 + col) * 2];
      const float f = mk == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mk - mx);
      sum = __builtin_fmaf(f, s_ml[(k * 16 + col) * 2 + 1], sum);
#pragma unroll
      for (int d = 0; d < DPL; d++) o[d] = __builtin_fmaf(f, s_o[(k * 16 + col) * OS + at + d], o[d]);
    }
    float* mine = z.parts + (size_t)I.part * CB * (z.hd + 2);
    if (col < I.ncols && at < z.hd) {
      const uint32_t d0 = first_dim<DPL>(tid & 15, z.hd);
      if (I.ns == 1) {
        const float inv = I.keys ? 1.0f / sum : 0.f;
        float* y = z.out + I.at(col, z.ld_out, z.hd) + d0;
        Words<DPL> x;
#pragma unroll
        for (int d = 0; d < DPL; d++) x.w[d] = __float_as_uint(o[d] * inv);
        *(Words<DPL>*)y = x;
      } else {
#pragma unroll
        for (int d = 0; d < DPL; d += 2) put2(mine + col * z.hd + d0 + d, o[d], o[d + 1]);
        if (d0 == 0) put2(mine + CB * z.hd + col * 2, mx, sum);
      }
    }
    if (I.ns > 1) join_16(z, I, s_o);
  }
}

// ---------------------------------------------------------------------------
// Many columns: each of the four waves has CT tiles of 16 columns of its own, Q
// and O^T in registers, and all share the keys, KT at a time through LDS (two
// stages, filled by DMA while the other is multiplied; one barrier a stage).
// A stage's rows are [K row][V row] regions of KT rows in 16-byte chunks, chunk
// c of row r at c ^ swizzle(r), so that the 16 rows that an operand read takes
// lie in different banks; the DMA writes lane after lane, so each lane picks
// its source chunk accordingly.  K operands are read as they lie; f16 and bf16
// values through the transposing LDS read, lane (4k + c) of 16 supplying dims
// 4c .. 4c+3 of the k-th of four keys and receiving one dim of all four.
// Bound by the matrix cores: 2000 rows behind 6000 keys, 32 heads on 8 of 128 dims,
// 229 GFLOP: f16 395 to 450 us, 1020 to 1160 TFLOP/s of split products (a large library
// product: 1097), bf16 510 to 560 us, 1230 to 1350 (1136), f32 1.98 ms, 116 (152).  A wave's
// stage is a chain of 6000 cycles for 2048 of products (f16), so the next stage's
// loads and the next weights go out between products, and shorter prompts wait for
// their longest blocks: four of 430 to 611 rows 42 us in f16, half of that rate.
// ---------------------------------------------------------------------------
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// 16 bytes per lane from base + off to LDS byte address lds + 16 * lane.  In asm
// so that the compiler does not see an LDS write, for which it would wait at the
// next LDS read; there is no destination register, and stage_done() waits.  One
// wait state between the write of M0 and its use; the compiler warns that M0 is
// reserved, and must keep nothing there across this.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2"
      :
      : "s"(lds), "v"(off), "s"(base)
      : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void stage_done() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// CHUNKS 16-byte chunks to a row: the rows whose chunks share a bank, 16 / CHUNKS
// of them in 256 bytes, get different keys
template <uint32_t CHUNKS>
__device__ __forceinline__ uint32_t swizzle(uint32_t r) {
  return CHUNKS >= 16 ? r & 15 : (r / (16 / CHUNKS)) & (CHUNKS - 1);
}

// 16s of dims that a stage's row has room for
template <int DPL>
constexpr uint32_t LINE = DPL <= 4 ? 4 : 8;

template <class MM_, int DPL>
struct Rows16 {
  typedef MM_ MM;
  typedef Tile16<MM, DPL> TILE;
  typedef typename MM::T T;
  static constexpr int CT = 2, KT = 64, NJ = KT / 16, TERMS = MM::TERMS;
  static constexpr uint32_t CHUNKS = 2 * LINE<DPL>, ROWB = 32 * LINE<DPL>;
  // scores of the CT tiles' columns against the stage's keys
  template <class BETWEEN>
  static __device__ __forceinline__ void scores(const uint8_t* k, uint32_t ln, uint32_t lg,
                                                const u32x4 (&Q)[CT][TILE::QREG], f32x4 (&S)[CT][NJ], BETWEEN between) {
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
      for (int j = 0; j < NJ; j++) S[c][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    // 32 keys and 32 dims a step, the next step's operands on their way: products of
    // one sum are CT * 2 apart, which covers the first's latency
    u32x4 x[2][2];
    auto load = [&](int step) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const uint32_t r = 16 * (step / TILE::KS * 2 + j) + ln;
        x[step & 1][j] = *(const u32x4*)(k + r * ROWB + ((4 * (step % TILE::KS) + lg) ^ swizzle<CHUNKS>(r)) * 16);
      }
    };
    constexpr int STEPS = NJ / 2 * TILE::KS;
    load(0);
#pragma unroll
    for (int step = 0; step < STEPS; step++) {
      if (step + 1 < STEPS) load(step + 1);
#pragma unroll
      for (int t = 0; t < TERMS; t++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int c = 0; c < CT; c++) {
            f32x4& sum = S[c][step / TILE::KS * 2 + j];
            sum = MM::mfma(x[step & 1][j], Q[c][step % TILE::KS * TERMS + t], sum);
          }
      between(step, STEPS);
    }
  }
  // O += V^T P^T, 32 keys at a time; the weights of the next 32 are worked out
  // between the products of these
  static __device__ __forceinline__ void add_pv(const uint8_t* v, uint32_t ln, uint32_t lg, f32x4 (&S)[CT][NJ],
                                                const float (&c)[CT], const float (&shift)[CT], float (&l)[CT],
                                                f32x4 (&O)[CT][DPL]) {
    u32x4 p[2][CT][TERMS];
    auto pair = [&](int h, int x) {  // of CT * 4 to 32 keys
      const int t = x / 4, k = x % 4;
      const f32x4 s = S[t][2 * h + k / 2];
      const float a = weight(s[k % 2 * 2], c[t], shift[t], l[t]), b = weight(s[k % 2 * 2 + 1], c[t], shift[t], l[t]);
      MM::split2(a, b, p[h & 1][t], k);
    };
#pragma unroll
    for (int x = 0; x < CT * 4; x++) pair(0, x);
#pragma unroll
    for (int h = 0; h < NJ / 2; h++) {
#pragma unroll
      for (int d = 0; d < DPL; d += 2) {
        u32x4 y[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          u32x2 x[2];
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const uint32_t r = 16 * (2 * h + j) + 4 * lg + ln / 4, cc = ln & 3;
            const uint8_t* at = v + r * ROWB + (((2 * (d + e) + cc / 2) ^ swizzle<CHUNKS>(r)) * 16) + (cc & 1) * 8;
            x[j] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at));
          }
          y[e] = (u32x4){x[0][0], x[0][1], x[1][0], x[1][1]};
        }
#pragma unroll
        for (int t = 0; t < TERMS; t++)
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int c = 0; c < CT; c++) O[c][d + e] = MM::mfma(y[e], p[h & 1][c][t], O[c][d + e]);
        if (h + 1 < NJ / 2) {
#pragma unroll
          for (int x = 0; x < CT * 4; x++)
            if (x * DPL / (CT * 4) / 2 * 2 == d) pair(h + 1, x);
        }
      }
    }
  }
  static __device__ __forceinline__ bool finite(u32x4 x) {
    bool ok = true;
#pragma unroll
    for (int k = 0; k < 4; k++)
      ok = ok && (x[k] & MM::EXPONENT) != MM::EXPONENT && (x[k] & (MM::EXPONENT << 16)) != (MM::EXPONENT << 16);
    return ok;
  }
};

template <int DPL>
struct Rows32 {
  typedef Tile32<DPL> TILE;
  typedef float T;
  static constexpr int CT = 1, KT = 32, NJ = KT / 16;
  static constexpr uint32_t CHUNKS = 4 * LINE<DPL>, ROWB = 64 * LINE<DPL>;
  template <class BETWEEN>
  static __device__ __forceinline__ void scores(const uint8_t* k, uint32_t ln, uint32_t lg,
                                                const u32x4 (&Q)[CT][TILE::QREG], f32x4 (&S)[CT][NJ], BETWEEN between) {
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      f32x4 a = (f32x4){0.f, 0.f, 0.f, 0.f}, b = a;
      const uint32_t r = 16 * j + ln;
#pragma unroll
      for (int s = 0; s < DPL; s++) {
        const f32x4 x = *(const f32x4*)(k + r * ROWB + ((4 * s + lg) ^ swizzle<CHUNKS>(r)) * 16);
        const f32x4 q = __builtin_bit_cast(f32x4, Q[0][s]);
        a = __builtin_amdgcn_mfma_f32_16x16x4f32(x[0], q[0], a, 0, 0, 0);
        b = __builtin_amdgcn_mfma_f32_16x16x4f32(x[1], q[1], b, 0, 0, 0);
        a = __builtin_amdgcn_mfma_f32_16x16x4f32(x[2], q[2], a, 0, 0, 0);
        b = __builtin_amdgcn_mfma_f32_16x16x4f32(x[3], q[3], b, 0, 0, 0);
      }
      S[0][j] = a + b;
      between(j, NJ);
    }
  }
  static __device__ __forceinline__ void add_pv(const uint8_t* v, uint32_t ln, uint32_t lg, f32x4 (&S)[CT][NJ],
                                                const float (&c)[CT], const float (&shift)[CT], float (&l)[CT],
                                                f32x4 (&O)[CT][DPL]) {
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int i = 0; i < 4; i++) S[0][j][i] = weight(S[0][j][i], c[0], shift[0], l[0]);
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int d = 0; d < DPL; d++) {
          const uint32_t r = 16 * j + 4 * lg + i;
          const float x = *(const float*)(v + r * ROWB + (((4 * d + ln / 4) ^ swizzle<CHUNKS>(r)) * 16) + (ln & 3) * 4);
          O[0][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, S[0][j][i], O[0][d], 0, 0, 0);
        }
  }
  static __device__ __forceinline__ bool finite(u32x4 x) {
    bool ok = true;
#pragma unroll
    for (int k = 0; k < 4; k++) ok = ok && (x[k] & 0x7F800000u) != 0x7F800000u;
    return ok;
  }
};

template <class ROWS, int DPL>
__device__ __forceinline__ void attention_rows_body(const AttArgs& args) {
  typedef typename ROWS::TILE TILE;
  typedef typename ROWS::T T;
  constexpr int CT = ROWS::CT, KT = ROWS::KT, NJ = ROWS::NJ, QREG = TILE::QREG;
  constexpr uint32_t CB = 64 * CT, ROWB = ROWS::ROWB, CHUNKS = ROWS::CHUNKS, REGION = KT * ROWB;
  static_assert(JOIN_ROOM * 4 <= 4 * REGION, "the weights of a join fit in the stages");
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];  // [2 stages][K, V][KT rows]
  uint32_t* s_odd = (uint32_t*)(lds + 4 * REGION);                // [2 stages][2] a bit to a key
  const uint32_t tid = threadIdx.x, lane = tid & 63, w = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t ln = lane & 15, lg = lane >> 4;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  Items<true> items;
  find_items(args, s_odd + 4, items);

  for (Turn turn(items.total, true); turn.item < items.total; turn.next(again(), items.total)) {
    const AttArgs& a = again();
    const uint32_t P = 1u << a.shift, hd = a.hd;
    const Item I(a, items, turn.item, CB, KT);
    const uint32_t k0 = I.k0, k1 = I.k1;
    // ---- this wave's share of a stage: KT / 4 rows of K and of V, 8 or 16, a page to 8 ----
    constexpr uint32_t SHARE = KT / 4, RPI = 1024 / ROWB, PARTS = SHARE / 8, INSTR = 8 / RPI;  // rows, instructions to 8 rows
    constexpr uint32_t AHEAD = 64 / PARTS;
    const int32_t* table = a.tables + (size_t)I.b * a.max_pages;
    const size_t head_len = (size_t)hd << a.shift;
    uint32_t bad = 0, pages = 0, ahead = AHEAD;  // lane PARTS x + h: page of this wave's h-th 8 rows x stages on
    const size_t page_bytes = a.nKV * head_len * sizeof(T);
    const uint8_t* const k_head = (const uint8_t*)a.kpages + I.kvh * head_len * sizeof(T);
    const ptrdiff_t to_v = (const uint8_t*)a.vpages - (const uint8_t*)a.kpages;
    auto look_up = [&](uint32_t t, uint32_t lane) {
      if (ahead == AHEAD) {
        const uint32_t k = t + lane / PARTS * KT + w * SHARE + lane % PARTS * 8;
        const uint32_t p = (uint32_t)table[(k < k1 ? k : k1 - 1) >> a.shift];
        bad |= (uint32_t)(p >= a.n_pages);
        pages = p < a.n_pages ? p : 0u;
        ahead = 0;
      }
    };
    // the piece-th of PIECES 16 bytes a lane, of K and of V, of the stage at key t
    constexpr uint32_t PIECES = PARTS * INSTR;
    auto fetch = [&](uint32_t t, uint32_t stage, uint32_t lane, uint32_t piece) {
      const uint32_t h = piece / INSTR, r = piece % INSTR * RPI + lane / CHUNKS;  // row of the part's 8
      const uint32_t p = (uint32_t)__builtin_amdgcn_readlane((int)pages, (int)(ahead * PARTS + h));
      const uint32_t first = t + w * SHARE + 8 * h;  // rows from k1 on: others of the page
      const uint8_t* at = k_head + (p * page_bytes + (size_t)(first & (P - 1)) * (hd * sizeof(T)));
      uint32_t c = (lane % CHUNKS) ^ swizzle<CHUNKS>(w * SHARE + 8 * h + r);
      const uint32_t last = hd * sizeof(T) / 16 - 1;  // past the head: against zeros of Q, into dims that nobody reads
      c = c < last ? c : last;
      const uint32_t off = r * hd * sizeof(T) + c * 16, to = lds0 + stage * 2 * REGION + w * SHARE * ROWB + piece * 1024;
      dma16(at, off, to);
      dma16(at + to_v, off, to + REGION);
    };
    // ---- this wave's columns, their loads ahead of the keys' ----
    f32x4 raw[CT][TILE::QRAW];
#pragma unroll
    for (int t = 0; t < CT; t++) {
      const uint32_t col = (w * CT + t) * 16 + ln;
      TILE::load_q(a.q + I.at(col < I.ncols ? col : 0, a.ld_q, hd), lg, hd, raw[t]);
    }
    __syncthreads();  // the stages and s_odd are free
    if (k0 < k1) {
      look_up(k0, lane);
#pragma unroll
      for (uint32_t x = 0; x < PIECES; x++) fetch(k0, 0, lane, x);
      ahead++;
    }
    u32x4 Q[CT][QREG];
    f32x4 O[CT][DPL];
    float m[CT], l[CT], c[CT];
#pragma unroll
    for (int t = 0; t < CT; t++) {
      const uint32_t col = (w * CT + t) * 16 + ln;
      int e2;
      TILE::split_q(raw[t], col < I.ncols, lg, hd, a.q_factor, e2, [](int) { return true; },
                    [&](int k, u32x4 x) { Q[t][k] = x; });
      c[t] = score_factor(a.c_exp - e2);
      m[t] = -__builtin_inff();
      l[t] = 0.f;
#pragma unroll
      for (int d = 0; d < DPL; d++) O[t][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    const bool some = w * CT * 16 < I.ncols;  // this wave has columns

    uint32_t stage = 0;
    for (uint32_t t0 = k0; t0 < k1; t0 += KT, stage ^= 1) {
      uint8_t* k = lds + stage * 2 * REGION;
      uint8_t* v = k + REGION;
      const bool masked = t0 + KT > I.least || t0 + KT > k1;
      uint32_t* odd = s_odd + 2 * stage;
      if (masked && tid < 2) odd[tid] = 0;
      stage_done();  // this stage is there, and the other one read by all
      // with two tiles of columns the lanes' places are worked out anew for every
      // stage: kept over the loop they cost registers that Q, S and O need (spills,
      // which wait for the DMA)
      uint32_t here = lane;
      if (CT > 1) asm volatile("" : "+v"(here));
      const uint32_t hn = here & 15, hg = here >> 4;
      const bool more = t0 + KT < k1;
      if (more) look_up(t0 + KT, here);
      if (masked) {
        // a weight of 0 does not hide a value that is not finite: values behind
        // the block's keys go to 0, and so do chunks with such a value that only
        // some rows may see; the sums of those rows take it up instead
        for (uint32_t x = tid; x < KT * CHUNKS; x += 256) {
          const uint32_t r = x / CHUNKS;
          u32x4* at = (u32x4*)(v + x * 16);
          const bool hide = t0 + r >= k1;
          if (hide || !ROWS::finite(*at)) {
            *at = (u32x4){0u, 0u, 0u, 0u};
            if (!hide) atomicOr(&odd[r >> 5], 1u << (r & 31));
          }
        }
        __syncthreads();
      }
      // the next stage's loads go out between the products of this one's scores
      auto piece = [&](uint32_t x) {
        if (more) fetch(t0 + KT, stage ^ 1, here, x);
      };
      if (!some) {
#pragma unroll
        for (uint32_t x = 0; x < PIECES; x++) piece(x);
        ahead++;
        continue;
      }
      f32x4 S[CT][NJ];
      float shift[CT];
      ROWS::scores(k, hn, hg, Q, S, [&](int step, int steps) {
#pragma unroll
        for (uint32_t x = 0; x < PIECES; x++)
          if ((int)(x * steps / PIECES) == step) piece(x);
      });
      ahead++;
#pragma unroll
      for (int t = 0; t < CT; t++) {
        if (masked) {
          // the lane's first hidden key behind t0 + 4 lg
          const uint32_t limit = I.least + I.row_of((w * CT + t) * 16 + hn);
          const int end = (int)((limit < k1 ? limit : k1) - t0 - 4 * hg);
          const uint64_t marks = ((uint64_t)(KT > 32 ? odd[1] : 0u) << 32 | odd[0]) >> (4 * hg);
#pragma unroll
          for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (16 * j + i >= end) S[t][j][i] = -__builtin_inff();
          if (__any(marks != 0)) {
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
              for (int i = 0; i < 4; i++)
                if (16 * j + i < end && (marks >> (16 * j + i) & 1)) l[t] = __builtin_nanf("");
          }
        }
        shift[t] = follow<TILE, NJ, DPL>(S[t], c[t], m[t], l[t], O[t]);
      }
      ROWS::add_pv(v, hn, hg, S, c, shift, l, O);
    }
    const AttArgs& z = again();
    if (bad) paged_err(z.err, PAGED_ERR_ATT_PAGE, I.b);
    turn.take(z, items.total);

    // ---- out, or a partial ----
    float* mine = z.parts + (size_t)I.part * CB * (z.hd + 2);
#pragma unroll
    for (int t = 0; t < CT; t++) {
      const uint32_t col = (w * CT + t) * 16 + ln;
      l[t] = add_xor32(add_xor16(l[t]));
      if (col >= I.ncols) continue;
      if (I.ns == 1) {
        const float inv = I.keys ? 1.0f / l[t] : 0.f;
        float* y = z.out + I.at(col, z.ld_out, z.hd) + 4 * lg;
#pragma unroll
        for (int d = 0; d < DPL; d++)
          if (16 * d + 4 * lg < z.hd) store4(y + 16 * d, O[t][d] * inv);
      } else {
#pragma unroll
        for (int d = 0; d < DPL; d++)
          if (16 * d + 4 * lg < z.hd) {
            put2(mine + col * z.hd + 16 * d + 4 * lg, O[t][d][0], O[t][d][1]);
            put2(mine + col * z.hd + 16 * d + 4 * lg + 2, O[t][d][2], O[t][d][3]);
          }
        if (lg == 0) put2(mine + CB * z.hd + col * 2, m[t], l[t]);
      }
    }
    if (I.ns > 1) join_many(z, I, CB, (float*)lds, REGION);
  }
}

#define DEF_ATTENTION(NAME, BODY, ...)                             \
  extern "C" __global__ __launch_bounds__(256, 2) void NAME(AttArgs a) { \
    BODY<__VA_ARGS__>(a);                                          \
  }
// Named by page type and head dims held (64, 96 or 128); _s for pages of less than
// 16 keys.  Heads of 96 (12 on 4) held as 96 dims against 128: 100 requests of 4000 keys,
// f32, 231 against 243 us, f16 115 and 116; 20 mixed requests of up to 1500, f32, 37 and
// 42, f16 25 and 28; a prompt of 1300 rows 76 and 75 (f32), 35 and 37 (f16), 38 and 48
// (bf16).
#define DEF_ATTENTIONS(TYPE, D, DPL, TILE, ROWS)                                                 \
  DEF_ATTENTION(smith_paged_attention_##TYPE##_d##D, attention_body, TILE, DPL, false)           \
  DEF_ATTENTION(smith_paged_attention_##TYPE##_d##D##_s, attention_body, TILE, DPL, true)        \
  DEF_ATTENTION(smith_paged_attention_rows_##TYPE##_d##D, attention_rows_body, ROWS, DPL)
typedef Tile16<MmF16, 4> TileF16d64;
typedef Tile16<MmF16, 6> TileF16d96;
typedef Tile16<MmF16, 8> TileF16d128;
typedef Tile16<MmBf16, 4> TileBf16d64;
typedef Tile16<MmBf16, 6> TileBf16d96;
typedef Tile16<MmBf16, 8> TileBf16d128;
typedef Rows16<MmF16, 4> RowsF16d64;
typedef Rows16<MmF16, 6> RowsF16d96;
typedef Rows16<MmF16, 8> RowsF16d128;
typedef Rows16<MmBf16, 4> RowsBf16d64;
typedef Rows16<MmBf16, 6> RowsBf16d96;
typedef Rows16<MmBf16, 8> RowsBf16d128;
DEF_ATTENTIONS(f32, 64, 4, Tile32<4>, Rows32<4>)
DEF_ATTENTIONS(f32, 96, 6, Tile32<6>, Rows32<6>)
DEF_ATTENTIONS(f32, 128, 8, Tile32<8>, Rows32<8>)
DEF_ATTENTIONS(f16, 64, 4, TileF16d64, RowsF16d64)
DEF_ATTENTIONS(f16, 96, 6, TileF16d96, RowsF16d96)
DEF_ATTENTIONS(f16, 128, 8, TileF16d128, RowsF16d128)
DEF_ATTENTIONS(bf16, 64, 4, TileBf16d64, RowsBf16d64)
DEF_ATTENTIONS(bf16, 96, 6, TileBf16d96, RowsBf16d96)
DEF_ATTENTIONS(bf16, 128, 8, TileBf16d128, RowsBf16d128)
