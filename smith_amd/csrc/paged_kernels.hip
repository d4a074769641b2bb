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

#include "paged_attention.h"

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
// Attention over all keys of a request
// ---------------------------------------------------------------------------
DEF_ALL_ATTENTIONS(, ALL)
