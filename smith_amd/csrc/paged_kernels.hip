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

// One 64-bit word of host-mapped memory: (code, argument), the first one kept.
__device__ __forceinline__ void paged_err(uint64_t* __restrict__ err, uint32_t code, uint32_t arg) {
  if (__hip_atomic_load(err, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM) == 0u)
    __hip_atomic_store(err, ((uint64_t)arg << 32) | code, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
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
// itself (they are a few KB, in L2) and then serves its PLAN_ROWS rows: a
// row's request by bisection, its page from the table or, if it is a new one,
// from the free list; the row that opens a page writes the table entry.
// ---------------------------------------------------------------------------
#define PLAN_THREADS 256

extern "C" __global__ __launch_bounds__(PLAN_THREADS) void smith_paged_plan(
    const int32_t* __restrict__ cached, const int32_t* __restrict__ added, uint32_t n_req,
    const int32_t* __restrict__ free_pages, const int32_t* __restrict__ free_count, uint32_t n_pages, uint32_t shift,
    uint32_t max_pages, uint32_t max_rows, int32_t* __restrict__ tables, int32_t* __restrict__ row_start,
    int32_t* __restrict__ lens, int32_t* __restrict__ slots, int32_t* __restrict__ positions,
    int32_t* __restrict__ free_left, uint64_t* __restrict__ err) {
  __shared__ uint32_t s_row[PAGED_MAX_REQ + 1], s_page[PAGED_MAX_REQ];
  __shared__ uint64_t s_wr[PLAN_THREADS / 64], s_wp[PLAN_THREADS / 64];
  __shared__ uint32_t s_bad[PLAN_THREADS / 64];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t P = 1u << shift;
  const uint64_t cap = (uint64_t)max_pages << shift;
  const uint32_t per = (n_req + PLAN_THREADS - 1) / PLAN_THREADS;
  const int64_t have = free_count[0];
  // this thread's requests: rows and new pages (64-bit sums: nothing wraps)
  uint64_t rows = 0, pages = 0;
  uint32_t bad = 0;  // 1 + the first request whose lengths do not fit
  for (uint32_t k = 0; k < per; k++) {
    const uint32_t b = tid * per + k;
    if (b >= n_req) break;
    const int64_t c = cached[b], a = added[b];
    if ((c < 0 || a < 0 || (uint64_t)(c + a) > cap) && !bad) bad = b + 1;
    if (bad) break;
    rows += (uint64_t)a;
    pages += ((uint64_t)(c + a + P - 1) >> shift) - ((uint64_t)(c + P - 1) >> shift);
  }
  // prefix sums over the workgroup
  uint64_t ir = rows, ip = pages;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t r = __shfl_up(ir, d), p = __shfl_up(ip, d);
    if (lane >= (uint32_t)d) {
      ir += r;
      ip += p;
    }
  }
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
                        : have < 0 || have > (int64_t)n_pages || tp > (uint64_t)have ? PAGED_ERR_PLAN_PAGES
                                            : 0u;
  if (code && blockIdx.x == 0 && tid == 0) paged_err(err, code, bad_req ? bad_req - 1 : code == PAGED_ERR_PLAN_ROWS ? max_rows : (uint32_t)have);
  br += ir - rows;
  bp += ip - pages;
  for (uint32_t k = 0; k < per; k++) {
    const uint32_t b = tid * per + k;
    if (b >= n_req) break;
    const int64_t c = cached[b], a = code ? 0 : added[b];
    if (!code) {
      s_row[b] = (uint32_t)br;
      s_page[b] = (uint32_t)bp;
    }
    if (blockIdx.x == 0) {
      row_start[b] = code ? 0 : (int32_t)br;
      lens[b] = (int32_t)(c + a);
    }
    br += (uint64_t)a;
    if (!code) bp += ((uint64_t)(c + a + P - 1) >> shift) - ((uint64_t)(c + P - 1) >> shift);
  }
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
    const uint32_t c = (uint32_t)cached[lo], p = c + (r - s_row[lo]);
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
// (two 16-byte loads of x, one each of cos and sin), or eight elements of v.
// ---------------------------------------------------------------------------
template <bool VEC>
__device__ __forceinline__ f32x4 load4(const float* p) {
  if (VEC) return *(const f32x4*)p;
  return (f32x4){p[0], p[1], p[2], p[3]};
}
template <bool VEC>
__device__ __forceinline__ void store4(float* p, f32x4 v) {
  if (VEC) {
    *(f32x4*)p = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = v[i];
  }
}
template <class KV>
__device__ __forceinline__ void put4(typename KV::T* p, f32x4 v) {
  typedef typename KV::T T4 __attribute__((ext_vector_type(4)));
  T4 t;
#pragma unroll
  for (int i = 0; i < 4; i++) t[i] = KV::down(v[i]);
  *(T4*)p = t;
}

template <class KV, bool VEC>
__device__ __forceinline__ void append_body(const float* qkv, uint32_t ld, const int32_t* __restrict__ slots,
                                            const int32_t* __restrict__ positions, uint32_t nH, uint32_t nKV,
                                            uint32_t hd, uint32_t rope, const float* __restrict__ cosT,
                                            const float* __restrict__ sinT, uint32_t rope_len,
                                            typename KV::T* __restrict__ kpages, typename KV::T* __restrict__ vpages,
                                            uint32_t n_slots, uint32_t shift, float* q_out, uint32_t ld_q,
                                            uint64_t* __restrict__ err) {
  const uint32_t r = blockIdx.y, item = blockIdx.x * 256 + threadIdx.x;
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
    f32x4 x0 = load4<VEC>(x + e0), x1 = load4<VEC>(x + e0 + half);
    if (rope) {
      const size_t a = (size_t)(uint32_t)pos * half + t;
      const f32x4 c = load4<VEC>(cosT + a), s = load4<VEC>(sinT + a);
      const f32x4 y0 = x0 * c - x1 * s;
      x1 = x0 * s + x1 * c;
      x0 = y0;
    }
    if (isq) {
      store4<VEC>(q_out + (size_t)r * ld_q + e0, x0);
      store4<VEC>(q_out + (size_t)r * ld_q + e0 + half, x1);
    } else {
      put4<KV>(kpages + at(e0), x0);
      put4<KV>(kpages + at(e0 + half), x1);
    }
  } else if (item < nq + 2 * nk) {
    const uint32_t e = 8 * (item - nq - nk);
    const float* x = row + Wq + Wk + e;
    put4<KV>(vpages + at(e), load4<VEC>(x));
    put4<KV>(vpages + at(e) + 4, load4<VEC>(x + 4));
  }
}

#define DEF_APPEND(NAME, KV, VEC)                                                                                   \
  extern "C" __global__ __launch_bounds__(256) void NAME(                                                          \
      const float* qkv, uint32_t ld, const int32_t* __restrict__ slots, const int32_t* __restrict__ positions,      \
      uint32_t nH, uint32_t nKV, uint32_t hd, uint32_t rope, const float* __restrict__ cosT,                        \
      const float* __restrict__ sinT, uint32_t rope_len, KV::T* __restrict__ kpages, KV::T* __restrict__ vpages,    \
      uint32_t n_slots, uint32_t shift, float* q_out, uint32_t ld_q, uint64_t* __restrict__ err) {                  \
    append_body<KV, VEC>(qkv, ld, slots, positions, nH, nKV, hd, rope, cosT, sinT, rope_len, kpages, vpages, n_slots, \
                         shift, q_out, ld_q, err);                                                                  \
  }
DEF_APPEND(smith_paged_append_f32, KvF32, true)
DEF_APPEND(smith_paged_append_f16, KvF16, true)
DEF_APPEND(smith_paged_append_bf16, KvBf16, true)
DEF_APPEND(smith_paged_append_f32_u, KvF32, false)
DEF_APPEND(smith_paged_append_f16_u, KvF16, false)
DEF_APPEND(smith_paged_append_bf16_u, KvBf16, false)

// ---------------------------------------------------------------------------
// Attention over the pages: row i of request b's n rows is position p = len -
// n + i and sees its keys 0 .. p; head h reads KV head h / (nH / nKV):
//   s_t = scale q.k_t,  out = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m).
// A row without keys gives zeros.  One workgroup to a row and head, 256 keys
// a step with a running maximum and sum.
// ---------------------------------------------------------------------------
template <class KV>
__device__ __forceinline__ void attention_body(const float* __restrict__ q, uint32_t ld_q, uint32_t max_rows,
                                               const int32_t* __restrict__ row_start, const int32_t* __restrict__ lens,
                                               const int32_t* __restrict__ tables, uint32_t n_req, uint32_t max_pages,
                                               uint32_t nH, uint32_t nKV, uint32_t hd, float scale,
                                               const typename KV::T* __restrict__ kpages,
                                               const typename KV::T* __restrict__ vpages, uint32_t n_pages,
                                               uint32_t shift, float* __restrict__ out, uint32_t ld_out,
                                               uint64_t* __restrict__ err) {
  __shared__ float s_q[128], s_p[256], s_red[8], s_o[2][128];
  __shared__ uint32_t s_slot[256];
  const uint32_t r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t P = 1u << shift, kvh = h / (nH / nKV);
  uint32_t b = r, i = 0, n = 1;
  if (row_start) {
    const int32_t total = row_start[n_req];
    if (total < 0 || (uint32_t)total > max_rows) {
      if (r == 0 && h == 0 && tid == 0) paged_err(err, PAGED_ERR_ATT_ROWS, (uint32_t)total);
      return;
    }
    if (r >= (uint32_t)total) return;
    uint32_t lo = 0, hi = n_req;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) >> 1;
      if ((uint32_t)row_start[mid] <= r) lo = mid;
      else hi = mid;
    }
    b = lo;
    const int32_t r0 = row_start[b], r1 = row_start[b + 1];
    if (r0 < 0 || (uint32_t)r0 > r || (uint32_t)r1 <= r || r1 > total) {  // starts that do not ascend
      if (h == 0 && tid == 0) paged_err(err, PAGED_ERR_ATT_LENGTH, b);
      return;
    }
    i = r - (uint32_t)r0;
    n = (uint32_t)(r1 - r0);
  }
  const int32_t len = lens[b];
  if (len < 0 || (row_start && (uint32_t)len < n) || (uint64_t)len > ((uint64_t)max_pages << shift)) {
    if (i == 0 && h == 0 && tid == 0) paged_err(err, PAGED_ERR_ATT_LENGTH, b);
    return;
  }
  const uint32_t keys = row_start ? (uint32_t)len - n + i + 1 : (uint32_t)len;
  if (tid < hd) s_q[tid] = q[(size_t)r * ld_q + h * hd + tid] * scale;
  float m = -__builtin_inff(), l = 0.f, o = 0.f;
  const uint32_t d = tid & 127, part = tid >> 7;
  __syncthreads();
  for (uint32_t t0 = 0; t0 < keys; t0 += 256) {
    const uint32_t t = t0 + tid, nt = keys - t0 < 256 ? keys - t0 : 256;
    float s = -__builtin_inff();
    if (t < keys) {
      uint32_t page = (uint32_t)tables[(size_t)b * max_pages + (t >> shift)];
      if (page >= n_pages) {
        paged_err(err, PAGED_ERR_ATT_PAGE, b);
        page = 0;
      }
      s_slot[tid] = (page << shift) + (t & (P - 1));
      const typename KV::T* k = kpages + (((size_t)page * nKV + kvh) * P + (t & (P - 1))) * hd;
      s = 0.f;
      for (uint32_t e = 0; e < hd; e++) s = __builtin_fmaf(s_q[e], KV::up(k[e]), s);
    }
    float x = s;
    for (int k = 32; k >= 1; k >>= 1) {
      const float y = __shfl_xor(x, k);
      x = y > x ? y : x;
    }
    if (lane == 0) s_red[wave] = x;
    __syncthreads();
    float mn = m;
    for (int w = 0; w < 4; w++) mn = s_red[w] > mn ? s_red[w] : mn;
    const float base = mn == -__builtin_inff() ? 0.f : mn;
    const float alpha = __expf(m - base), p = t < keys ? __expf(s - base) : 0.f;
    s_p[tid] = p;
    float y = p;
    for (int k = 32; k >= 1; k >>= 1) y += __shfl_xor(y, k);
    if (lane == 0) s_red[4 + wave] = y;
    __syncthreads();
    l = l * alpha + (s_red[4] + s_red[5] + s_red[6] + s_red[7]);
    o *= alpha;
    m = mn;
    if (d < hd)
      for (uint32_t k = part; k < nt; k += 2) {
        const uint32_t sl = s_slot[k];
        const size_t a = (((size_t)(sl >> shift) * nKV + kvh) * P + (sl & (P - 1))) * hd + d;
        o = __builtin_fmaf(s_p[k], KV::up(vpages[a]), o);
      }
    __syncthreads();
  }
  s_o[part][d] = o;
  __syncthreads();
  if (tid < hd) out[(size_t)r * ld_out + h * hd + tid] = keys ? (s_o[0][tid] + s_o[1][tid]) / l : 0.f;
}

#define DEF_ATTENTION(NAME, KV)                                                                                     \
  extern "C" __global__ __launch_bounds__(256) void NAME(                                                          \
      const float* __restrict__ q, uint32_t ld_q, uint32_t max_rows, const int32_t* __restrict__ row_start,         \
      const int32_t* __restrict__ lens, const int32_t* __restrict__ tables, uint32_t n_req, uint32_t max_pages,     \
      uint32_t nH, uint32_t nKV, uint32_t hd, float scale, const KV::T* __restrict__ kpages,                        \
      const KV::T* __restrict__ vpages, uint32_t n_pages, uint32_t shift, float* __restrict__ out, uint32_t ld_out, \
      uint64_t* __restrict__ err) {                                                                                \
    attention_body<KV>(q, ld_q, max_rows, row_start, lens, tables, n_req, max_pages, nH, nKV, hd, scale, kpages,    \
                       vpages, n_pages, shift, out, ld_out, err);                                                   \
  }
DEF_ATTENTION(smith_paged_attention_f32, KvF32)
DEF_ATTENTION(smith_paged_attention_f16, KvF16)
DEF_ATTENTION(smith_paged_attention_bf16, KvBf16)
