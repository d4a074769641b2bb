// pages_kernels.hip -- gfx950 kernels that give the pages of a paged key-value
// cache to other requests (smith_pages.hsaco): requests become continuations of
// others, the pages that nobody names become the free list, and live pages move
// to the low end of the pools.
//
// A page is live if a request names it among the pages of its keys (of those
// that a window leaves it).  That is a bit in a map that the calls keep in the
// context, all zero between calls: mark sets the bits, the next kernel ranks the
// pages by them, and the last one, which no longer reads them, clears them.  So
// nothing about sharing is stored: there are no counts that could go wrong.
//
// Everything that indexes memory is checked where it is read; what fails is
// recorded for the next synchronising call, and the call then copies nothing.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged.h"
#include "paged_dev.h"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

typedef PagesTables Tables;
typedef PagesWork Work;

// keys j P .. (j + 1) P - 1: is one of them a sink, or seen by the row behind the
// last key (at position len, of a window of w: the keys above len - w)
__device__ __forceinline__ bool is_kept(const Tables& t, uint32_t j, uint32_t len) {
  return !t.window || ((uint64_t)j << t.shift) < t.sinks || (((uint64_t)j + 1) << t.shift) + t.window > (uint64_t)len + 1;
}
// the request that b goes on from, -1 for none
__device__ __forceinline__ int32_t parent_of(const Tables& t, uint32_t b) { return t.parents ? t.parents[b] : (int32_t)b; }
__device__ __forceinline__ bool fits(const Tables& t, int32_t len) {
  return len >= 0 && (uint64_t)(uint32_t)len <= ((uint64_t)t.max_pages << t.shift);
}
__device__ __forceinline__ uint32_t pages_of(const Tables& t, int32_t len) {
  return (uint32_t)(((uint64_t)(uint32_t)len + (1u << t.shift) - 1) >> t.shift);
}

// Bits of the pages that request blockIdx.x names after the call, and its table
// but for the pages that it still has to get.  Bound by latency: the length, the
// entries and the bits are each a round trip (300 requests of 20 to 30 pages 5.6 us).
extern "C" __global__ __launch_bounds__(PAGES_THREADS) void smith_pages_mark(Tables t, Work w,
                                                                           int32_t* __restrict__ new_tables,
                                                                           uint64_t* __restrict__ err) {
  const uint32_t b = blockIdx.x;
  const int32_t p = parent_of(t, b);
  if (p == -1) return;
  const bool lead = threadIdx.x == 0 && blockIdx.y == 0;
  if (p < -1 || (uint32_t)p >= t.n_req) {
    if (lead) {
      paged_err(err, PAGED_ERR_FORK_PARENT, b);
      w.state[0] = 1;
    }
    return;
  }
  const int32_t len = t.lens[p];
  if (!fits(t, len)) {
    if (lead) {
      paged_err(err, PAGED_ERR_FORK_LENGTH, (uint32_t)p);
      w.state[0] = 1;
    }
    return;
  }
  const uint32_t n = pages_of(t, len);
  const int32_t* from = t.tables + (size_t)p * t.max_pages;
  int32_t* to = new_tables ? new_tables + (size_t)b * t.max_pages : nullptr;
  for (uint32_t j = blockIdx.y * PAGES_THREADS + threadIdx.x; j < n; j += gridDim.y * PAGES_THREADS) {
    const bool kept = is_kept(t, j, (uint32_t)len);
    const int32_t page = kept ? from[j] : -1;
    if (kept) {
      if ((uint32_t)page >= t.n_pages) {
        paged_err(err, PAGED_ERR_FORK_PAGE, (uint32_t)p);
        w.state[0] = 1;
      } else {
        // siblings name the same pages: most bits are there already
        uint32_t* word = w.map + ((uint32_t)page >> 5);
        const uint32_t bit = 1u << (page & 31);
        if (!(__hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & bit)) atomicOr(word, bit);
      }
    }
    if (to) to[j] = page;
  }
}

// sum over the workgroup of one number a thread, and over the threads before this one
__device__ __forceinline__ uint32_t sum_before(uint32_t v, uint32_t* s_wave, uint32_t& total) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, upto = scan64_lanes(v);
  __syncthreads();
  if (lane == 63) s_wave[wave] = upto;
  __syncthreads();
  uint32_t before = upto - v;
  total = 0;
#pragma unroll
  for (uint32_t k = 0; k < PAGES_THREADS / 64; k++) {
    if (k < wave) before += s_wave[k];
    total += s_wave[k];
  }
  return before;
}

// Live pages of each 256 words, for pools so large that to count all words in every
// workgroup costs more than this launch.
extern "C" __global__ __launch_bounds__(PAGES_THREADS) void smith_pages_count(Work w) {
  __shared__ uint32_t s_wave[PAGES_THREADS / 64];
  const uint32_t k = blockIdx.x * PAGES_THREADS + threadIdx.x;
  uint32_t total;
  (void)sum_before(k < w.words ? (uint32_t)__popc(w.map[k]) : 0u, s_wave, total);
  if (threadIdx.x == 0) w.counts[blockIdx.x] = total;
}

// Live pages of all words, of those before `word0` (a multiple of 256) and of the
// pages below `line`.
struct Live {
  uint32_t all, before, below;
};
__device__ __forceinline__ Live count_live(const Work& w, uint32_t word0, uint32_t line, uint32_t* s_wave) {
  uint32_t all = 0, before = 0, below = 0;
  auto word = [&](uint32_t k, uint32_t x) {  // bits of word k below the line
    const uint32_t first = 32 * k;
    return first >= line ? 0u : (uint32_t)__popc(line - first >= 32 ? x : x & ((1u << (line - first)) - 1));
  };
  if (w.counts) {
    const uint32_t blocks = (w.words + PAGES_THREADS - 1) / PAGES_THREADS, at = line / (32 * PAGES_THREADS);
#pragma unroll 4
    for (uint32_t k = threadIdx.x; k < blocks; k += PAGES_THREADS) {
      const uint32_t n = w.counts[k];
      all += n;
      if (k < word0 / PAGES_THREADS) before += n;
      if (k < at) below += n;
    }
    const uint32_t k = at * PAGES_THREADS + threadIdx.x;  // the words about the line
    if (k < w.words) below += word(k, w.map[k]);
  } else {
#pragma unroll 4
    for (uint32_t k = threadIdx.x; k < w.words; k += PAGES_THREADS) {
      const uint32_t x = w.map[k], n = (uint32_t)__popc(x);
      all += n;
      if (k < word0) before += n;
      below += word(k, x);
    }
  }
  Live l;
  (void)sum_before(all, s_wave, l.all);
  (void)sum_before(before, s_wave, l.before);
  (void)sum_before(below, s_wave, l.below);
  return l;
}

// f(page, live, live pages before it) of the workgroup's 256 words' pages, a lane to a page
template <class F>
__device__ __forceinline__ void each_page(const Work& w, uint32_t n_pages, uint32_t word0, uint32_t before,
                                          uint32_t* s_wave, F f) {
  const uint32_t lane = threadIdx.x & 63, mine = word0 + threadIdx.x;
  const uint32_t x = mine < w.words ? w.map[mine] : 0u;
  uint32_t total;
  const uint32_t from = before + sum_before((uint32_t)__popc(x), s_wave, total);
  for (uint32_t i = 0; i < 32; i++) {
    const uint32_t k = 2 * i + (lane >> 5), bit = lane & 31;
    const uint32_t bits = (uint32_t)__shfl((int)x, (int)k), rank = (uint32_t)__shfl((int)from, (int)k);
    const uint32_t page = ((word0 + (threadIdx.x & ~63u) + k) << 5) + bit;
    if (page < n_pages) f(page, (bits >> bit) & 1, rank + (uint32_t)__popc(bits & ((1u << bit) - 1)));
  }
}

// New lengths, the free list and the copies of a fork.  The requests that go on
// from one parent share its full pages; the partly filled one stays with the
// first of them, and the others, in order, take the lowest free pages for copies
// of it.  The rest is the free list, highest first.  No exchange between
// workgroups: each counts all bits and ranks the copying requests by itself, then
// serves the pages of its 256 words.
extern "C" __global__ __launch_bounds__(PAGES_THREADS) void smith_pages_fork(Tables t, Work w,
                                                                           int32_t* __restrict__ new_lens,
                                                                           int32_t* __restrict__ new_tables,
                                                                           int32_t* __restrict__ free_pages,
                                                                           int32_t* __restrict__ free_count,
                                                                           uint64_t* __restrict__ err) {
  __shared__ uint32_t s_first[PAGED_MAX_REQ], s_who[PAGED_MAX_REQ], s_wave[PAGES_THREADS / 64];
  const uint32_t tid = threadIdx.x, P = 1u << t.shift;
  const bool lead = blockIdx.x == 0 && tid == 0;
  if (w.state[0]) {  // a request that does not fit: no copies, no free list
    if (lead) {
      free_count[0] = 0;
      w.state[1] = 0;
    }
    return;
  }
  for (uint32_t b = tid; b < t.n_req; b += PAGES_THREADS) s_first[b] = ~0u;
  __syncthreads();
  for (uint32_t b = tid; b < t.n_req; b += PAGES_THREADS) {
    const int32_t p = parent_of(t, b);
    if (p >= 0) atomicMin(&s_first[p], b);
    if (blockIdx.x == 0) new_lens[b] = p >= 0 ? t.lens[p] : 0;
  }
  __syncthreads();
  const uint32_t per = (t.n_req + PAGES_THREADS - 1) / PAGES_THREADS;
  auto copies = [&](uint32_t b) {
    const int32_t p = parent_of(t, b);
    return p >= 0 && s_first[p] != b && (t.lens[p] & (int32_t)(P - 1));
  };
  uint32_t n = 0, need;
  for (uint32_t k = 0; k < per; k++)
    if (tid * per + k < t.n_req) n += copies(tid * per + k);
  uint32_t at = sum_before(n, s_wave, need);
  for (uint32_t k = 0; k < per; k++)
    if (tid * per + k < t.n_req && copies(tid * per + k)) s_who[at++] = tid * per + k;
  const uint32_t word0 = blockIdx.x * PAGES_THREADS;
  const Live live = count_live(w, word0, 0, s_wave);
  const uint32_t frees = t.n_pages - live.all;
  if (need > frees) {  // the same in every workgroup
    if (lead) {
      paged_err(err, PAGED_ERR_FORK_FREE, frees);
      free_count[0] = 0;
      w.state[1] = 0;
    }
    return;
  }
  if (lead) {
    free_count[0] = (int32_t)(frees - need);
    w.state[1] = need;
  }
  __syncthreads();  // s_who
  each_page(w, t.n_pages, word0, live.before, s_wave, [&](uint32_t page, uint32_t is_live, uint32_t lives) {
    if (is_live) return;
    const uint32_t rank = page - lives;  // free pages before it
    if (rank >= need) {
      free_pages[frees - 1 - rank] = (int32_t)page;
      return;
    }
    const uint32_t b = s_who[rank];
    const int32_t p = parent_of(t, b), len = t.lens[p];
    const uint32_t j = (uint32_t)len >> t.shift;
    w.src[rank] = (uint32_t)t.tables[(size_t)p * t.max_pages + j];
    w.dst[rank] = page;
    w.keys[rank] = (uint32_t)len & (P - 1);
    new_tables[(size_t)b * t.max_pages + j] = (int32_t)page;
  });
}

// mark and fork in one launch of one workgroup, the map in LDS, for few requests and
// pages: what mark's workgroups spread over the card is then less than a launch takes.
// A thread to a request, then the entries of all tables one after another, a request
// found by bisection, then a lane to a page.  Bound by latency, parent, length, entry
// and what is made of them one after another: 8 requests on 700 keys 5.2 us, 160 of 1000
// 9.6 (7.6 and 5.3 as two launches over the card, and the time between them).
#define SMALL_THREADS 1024u
extern "C" __global__ __launch_bounds__(SMALL_THREADS) void smith_pages_fork_small(Tables t, Work w, int32_t* __restrict__ new_lens,
                                                                                  int32_t* __restrict__ new_tables,
                                                                                  int32_t* __restrict__ free_pages,
                                                                                  int32_t* __restrict__ free_count,
                                                                                  uint64_t* __restrict__ err) {
  constexpr uint32_t WAVES = SMALL_THREADS / 64, REQ = PAGES_SMALL_REQ, WORDS = PAGES_SMALL_PAGES / 32;
  static_assert(REQ == SMALL_THREADS && WORDS == 2 * SMALL_THREADS, "a thread to a request, and to two words");
  __shared__ uint32_t s_map[WORDS], s_before[WORDS], s_start[REQ + 1], s_first[REQ], s_who[REQ], s_wave[WAVES], s_bad;
  __shared__ int32_t s_parent[REQ], s_len[REQ];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, P = 1u << t.shift;
  // sum over the threads before this one, and over all
  auto scan = [&](uint32_t v, uint32_t& total) {
    const uint32_t upto = scan64_lanes(v);
    __syncthreads();
    if (lane == 63) s_wave[wave] = upto;
    __syncthreads();
    uint32_t before = upto - v;
    total = 0;
#pragma unroll
    for (uint32_t k = 0; k < WAVES; k++) {
      if (k < wave) before += s_wave[k];
      total += s_wave[k];
    }
    return before;
  };
  int32_t p = -1, len = 0;
  if (tid < t.n_req) p = t.parents[tid];
  s_map[tid] = s_map[tid + SMALL_THREADS] = 0;
  s_first[tid] = ~0u;
  if (tid == 0) s_bad = 0;
  __syncthreads();
  if (p != -1) {
    if (p < -1 || (uint32_t)p >= t.n_req) {
      paged_err(err, PAGED_ERR_FORK_PARENT, tid);
      s_bad = 1;
      p = -1;
    } else {
      len = t.lens[p];
      if (!fits(t, len)) {
        paged_err(err, PAGED_ERR_FORK_LENGTH, (uint32_t)p);
        s_bad = 1;
        len = 0;
      }
      atomicMin(&s_first[p], tid);
    }
  }
  s_parent[tid] = p;
  s_len[tid] = len;
  const uint32_t pages = pages_of(t, len);
  uint32_t entries;
  s_start[tid] = scan(pages, entries);
  if (tid == 0) s_start[REQ] = entries;
  __syncthreads();
  const bool copy = p >= 0 && s_first[p] != tid && (len & (int32_t)(P - 1));
  if (tid < t.n_req) new_lens[tid] = len;
  constexpr uint32_t BATCH = 4;
  for (uint32_t e0 = tid; e0 < entries; e0 += BATCH * SMALL_THREADS) {
    int32_t page[BATCH];
    uint32_t of[BATCH], j[BATCH];
    bool kept[BATCH];
#pragma unroll
    for (uint32_t k = 0; k < BATCH; k++) {
      const uint32_t e = e0 + k * SMALL_THREADS < entries ? e0 + k * SMALL_THREADS : entries - 1;
      // the last request that starts at or before e (those without pages start there too)
      uint32_t lo = 0;
#pragma unroll
      for (uint32_t step = REQ / 2; step; step >>= 1)
        if (s_start[lo + step] <= e) lo += step;
      of[k] = lo;
      j[k] = e - s_start[lo];
      kept[k] = is_kept(t, j[k], (uint32_t)s_len[lo]);
      page[k] = kept[k] ? t.tables[(size_t)s_parent[lo] * t.max_pages + j[k]] : -1;
    }
#pragma unroll
    for (uint32_t k = 0; k < BATCH; k++) {
      if (e0 + k * SMALL_THREADS >= entries) continue;
      if (kept[k]) {
        if ((uint32_t)page[k] >= t.n_pages) {
          paged_err(err, PAGED_ERR_FORK_PAGE, (uint32_t)s_parent[of[k]]);
          s_bad = 1;
          continue;
        }
        atomicOr(&s_map[(uint32_t)page[k] >> 5], 1u << (page[k] & 31));
      }
      // the last entry of a request that copies is written below
      const int32_t n = s_len[of[k]];
      if (s_first[s_parent[of[k]]] == of[k] || !(n & (int32_t)(P - 1)) || j[k] != (uint32_t)n >> t.shift)
        new_tables[(size_t)of[k] * t.max_pages + j[k]] = page[k];
    }
  }
  uint32_t need, lives;
  const uint32_t at = scan(copy, need);
  if (copy) s_who[at] = tid;
  const uint32_t x0 = s_map[2 * tid], x1 = s_map[2 * tid + 1];
  const uint32_t before = scan((uint32_t)(__popc(x0) + __popc(x1)), lives), frees = t.n_pages - lives;
  s_before[2 * tid] = before;
  s_before[2 * tid + 1] = before + (uint32_t)__popc(x0);
  __syncthreads();
  const bool bad = s_bad || need > frees;
  if (tid == 0) {
    if (!s_bad && bad) paged_err(err, PAGED_ERR_FORK_FREE, frees);
    free_count[0] = bad ? 0 : (int32_t)(frees - need);
    w.state[1] = bad ? 0 : need;
  }
  if (bad) return;
  for (uint32_t page = tid; page < t.n_pages; page += SMALL_THREADS) {
    const uint32_t bits = s_map[page >> 5], bit = page & 31;
    if (bits >> bit & 1) continue;
    const uint32_t rank = page - s_before[page >> 5] - (uint32_t)__popc(bits & ((1u << bit) - 1));  // free pages before it
    if (rank >= need) {
      free_pages[frees - 1 - rank] = (int32_t)page;
      continue;
    }
    const uint32_t b = s_who[rank], n = (uint32_t)s_len[b], j = n >> t.shift;
    w.src[rank] = (uint32_t)t.tables[(size_t)s_parent[b] * t.max_pages + j];
    w.dst[rank] = page;
    w.keys[rank] = n & (P - 1);
    new_tables[(size_t)b * t.max_pages + j] = (int32_t)page;
  }
}

// The moves of a compaction: of n live pages, those at n and above go to the free
// ones below n, lowest to lowest.  A page that is read is never written.
extern "C" __global__ __launch_bounds__(PAGES_THREADS) void smith_pages_line(Work w, uint32_t n_pages,
                                                                           int32_t* __restrict__ free_pages,
                                                                           int32_t* __restrict__ free_count) {
  __shared__ uint32_t s_wave[PAGES_THREADS / 64];
  const bool lead = blockIdx.x == 0 && threadIdx.x == 0;
  if (w.state[0]) {
    if (lead) {
      free_count[0] = 0;
      w.state[1] = 0;
    }
    return;
  }
  const uint32_t word0 = blockIdx.x * PAGES_THREADS;
  const uint32_t n = count_live(w, word0, 0, s_wave).all;
  const Live live = count_live(w, word0, n, s_wave);
  if (lead) {
    free_count[0] = (int32_t)(n_pages - n);
    w.state[1] = n - live.below;
  }
  each_page(w, n_pages, word0, live.before, s_wave, [&](uint32_t page, uint32_t is_live, uint32_t lives) {
    if (page < n && !is_live) w.dst[page - lives] = page;
    if (page >= n) {
      free_pages[n_pages - 1 - page] = (int32_t)page;
      if (is_live) {
        w.src[lives - live.below] = page;
        w.rank[page] = lives - live.below;
      }
    }
  });
}

// Tables of the pages where they are after smith_pages_line's moves.
extern "C" __global__ __launch_bounds__(PAGES_THREADS) void smith_pages_remap(Tables t, Work w,
                                                                            const int32_t* __restrict__ free_count,
                                                                            int32_t* new_tables) {
  if (w.state[0]) return;
  const uint32_t b = blockIdx.x, line = t.n_pages - (uint32_t)free_count[0];
  const int32_t len = t.lens[b];
  const uint32_t n = pages_of(t, len);
  for (uint32_t j = blockIdx.y * PAGES_THREADS + threadIdx.x; j < n; j += gridDim.y * PAGES_THREADS) {
    const size_t at = (size_t)b * t.max_pages + j;
    int32_t page = -1;
    if (is_kept(t, j, (uint32_t)len)) {
      page = t.tables[at];
      if ((uint32_t)page >= line) page = (int32_t)w.dst[w.rank[page]];
    }
    new_tables[at] = page;
  }
}

// The moves' keys in every pool, 16 KB to a workgroup at a time, and the map is
// cleared for the next call.  Of a page [n_kv][P][head dim] the first keys[m] of
// each head: contiguous runs.  Bound by memory: 784 MB read and written in 174 us, 4.5
// TB/s (a large copy: 5.2).
extern "C" __global__ __launch_bounds__(PAGES_THREADS) void smith_pages_move(PagesPools pools, Work w, uint32_t n_pools,
                                                                           uint32_t n_kv, uint32_t row16, uint32_t shift,
                                                                           uint32_t clear) {
  constexpr uint32_t UNROLL = 4, CHUNK = PAGES_THREADS * UNROLL;  // 16-byte units
  const uint32_t tid = threadIdx.x;
  const uint32_t moves = w.state[1];
  const uint32_t head = row16 << shift, page = n_kv * head, chunks = (page + CHUNK - 1) / CHUNK;
  const uint64_t items = (uint64_t)moves * n_pools * chunks;
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const uint32_t chunk = (uint32_t)(item % chunks);
    const uint64_t rest = item / chunks;
    const uint32_t pool = (uint32_t)(rest % n_pools), m = (uint32_t)(rest / n_pools);
    const uint32_t run = w.keys ? w.keys[m] * row16 : head, total = n_kv * run;
    if (chunk * CHUNK >= total) continue;
    const u32x4* from = (const u32x4*)pools.p[pool] + (size_t)w.src[m] * page;
    u32x4* to = (u32x4*)pools.p[pool] + (size_t)w.dst[m] * page;
    u32x4 x[UNROLL];
    uint32_t at[UNROLL];
#pragma unroll
    for (uint32_t k = 0; k < UNROLL; k++) {
      const uint32_t u = chunk * CHUNK + k * PAGES_THREADS + tid, v = u < total ? u : total - 1;
      at[k] = run == head ? v : v / run * head + v % run;
      x[k] = from[at[k]];
    }
#pragma unroll
    for (uint32_t k = 0; k < UNROLL; k++)
      if (chunk * CHUNK + k * PAGES_THREADS + tid < total) to[at[k]] = x[k];
  }
  if (!clear) return;
  if (blockIdx.x == 0 && tid == 0) w.state[0] = 0;
  for (uint32_t k = blockIdx.x * PAGES_THREADS + tid; k < w.words; k += gridDim.x * PAGES_THREADS) w.map[k] = 0;
}
