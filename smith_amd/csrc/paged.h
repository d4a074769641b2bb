// paged.h -- what the paged cache's and smith_logprobs' kernels and the bridge share: limits,
// arguments and the codes of what a kernel finds wrong in device memory.
#pragma once
#include <stdint.h>

// the kernels keep prefix sums over the requests of a step in LDS
#define PAGED_MAX_REQ 4096u

// attention: most splits of a block (their weights are kept in LDS, 16 columns of them)
#define PAGED_SPLIT_MAX 128u

// items wanted of a call, two workgroups to a CU, and partials at most: a block that is
// cut has more than 5/4 C keys and so less than twice its keys / C splits, 2 W / C <= 2
// target of them in all (and some for what f32 rounds)
#define PAGED_TARGET 512u
#define PAGED_MAX_PARTS (2u * PAGED_TARGET + 16u)

// attention
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
// a request's group: its shared keys (-1: it does not fit), its first partial, splits of
// its blocks, first row, rows, blocks
struct SharedOf {
  int32_t keys;
  uint32_t part, splits, row0, rows, blocks;
};
// and of the kernels whose rows do not see all keys, or not all at once
struct ReachArgs : AttArgs {
  uint32_t window, sinks;       // WINDOW
  uint32_t most_keys;           // WINDOW: no block visits more
  uint32_t n_groups;            // SHARED (n_req are the groups there)
  uint32_t n_all;               // SHARED: requests
  const int32_t* group_start;
  const int32_t* shared;
  SharedOf* from;               // [requests], written by SHARED, read by OWN
  float* prior;                 // [max_rows][heads][head dim] O of shared keys that are not cut
  float* prior_ml;              // [max_rows][heads][2] and m, l
  // OWN: SHARED's parts, columns of each, rows_blk, heads_blk and groups
  const float* s_parts;
  uint32_t s_columns, s_rows_blk, s_heads_blk, s_groups;
  uint32_t whole;  // OWN: all of a request's keys are its own
};

// fork and compact: pools whose addresses go to a kernel at once, and in all
#define PAGES_POOLS_LAUNCH 440u
#define PAGES_MAX_POOLS 4096u
#define PAGES_THREADS 256u
// a fork in one workgroup: most requests and pages
#define PAGES_SMALL_REQ 1024u
#define PAGES_SMALL_PAGES 65536u

// a request's table as the calls see it
struct PagesTables {
  const int32_t* lens;
  const int32_t* tables;
  const int32_t* parents;  // null: every request is its own
  uint32_t n_req, max_pages, n_pages, shift, window, sinks;
};
// what the kernels of a call hand on: device memory of the context
struct PagesWork {
  uint32_t* map;     // [words] a bit to a page; zero between calls
  uint32_t* state;   // [0] something was wrong (zero between calls), [1] the moves
  uint32_t* counts;  // [words / 256] live pages of 256 words' pages; null: not counted
  uint32_t* src;     // [moves] pages, from and to
  uint32_t* dst;
  uint32_t* keys;    // [moves] keys of each; null: whole pages
  uint32_t* rank;    // [n_pages] compact: the move of a page
  uint32_t words;
};
struct PagesPools {
  uint8_t* p[PAGES_POOLS_LAUNCH];
};

// log probabilities: threads of a workgroup, elements that a wave takes at once, most splits
// of a row (a lane each where they are joined) and top alternatives (a lane each)
#define SCORE_THREADS 256u
#define SCORE_WAVE_CHUNK 1024u
#define SCORE_MAX_SPLITS 64u
#define SCORE_MAX_TOP 64u
struct ScoreArgs {
  const void* logits;
  const int32_t* tokens;
  float* logprobs;
  float* entropy;
  int32_t* top_ids;
  float* top_logprobs;
  uint64_t* parts;     // [rows][splits][2 + top]
  uint32_t* counters;  // splits of a row that are done; zero between calls
  uint64_t* err;
  uint32_t ld, vocab, given, top, splits, per_split, row0;
};

#define PAGED_ROPE_ROW 1u   // SMITH_ROPE_ROW
#define PAGED_ROPE_HEAD 2u  // SMITH_ROPE_HEAD

enum {
  PAGED_ERR_PLAN_LENGTH = 1,  // argument: the request
  PAGED_ERR_PLAN_ROWS,        // the rows there is room for
  PAGED_ERR_PLAN_PAGES,       // the free pages
  PAGED_ERR_PLAN_PAGE,        // the request
  PAGED_ERR_APPEND_SLOT,      // the row
  PAGED_ERR_APPEND_POS,       // the row
  PAGED_ERR_ATT_ROWS,         // row_start's total
  PAGED_ERR_ATT_LENGTH,       // the request
  PAGED_ERR_ATT_PAGE,         // the request
  PAGED_ERR_FORK_PARENT,      // the request
  PAGED_ERR_FORK_LENGTH,      // the request
  PAGED_ERR_FORK_PAGE,        // the request
  PAGED_ERR_FORK_FREE,        // the free pages
  PAGED_ERR_SCORE_TOKEN,      // the row
  PAGED_ERR_ATT_GROUP,        // the group
  PAGED_ERR_ATT_SHARED,       // the request
};
