// paged.h -- what the paged cache's kernels and the bridge share: limits and
// the codes of what a kernel finds wrong in device memory.
#pragma once

// the kernels keep prefix sums over the requests of a step in LDS
#define PAGED_MAX_REQ 4096u

// attention: most splits of a block (their weights are kept in LDS, 16 columns of them)
#define PAGED_SPLIT_MAX 128u

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
};
