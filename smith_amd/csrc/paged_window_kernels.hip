// paged_window_kernels.hip -- gfx950 kernels of smith_paged_attention_window
// (smith_paged_window.hsaco): the row at position p sees keys t <= p with t > p - W
// or t < S.
//
// The keys that a block of rows visits are numbered without the gap between the sinks
// and its first row's window, in whole tiles, so that the key loops of
// paged_attention.h run over them as they are; only tiles at the edges are masked.
// A page of which no row sees a key is not looked up (it may be gone).
//
// Bound by memory for one row a request: 64 requests of up to 30000 keys, W 4096, S 4,
// 32 heads on 8 of 128, bf16 (199 MB) 47 us, 4.2 TB/s; 3 of a window of 512 f32 keys 8.5
// us, latency.  By the matrix cores for many: 1500 rows, W 2048, S 64, f16 127 us, 820
// TFLOP/s of split products, for MFMAs 33 % busy (a wave waits for its chain of products,
// exponentials and LDS reads, and 752 blocks are one or two rounds of 512 workgroups).
#include "paged_attention.h"

DEF_PART_ATTENTIONS(_window, WINDOW)
