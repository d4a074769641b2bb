// paged_own_kernels.hip -- gfx950 kernels of smith_paged_attention_shared
// (smith_paged_own.hsaco): each request's own keys, joined with the shared ones:
//   out = sum w O / sum w l,  w = 2^(m - max m), over the own keys and the splits of
// the shared ones.  The splits of a column go to the waves in turn, 16 lanes to a
// column so that a load is 512 bytes in a row: 64 requests, 26 splits, 22 us, and 31
// in the layout of the sums.
//
// Bound by memory: 192 requests of up to 500 own bf16 keys behind shared ones (208 MB)
// 65 us; 64 of up to 300 f16 keys 15 us.  Of few keys in all (`whole`) it is the whole
// call, and reads shared keys as each request's own.
#include "paged_attention.h"

DEF_PART_ATTENTIONS(_own, OWN)
