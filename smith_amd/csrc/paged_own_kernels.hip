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
//
// The kernels of many rows and 128 dims keep 33 registers (f32) or 13 (f16, bf16) in
// scratch where they add four splits at once, behind the loop over the keys: 4 requests
// of 813 rows in all 29 us (f16), 30 (bf16), 55 (f32), beside 240, 298 and 1145 for
// the 8000 shared keys before them.
#include "paged_attention.h"

DEF_PART_ATTENTIONS(_own, OWN)
