// paged_shared_kernels.hip -- gfx950 kernels of smith_paged_attention_shared
// (smith_paged_shared.hsaco): the keys that the requests of a group have in
// common, once for all their columns.
//
// The (row, head) pairs of all the group's rows are the columns of one product, none
// masked; each split of the keys leaves (O, m, l) of its columns, which
// paged_own_kernels.hip's launch joins: spread over all of its workgroups, where a
// block's last split would read them alone (64 requests behind 6001 f16 keys, 32 heads
// on 8 of 128: 58 us with that join, 28 without).
//
// Bound by the matrix cores: 12 groups of 16 requests of 1 to 4 rows behind 2400 to
// 9000 bf16 keys 175 us, the products in three parts 35 % of it (items of unequal
// length leave a third of the waves' time idle); 64 rows behind 6001 f16 keys 23 us.
#include "paged_attention.h"

DEF_PART_ATTENTIONS(_shared, SHARED)
