// paged_shared_kernels.hip -- gfx950 kernels of smith_paged_attention_shared
// (smith_paged_shared.hsaco): the keys that the requests of a group have in
// common, once for all their columns.
#include "paged_attention.h"

DEF_PART_ATTENTIONS(_shared, SHARED)
