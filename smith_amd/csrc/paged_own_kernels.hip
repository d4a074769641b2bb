// paged_own_kernels.hip -- gfx950 kernels of smith_paged_attention_shared
// (smith_paged_own.hsaco): each request's own keys, joined with the shared ones.
#include "paged_attention.h"

DEF_PART_ATTENTIONS(_own, OWN)
