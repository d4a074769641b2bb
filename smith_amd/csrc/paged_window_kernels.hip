// paged_window_kernels.hip -- gfx950 kernels of smith_paged_attention_window
// (smith_paged_window.hsaco): rows see the first keys and a window of the last.
#include "paged_attention.h"

DEF_PART_ATTENTIONS(_window, WINDOW)
