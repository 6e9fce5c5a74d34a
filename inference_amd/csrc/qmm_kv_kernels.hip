// The third gfx950 code object: the cache in pages and the operators over it, and the
// beam search's selection.
#include "qmm_kv_common.h"
#include "qmm_kv_page_kernels.h"
#include "qmm_kv_attn_kernels.h"
#include "qmm_beam_kernels.h"
