// Cache attention for f32 queries, see ltq_cache_attention.cuh.
#include "../../include/ltq.h"
#define LTQ_ATTN_DT LTQ_F32
#define LTQ_ATTN_LAUNCH launch_attention_f32
#include "ltq_cache_attention.cuh"
