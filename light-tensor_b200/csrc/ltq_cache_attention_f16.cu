// Cache attention for f16 queries, see ltq_cache_attention.cuh.
#include "../../include/ltq.h"
#define LTQ_ATTN_DT LTQ_F16
#define LTQ_ATTN_LAUNCH launch_attention_f16
#define LTQ_ATTN_JOIN launch_attention_join_f16
#include "ltq_cache_attention.cuh"
