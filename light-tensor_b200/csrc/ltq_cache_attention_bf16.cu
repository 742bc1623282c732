// Cache attention for bf16 queries, see ltq_cache_attention.cuh.
#include "../../include/ltq.h"
#define LTQ_ATTN_DT LTQ_BF16
#define LTQ_ATTN_LAUNCH launch_attention_bf16
#define LTQ_ATTN_JOIN launch_attention_join_bf16
#include "ltq_cache_attention.cuh"
