// The 8-bit key/value cache (ltq_kv_cache): what its append and attention kernels share.
#pragma once
#include "ltq_common.cuh"
#include "ltq_tokens.cuh"

namespace ltq {

// A batch of sequences as the kernels see it.
struct CacheBatch {
    const int32_t *offsets, *lengths, *table;
    uint64_t tokens;        // rows of the row arrays
    uint32_t seqs, table_width, max_new;
    int log2_bt;            // log2 of block_tokens
    uint32_t *status;
};

struct CacheSeq {
    int32_t off, n, len;    // first row, tokens of this call, tokens in all
    bool ok;
};
// Reads and checks sequence b; every CTA that meets a bad one reports it.
__device__ __forceinline__ CacheSeq cache_seq(const CacheBatch &bt, uint32_t b)
{
    CacheSeq s;
    const int32_t a = bt.offsets[b], e = bt.offsets[b + 1];
    s.len = bt.lengths[b];
    s.off = a;
    s.n = e - a;
    s.ok = a >= 0 && e >= a && (uint64_t)e <= bt.tokens && (uint32_t)s.n <= bt.max_new && s.len >= 0 &&
           (uint64_t)s.len <= ((uint64_t)bt.table_width << bt.log2_bt);
    if (!s.ok && threadIdx.x == 0) atomicCAS(bt.status, 0u, STATUS_BAD_SEQUENCE);
    return s;
}

cudaError_t launch_cache_append(const ltq_kv_cache &c, const CacheBatch &bt, const void *k, const void *v, int dtype, uint64_t ld,
                                cudaStream_t stream);

struct AttnArgs {
    ltq_kv_cache cache;
    CacheBatch bt;
    const void *q;
    void *out;
    uint64_t ld_q;
    uint32_t q_heads, group;       // group = q_heads / kv_heads
    float scale_log2;              // softmax scale * log2(e)
    uint32_t splits;               // CTAs that share one sequence's keys
    float *part_o;                 // [splits][tokens][q_heads][head_dim]
    float2 *part_ml;               // [splits][tokens][q_heads]: running maximum (base 2), sum
};
// Rows of (token, head of the group) that one CTA of the attention kernel takes.
uint32_t attn_rows_per_tile(int dtype, uint32_t head_dim, uint64_t rows);
cudaError_t launch_attention_f32(const AttnArgs &a, cudaStream_t stream);
cudaError_t launch_attention_f16(const AttnArgs &a, cudaStream_t stream);
cudaError_t launch_attention_bf16(const AttnArgs &a, cudaStream_t stream);

}  // namespace ltq
