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
    uint32_t *status;       // word for expired waits
    uint32_t *refused;      // word for what contradicts the bounds
};

struct CacheSeq {
    int32_t off, n, len;    // first row, tokens of this call, tokens in all
    bool ok;
};
// Reads and checks sequence b.
__device__ __forceinline__ CacheSeq cache_seq(const CacheBatch &bt, uint32_t b)
{
    CacheSeq s;
    const int32_t a = bt.offsets[b], e = bt.offsets[b + 1];
    s.len = bt.lengths[b];
    s.off = a;
    s.n = e - a;
    s.ok = a >= 0 && e >= a && (uint64_t)e <= bt.tokens && (uint32_t)s.n <= bt.max_new && s.len >= 0 &&
           (uint64_t)s.len <= ((uint64_t)bt.table_width << bt.log2_bt);
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
    bool q_vec, out_vec;           // rows start aligned to four elements
    bool q_vec8, out_vec8;         // to 16 bytes
    // Workspace: what warps leave of (row tile, head) items that they share with other warps, see ltq_cache_attention.cuh.
    float *part_o;                 // [2 * warps][rows per tile][head_dim]
    float2 *part_ml;               // [2 * warps][rows per tile]: running maximum (base 2), sum
    int2 *item;                    // [seqs][row tiles][kv_heads]: first slot, last warp
    uint32_t ctas, row_tiles;      // (tensor-core form: the SMs, groups of row tiles)
    uint32_t splits;               // tensor-core form: CTAs that share one's keys
    uint32_t cluster;              // CTAs per item in the form without workspace; 0: the form with
    uint32_t few_rows;             // up to so many rows are joined by a CTA each: eight for every SM
};
constexpr uint32_t ATTN_WARPS = 4;             // per CTA
constexpr uint32_t ATTN_MIN_STEPS = 4;         // fewer 16-key steps than this are not worth a warp of their own
constexpr uint32_t ATTN_CLUSTER_STEPS = 16;    // up to this many per warp one launch without workspace is faster
// Rows of (token, head of the group) that one CTA of the attention kernel takes.
uint32_t attn_rows_per_tile(int dtype, uint32_t head_dim, uint64_t rows);
// CTAs of it that fit an SM at once.
uint32_t attn_ctas_per_sm(int dtype, uint32_t head_dim, uint32_t rows_per_tile);
cudaError_t launch_attention_f32(const AttnArgs &a, cudaStream_t stream);
cudaError_t launch_attention_f16(const AttnArgs &a, cudaStream_t stream);
cudaError_t launch_attention_bf16(const AttnArgs &a, cudaStream_t stream);
// The tensor-core form for many new tokens (half and bfloat16 queries), ltq_cache_attention_tc.cu.
cudaError_t launch_attention_tc(const AttnArgs &a, int dtype, cudaStream_t stream);
uint32_t attn_tc_rows(uint32_t head_dim);      // rows per CTA
constexpr uint32_t ATTN_TC_MIN_TILES = 4;      // a split takes at least as many tiles of 64 keys
// Joins its parts.
cudaError_t launch_attention_join_f16(const AttnArgs &a, uint32_t rows_per_tile, cudaStream_t stream);
cudaError_t launch_attention_join_bf16(const AttnArgs &a, uint32_t rows_per_tile, cudaStream_t stream);

}  // namespace ltq
