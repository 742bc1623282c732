// The 8-bit key/value cache: entry points (include/ltq.h) and the kernel that appends to it.  The attention kernels are in
// ltq_cache_attention.cuh.
#include "ltq_cache.cuh"
#include "ltq_ptx.cuh"
#include "ltq_quant.cuh"

namespace ltq {

namespace {

constexpr int APPEND_THREADS = 128, APPEND_KEEP = 8;
constexpr float SMALLEST_SCALE = 1.17549435e-38f;   // 2^-126

// A 16-byte vector of 8 (float: 4) neighbouring elements, element by element where it is not aligned.
template <int DT>
struct Vec {
    static constexpr int N = DT == LTQ_F32 ? 4 : 8;
    uint32_t w[4];
    __device__ __forceinline__ void load(const void *base, uint64_t at, bool vec)
    {
        if (DT == LTQ_F32) {
            const uint32_t *p = static_cast<const uint32_t *>(base) + at;
            if (vec) *reinterpret_cast<uint4 *>(w) = __ldg(reinterpret_cast<const uint4 *>(p));
            else
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = p[i];
        } else {
            const uint16_t *p = static_cast<const uint16_t *>(base) + at;
            if (vec) *reinterpret_cast<uint4 *>(w) = __ldg(reinterpret_cast<const uint4 *>(p));
            else
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ float4 four(int h) const   // elements 4 h .. 4 h + 3
    {
        if (DT == LTQ_F32) return make_float4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3]));
        const uint32_t a = w[2 * h % 4], b = w[(2 * h + 1) % 4];
        if (DT == LTQ_F16) {
            const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&a)), y = __half22float2(*reinterpret_cast<const __half2 *>(&b));
            return make_float4(x.x, x.y, y.x, y.y);
        }
        return make_float4(__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u), __uint_as_float(b << 16), __uint_as_float(b & 0xFFFF0000u));
    }
};
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

}  // namespace

// One CTA per (block that a sequence touches, head, K or V): the largest magnitude of the block's new tokens fixes its scale,
// older codes of the block follow if the scale grew, the new codes are written.  The first APPEND_KEEP vectors of every thread (64
// tokens of 128 halves) stay in registers in between, all loads on their way at once; what goes beyond is read again, out of L2.
// Bound by HBM at large sizes (element + 1 bytes per value), by launch latency for one token per sequence.
// Grid: (2 * blocks per sequence, kv_heads, sequences).
template <int DT>
__global__ void __launch_bounds__(APPEND_THREADS)
cache_append_kernel(const ltq_kv_cache cache, const CacheBatch bt, const void *__restrict__ k, const void *__restrict__ v, uint64_t ld, bool vec)
{
    griddep_launch_dependents();
    griddep_wait();
    const CacheSeq s = cache_seq(bt, blockIdx.z);
    if (!s.ok && threadIdx.x == 0) atomicCAS(bt.refused, 0u, REFUSED_SEQUENCE);
    if (!s.ok || s.n == 0) return;
    const bool is_v = blockIdx.x & 1;
    const int bt_tokens = 1 << bt.log2_bt, start = s.len - s.n < 0 ? 0 : s.len - s.n;   // first position that is stored
    const int64_t blk = (int64_t)(start >> bt.log2_bt) + (blockIdx.x >> 1);
    const int64_t first = blk << bt.log2_bt;                                              // the block's first position
    if (first >= s.len) return;
    const int used = first >= start ? 0 : (int)(start - first);                           // tokens it holds already
    const int end = s.len - first < bt_tokens ? (int)(s.len - first) : bt_tokens;
    const int32_t page = bt.table[(uint64_t)blockIdx.z * bt.table_width + blk];
    if ((uint32_t)page >= cache.blocks) {
        if (threadIdx.x == 0) atomicCAS(bt.refused, 0u, REFUSED_BLOCK);
        return;
    }
    constexpr int VN = Vec<DT>::N;
    const uint32_t D = cache.head_dim, h = blockIdx.y, per = D / VN;
    const uint64_t slot = (uint64_t)(uint32_t)page * cache.kv_heads + h;
    uint32_t *codes = reinterpret_cast<uint32_t *>((is_v ? cache.v_dev : cache.k_dev) + (slot << bt.log2_bt) * D);
    ltq_qparams *qp = (is_v ? cache.v_qp_dev : cache.k_qp_dev) + slot;
    const void *src = is_v ? v : k;
    // row of the block's token i: the sequence's row of position p is off + p - (len - n)
    const uint64_t row0 = (uint64_t)((int64_t)s.off + first - (s.len - s.n));
    const uint32_t chunks = (uint32_t)(end - used) * per;
    auto load = [&](Vec<DT> &x, uint32_t i) {
        const uint32_t t = i / per;
        x.load(src, (row0 + used + t) * ld + (uint64_t)h * D + (i - t * per) * VN, vec);
    };

    float most = 0.f;
    auto look = [&](const Vec<DT> &x) {
#pragma unroll
        for (int k = 0; k < VN / 4; k++) {
            const float4 v = x.four(k);
            most = max_nan(max_nan(most, max_nan(fabsf(v.x), fabsf(v.y))), max_nan(fabsf(v.z), fabsf(v.w)));
        }
    };
    Vec<DT> keep[APPEND_KEEP];
#pragma unroll
    for (int j = 0; j < APPEND_KEEP; j++)
        if (threadIdx.x + j * APPEND_THREADS < chunks) load(keep[j], threadIdx.x + j * APPEND_THREADS);
#pragma unroll
    for (int j = 0; j < APPEND_KEEP; j++)
        if (threadIdx.x + j * APPEND_THREADS < chunks) look(keep[j]);
    for (uint32_t i = threadIdx.x + APPEND_KEEP * APPEND_THREADS; i < chunks; i += APPEND_THREADS) {
        Vec<DT> x;
        load(x, i);
        look(x);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
    __shared__ float s_most[APPEND_THREADS / 32];
    if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = most;
    const float old = used ? qp->scale : 0.f;
    __syncthreads();   // (also: everyone has read the old scale)
#pragma unroll
    for (int w = 0; w < APPEND_THREADS / 32; w++) most = max_nan(most, s_most[w]);
    float scale = max_nan(fmaxf(__fdiv_rn(most, 127.f), SMALLEST_SCALE), old);
    const bool finite = most < INFINITY && scale < INFINITY;   // false for NaN, a NaN that the block had before included
    if (threadIdx.x == 0) {
        const float stored = finite ? scale : __int_as_float(0x7FC00000);
        *reinterpret_cast<uint2 *>(qp) = make_uint2(__float_as_uint(stored), 128u);
    }
    const float inv = quant_row_inv(scale);
    if (finite && used && scale > old) {
        for (uint32_t i = threadIdx.x; i < (uint32_t)used * (D / 4); i += APPEND_THREADS) {
            const uint32_t w = codes[i];
            const float4 x = make_float4(__fmul_rn(old, (float)((int)(w & 0xFF) - 128)), __fmul_rn(old, (float)((int)((w >> 8) & 0xFF) - 128)),
                                         __fmul_rn(old, (float)((int)((w >> 16) & 0xFF) - 128)), __fmul_rn(old, (float)((int)(w >> 24) - 128)));
            codes[i] = quant4_row(x, scale, 128.f, inv);
        }
    }
    auto put = [&](const Vec<DT> &x, uint32_t i) {
        uint32_t w[VN / 4];
#pragma unroll
        for (int k = 0; k < VN / 4; k++) w[k] = finite ? quant4_row(x.four(k), scale, 128.f, inv) : 0x80808080u;
        uint32_t *at = codes + ((uint32_t)used * per + i) * (VN / 4);
        if (VN == 8) *reinterpret_cast<uint2 *>(at) = make_uint2(w[0], w[VN / 4 - 1]);
        else at[0] = w[0];
    };
#pragma unroll
    for (int j = 0; j < APPEND_KEEP; j++)
        if (threadIdx.x + j * APPEND_THREADS < chunks) put(keep[j], threadIdx.x + j * APPEND_THREADS);
    for (uint32_t i = threadIdx.x + APPEND_KEEP * APPEND_THREADS; i < chunks; i += APPEND_THREADS) {
        Vec<DT> x;
        load(x, i);
        put(x, i);
    }
}

cudaError_t launch_cache_append(const ltq_kv_cache &c, const CacheBatch &bt, const void *k, const void *v, int dtype, uint64_t ld,
                                cudaStream_t stream)
{
    // n tokens from any offset touch at most (n + block_tokens - 2) / block_tokens + 1 blocks
    const uint32_t bt_tokens = 1u << bt.log2_bt, blocks = (bt.max_new + bt_tokens - 2) / bt_tokens + 1;
    const dim3 grid(2 * blocks, c.kv_heads, bt.seqs);
    const bool vec = (ld * dtype_size(dtype)) % 16 == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
    count_launch();
    if (dtype == LTQ_F32) return launch_chained(cache_append_kernel<LTQ_F32>, grid, dim3(APPEND_THREADS), 0, stream, c, bt, k, v, ld, vec);
    if (dtype == LTQ_F16) return launch_chained(cache_append_kernel<LTQ_F16>, grid, dim3(APPEND_THREADS), 0, stream, c, bt, k, v, ld, vec);
    return launch_chained(cache_append_kernel<LTQ_BF16>, grid, dim3(APPEND_THREADS), 0, stream, c, bt, k, v, ld, vec);
}

uint32_t attn_rows_per_tile(int dtype, uint32_t head_dim, uint64_t rows)
{
    // sixteen rows share the conversion of the keys where the registers allow it
    return rows > 8 && head_dim * (dtype == LTQ_F32 ? 2 : 1) <= 128 ? 16 : 8;
}
uint32_t attn_ctas_per_sm(int dtype, uint32_t head_dim, uint32_t rows_per_tile)
{
    return head_dim * (rows_per_tile / 8) * (dtype == LTQ_F32 ? 2 : 1) <= 128 ? 3 : 2;
}

namespace {

int check_cache(const ltq_kv_cache *c)
{
    LTQ_REQUIRE(c && c->k_dev && c->v_dev && c->k_qp_dev && c->v_qp_dev, LTQ_ERR_INVALID_ARG, "Invalid argument");
    LTQ_REQUIRE(c->blocks >= 1 && c->blocks < (1ull << 31) && c->kv_heads >= 1 && c->kv_heads <= 65535, LTQ_ERR_INVALID_ARG,
                "a cache of %llu blocks with %u heads", (unsigned long long)c->blocks, c->kv_heads);
    LTQ_REQUIRE(c->block_tokens == 16 || c->block_tokens == 32 || c->block_tokens == 64 || c->block_tokens == 128, LTQ_ERR_UNSUPPORTED,
                "block_tokens must be 16, 32, 64 or 128, not %u", c->block_tokens);
    const uint32_t d = c->head_dim;
    LTQ_REQUIRE(d == 32 || d == 64 || d == 96 || d == 128 || d == 192 || d == 256, LTQ_ERR_UNSUPPORTED,
                "head_dim must be 32, 64, 96, 128, 192 or 256, not %u", d);
    LTQ_REQUIRE((((uintptr_t)c->k_dev | (uintptr_t)c->v_dev) & 15) == 0 && (((uintptr_t)c->k_qp_dev | (uintptr_t)c->v_qp_dev) & 7) == 0,
                LTQ_ERR_INVALID_ARG, "misaligned cache arrays");
    return LTQ_OK;
}

int check_batch(const ltq_kv_cache *c, const void *offsets, const void *lengths, const void *table, uint64_t tokens, uint64_t seqs,
                uint64_t table_width, uint64_t max_new)
{
    LTQ_REQUIRE(offsets && lengths && (table || table_width == 0), LTQ_ERR_INVALID_ARG, "Invalid argument");
    LTQ_REQUIRE((((uintptr_t)offsets | (uintptr_t)lengths | (uintptr_t)table) & 3) == 0, LTQ_ERR_INVALID_ARG, "misaligned array");
    LTQ_REQUIRE(seqs <= 65535, LTQ_ERR_TOO_LARGE, "%llu sequences: at most 65535", (unsigned long long)seqs);
    LTQ_REQUIRE(tokens < (1ull << 31) && max_new <= tokens && table_width <= 0x7FFFFFFFull / c->block_tokens, LTQ_ERR_INVALID_ARG,
                "%llu tokens, at most %llu per sequence, tables of %llu blocks", (unsigned long long)tokens, (unsigned long long)max_new,
                (unsigned long long)table_width);
    return LTQ_OK;
}

CacheBatch make_batch(const ltq_kv_cache *c, const int32_t *offsets, const int32_t *lengths, const int32_t *table, uint64_t tokens,
                      uint64_t seqs, uint64_t table_width, uint64_t max_new, uint32_t *status)
{
    CacheBatch bt;
    bt.offsets = offsets;
    bt.lengths = lengths;
    bt.table = table;
    bt.tokens = tokens;
    bt.seqs = (uint32_t)seqs;
    bt.table_width = (uint32_t)table_width;
    bt.max_new = (uint32_t)max_new;
    bt.log2_bt = c->block_tokens == 16 ? 4 : (c->block_tokens == 32 ? 5 : (c->block_tokens == 64 ? 6 : 7));
    bt.status = status;
    bt.refused = status + 1;
    return bt;
}

// How the attention call is laid out: CTAs, row tiles per sequence, and the workspace behind them.
struct AttnPlan {
    uint32_t rows_per_tile, row_tiles, ctas, cluster, splits;
    bool tc;
    uint64_t o_floats, ml, items, bytes;
};
AttnPlan attn_plan(const ltq_kv_cache *c, int dtype, uint32_t q_heads, uint64_t seqs, uint64_t table_width, uint64_t max_new, int sms)
{
    AttnPlan p{};
    const uint64_t rows = max_new * (q_heads / c->kv_heads), keys = table_width * c->block_tokens;
    const uint64_t heads = seqs * c->kv_heads, steps = keys / 16;
    // The tensor-core form needs its 256 (128) rows filled to be worth it, the others read the keys once per 8 or 16 rows.
    // Estimates in microseconds from a sweep over 1 to 64 sequences, 32 to 1024 rows, 300 to 4000 keys, head_dim 64, 128, 256:
    //   the others    10 + per row tile and head 0.02 + (0.00025 + head_dim * 0.000004) per 16 keys
    //   tensor cores  3 (6 with a join) + per wave of CTAs 11 + 1.05 (head_dim above 128: 1.7) per 64 keys
    // (8 x 8 heads of 128, 96 rows: 300 keys 29 us against 19, 4000 keys 102 us against 44; 1 x 8 heads, 256 rows: 300 keys 15 us
    // against 23, 4000 keys 46 us against 30).  Where it chose wrongly the other form was at most 28 % faster.
    if (dtype != LTQ_F32 && rows > 16) {
        AttnPlan t{};
        t.tc = true;
        t.rows_per_tile = attn_tc_rows(c->head_dim);
        const uint64_t tiles = (rows + t.rows_per_tile - 1) / t.rows_per_tile, waves = (heads * tiles + sms - 1) / sms;
        // where the groups of row tiles do not fill the device, several CTAs share a group's keys
        const uint64_t most = (keys + 64 * ATTN_TC_MIN_TILES - 1) / (64 * ATTN_TC_MIN_TILES), fit = (uint64_t)sms / (heads * tiles);
        t.splits = (uint32_t)(fit < 1 || most < 1 ? 1 : (most < fit ? most : fit));
        const uint32_t per = attn_rows_per_tile(dtype, c->head_dim, rows);
        const double other = 10 + (double)(heads * ((rows + per - 1) / per)) * (0.02 + (0.00025 + 0.000004 * c->head_dim) * (double)steps);
        const double tc = (t.splits > 1 ? 6 : 3) + (double)waves * (11 + (c->head_dim <= 128 ? 1.05 : 1.7) * (double)(keys / 64) / t.splits);
        if (tc < other && tiles <= 65535) {
            t.row_tiles = (uint32_t)tiles;
            t.ctas = (uint32_t)sms;
            t.items = heads * tiles;
            if (t.splits > 1) {
                t.ml = t.items * t.splits * t.rows_per_tile;
                t.o_floats = t.ml * c->head_dim;
            }
            t.bytes = t.splits > 1 ? t.o_floats * sizeof(float) + t.ml * sizeof(float2) + t.items * sizeof(int2) : 0;
            return t;
        }
    }
    p.rows_per_tile = attn_rows_per_tile(dtype, c->head_dim, rows);
    p.row_tiles = (uint32_t)((rows + p.rows_per_tile - 1) / p.rows_per_tile);
    p.items = heads * p.row_tiles;
    // Few keys: a cluster per item (see cache_attention_cluster_kernel), as many CTAs as the device holds at once, up to eight.
    const uint64_t slots = (uint64_t)sms * attn_ctas_per_sm(dtype, c->head_dim, p.rows_per_tile);
    p.cluster = 8;
    while (p.cluster > 1 && p.items * p.cluster > slots) p.cluster /= 2;
    if (steps <= (uint64_t)p.cluster * ATTN_WARPS * ATTN_CLUSTER_STEPS) {
        return p;   // (no workspace)
    }
    p.cluster = 0;
    const uint64_t most = (p.items * steps + ATTN_MIN_STEPS - 1) / ATTN_MIN_STEPS;
    p.ctas = (uint32_t)(most < slots ? most : slots);
    p.ml = (uint64_t)2 * ATTN_WARPS * p.ctas * p.rows_per_tile;
    p.o_floats = p.ml * c->head_dim;
    p.bytes = p.o_floats * sizeof(float) + p.ml * sizeof(float2) + p.items * sizeof(int2);
    return p;
}

}  // namespace
}  // namespace ltq

using namespace ltq;

extern "C" {

int ltq_cache_append(const ltq_kv_cache *cache, const void *k_dev, const void *v_dev, int dtype, uint64_t ld, uint64_t tokens,
                     const int32_t *offsets_dev, const int32_t *lengths_dev, const int32_t *table_dev, uint64_t seqs, uint64_t table_width,
                     uint64_t max_new, int device, void *stream)
{
    int rc = check_cache(cache);
    if (rc != LTQ_OK) return rc;
    LTQ_REQUIRE(dtype_ok(dtype), LTQ_ERR_INVALID_ARG, "unknown element type %d", dtype);
    if (tokens == 0 || seqs == 0 || max_new == 0) return LTQ_OK;
    LTQ_REQUIRE(k_dev && v_dev, LTQ_ERR_INVALID_ARG, "Invalid argument");
    rc = check_batch(cache, offsets_dev, lengths_dev, table_dev, tokens, seqs, table_width, max_new);
    if (rc != LTQ_OK) return rc;
    const uint64_t row = (uint64_t)cache->kv_heads * cache->head_dim;
    LTQ_REQUIRE(ld >= row && ld < (1ull << 31), LTQ_ERR_INVALID_ARG, "tokens of %llu elements cannot be %llu apart", (unsigned long long)row,
                (unsigned long long)ld);
    LTQ_REQUIRE((((uintptr_t)k_dev | (uintptr_t)v_dev) % dtype_size(dtype)) == 0, LTQ_ERR_INVALID_ARG, "misaligned array");
    LTQ_ENTER_DEVICE(device);
    GemmDevice *dev;
    rc = device_state(device, &dev);
    if (rc != LTQ_OK) return rc;
    LTQ_CUDA_TRY(launch_cache_append(*cache, make_batch(cache, offsets_dev, lengths_dev, table_dev, tokens, seqs, table_width, max_new, dev->status),
                                     k_dev, v_dev, dtype, ld, (cudaStream_t)stream));
    return LTQ_OK;
}

uint64_t ltq_cache_attention_workspace(const ltq_kv_cache *cache, uint64_t tokens, uint32_t q_heads, uint64_t seqs, uint64_t table_width,
                                       uint64_t max_new, int device)
{
    // (0 too where the call itself would be refused for its sizes)
    if (check_cache(cache) != LTQ_OK || q_heads == 0 || q_heads % cache->kv_heads != 0 || q_heads / cache->kv_heads > 1024 || tokens == 0 || seqs == 0 ||
        max_new == 0 || seqs > 65535 || tokens >= (1ull << 31) || max_new > tokens || table_width > 0x7FFFFFFFull / cache->block_tokens ||
        max_new * q_heads >= (1ull << 31))
        return 0;
    DeviceGuard guard(device);
    GemmDevice *dev;
    if (guard.err != cudaSuccess || device_state(device, &dev) != LTQ_OK) return 0;
    const uint64_t a = attn_plan(cache, LTQ_F32, q_heads, seqs, table_width, max_new, dev->sms).bytes;
    const uint64_t b = attn_plan(cache, LTQ_BF16, q_heads, seqs, table_width, max_new, dev->sms).bytes;
    return a > b ? a : b;   // the type of q is not known here
}

int ltq_cache_attention(const ltq_kv_cache *cache, const void *q_dev, int dtype, uint64_t ld_q, uint64_t tokens, uint32_t q_heads,
                        const int32_t *offsets_dev, const int32_t *lengths_dev, const int32_t *table_dev, uint64_t seqs,
                        uint64_t table_width, uint64_t max_new, float scale, void *out_dev, void *workspace_dev, uint64_t workspace_bytes,
                        int device, void *stream)
{
    int rc = check_cache(cache);
    if (rc != LTQ_OK) return rc;
    LTQ_REQUIRE(dtype_ok(dtype), LTQ_ERR_INVALID_ARG, "unknown element type %d", dtype);
    LTQ_REQUIRE(q_heads >= 1 && q_heads % cache->kv_heads == 0 && q_heads / cache->kv_heads <= 1024, LTQ_ERR_INVALID_ARG,
                "%u query heads do not divide over %u key/value heads", q_heads, cache->kv_heads);
    if (tokens == 0 || seqs == 0 || max_new == 0) return LTQ_OK;
    LTQ_REQUIRE(q_dev && out_dev, LTQ_ERR_INVALID_ARG, "Invalid argument");
    rc = check_batch(cache, offsets_dev, lengths_dev, table_dev, tokens, seqs, table_width, max_new);
    if (rc != LTQ_OK) return rc;
    const uint64_t row = (uint64_t)q_heads * cache->head_dim;
    LTQ_REQUIRE(ld_q >= row && ld_q < (1ull << 31), LTQ_ERR_INVALID_ARG, "tokens of %llu elements cannot be %llu apart", (unsigned long long)row,
                (unsigned long long)ld_q);
    LTQ_REQUIRE((((uintptr_t)q_dev | (uintptr_t)out_dev) % dtype_size(dtype)) == 0 && ((uintptr_t)workspace_dev & 15) == 0, LTQ_ERR_INVALID_ARG,
                "misaligned array");
    const float scale_log2 = scale * 1.4426950408889634f;
    LTQ_REQUIRE(scale_log2 - scale_log2 == 0.f, LTQ_ERR_INVALID_ARG, "the softmax scale must be finite, its product with log2(e) too");
    LTQ_REQUIRE(max_new * q_heads < (1ull << 31), LTQ_ERR_TOO_LARGE, "max_new * q_heads must be below 2^31");
    LTQ_ENTER_DEVICE(device);
    GemmDevice *dev;
    rc = device_state(device, &dev);
    if (rc != LTQ_OK) return rc;
    AttnArgs a;
    a.cache = *cache;
    a.bt = make_batch(cache, offsets_dev, lengths_dev, table_dev, tokens, seqs, table_width, max_new, dev->status);
    a.q = q_dev;
    a.out = out_dev;
    a.ld_q = ld_q;
    a.q_heads = q_heads;
    a.group = q_heads / cache->kv_heads;
    a.scale_log2 = scale_log2;
    const AttnPlan p = attn_plan(cache, dtype, q_heads, seqs, table_width, max_new, dev->sms);
    LTQ_REQUIRE(p.bytes == 0 || (workspace_dev && workspace_bytes >= p.bytes), LTQ_ERR_INVALID_ARG, "the workspace holds %llu bytes, %llu are needed",
                (unsigned long long)workspace_bytes, (unsigned long long)p.bytes);
    a.q_vec = ld_q % 4 == 0 && ((uintptr_t)q_dev % (4 * dtype_size(dtype))) == 0;
    a.q_vec8 = (ld_q * dtype_size(dtype)) % 16 == 0 && ((uintptr_t)q_dev & 15) == 0;
    a.out_vec8 = ((uintptr_t)out_dev & 15) == 0;
    a.out_vec = ((uintptr_t)out_dev % (4 * dtype_size(dtype))) == 0;
    a.cluster = p.cluster;
    a.few_rows = 8 * (uint32_t)dev->sms;
    a.splits = p.splits;
    a.ctas = p.ctas;
    a.row_tiles = p.row_tiles;
    a.part_o = static_cast<float *>(workspace_dev);
    a.part_ml = reinterpret_cast<float2 *>(a.part_o + p.o_floats);
    a.item = reinterpret_cast<int2 *>(a.part_ml + p.ml);
    cudaStream_t st = (cudaStream_t)stream;
    if (p.tc) {
        LTQ_CUDA_TRY(launch_attention_tc(a, dtype, st));
        note_kernel("cache_attention_tc_kernel<%s,%u> (keys in %u)", dtype_name(dtype), cache->head_dim, p.splits);
        return LTQ_OK;
    }
    LTQ_CUDA_TRY(dtype == LTQ_F32 ? launch_attention_f32(a, st) : (dtype == LTQ_F16 ? launch_attention_f16(a, st) : launch_attention_bf16(a, st)));
    if (p.cluster) note_kernel("cache_attention_cluster_kernel<%s,%u,%u> (clusters of %u)", dtype_name(dtype), cache->head_dim, p.rows_per_tile, p.cluster);
    else note_kernel("cache_attention_kernel<%s,%u,%u>", dtype_name(dtype), cache->head_dim, p.rows_per_tile);
    return LTQ_OK;
}

}  // extern "C"
