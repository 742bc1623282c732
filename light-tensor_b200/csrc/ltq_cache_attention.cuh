// Attention of a few new tokens over the 8-bit cache, one instantiation per element type of q (the including file defines
// LTQ_ATTN_DT and LTQ_ATTN_LAUNCH).
//
// Reading the cache is the floor (2 * head_dim bytes per key and head); all query heads of a group and all new tokens of a
// sequence share that read.  A warp streams 16 keys at a time straight from global memory into the operand layout of
// mma.m16n8k16, without a pass through shared memory, by transposing the whole computation:
//
//   S^T [16 keys x 8 rows] = K [16 keys x D] . Q^T [D x 8 rows]
//   O^T [D x 8 rows]      += V^T [D x 16 keys] . P^T [16 keys x 8 rows]
//
// (row = one query head of one new token; eight of them fill the MMA's narrow side, so a group of up to eight heads
// wastes nothing).  Which head dimension sits in which column of an operand is free as long as both operands agree, so
// lane (g = lane / 4, c = lane % 4) takes 16 neighbouring bytes of keys g and g + 8 for K and of keys 2c, 2c+1, 2c+8,
// 2c+9 for V: wide loads, whole sectors.  P^T leaves the accumulators transposed and is turned with movmatrix.
//
// A code b becomes the half 1024 + b by putting 0x64 above it (a byte permute) and (code - zero point) by one exact
// subtraction; block scales multiply the float results.  q is scaled by a power of two per row so that halves hold it;
// float q is split into two halves (22 bits), and so are the probabilities then.
//
// Softmax keeps its running maximum only approximately: the reference value m moves when some score exceeds it by more
// than 8 (in base 2), so that probabilities stay below 2^8 and almost every step does without a reduction over lanes.
#include <cuda_fp16.h>

#include "ltq_cache.cuh"
#include "ltq_ptx.cuh"

namespace ltq {

namespace {

constexpr int DT = LTQ_ATTN_DT;
constexpr int TERMS = DT == LTQ_F32 ? 2 : 1;
constexpr int WARPS = 4;
constexpr float MAX_STEP = 8.f;   // how far a score may exceed the reference maximum before it moves

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b)
{
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    const __half2 r = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ float2 unpack2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ uint32_t movmatrix(uint32_t a)
{
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int D>
struct Geo {
    static constexpr int KW = D / 16;   // words of a key that a lane holds for K (4 head dimensions each)
    static constexpr int VW = D / 32;   // words of a key that a lane holds for V
    static constexpr int TILES = D / 16;
    // first head dimension of word w in lane c (K) / lane g (V): segments of 64 / pieces of 128, then what is left
    static __device__ __forceinline__ int k_dim(int w, int c)
    {
        const int seg = w / 4, width = (D - seg * 64) < 64 ? (D - seg * 64) : 64;
        return seg * 64 + c * (width / 4) + 4 * (w % 4);
    }
    static __device__ __forceinline__ int v_dim(int w, int g)
    {
        const int p128 = D / 128, rest = D - p128 * 128;   // rest: 0, 32, 64 or 96
        if (w < p128 * 4) return (w / 4) * 128 + g * 16 + 4 * (w % 4);
        const int r = w - p128 * 4, base = p128 * 128;
        if (rest >= 64) {
            if (r < 2) return base + g * 8 + 4 * r;
            return base + 64 + g * 4;
        }
        return base + g * 4;
    }
};

// `n` words starting at p, in the widest loads that the geometry guarantees (see k_dim / v_dim).
__device__ __forceinline__ void load_words(uint32_t *w, const uint8_t *p, int n)
{
    if (n == 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if (n == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
        w[0] = v.x; w[1] = v.y;
    } else {
        w[0] = __ldg(reinterpret_cast<const uint32_t *>(p));
    }
}

// What a lane holds of 16 keys.
template <int D>
struct Keys {
    uint32_t k[2][Geo<D>::KW];   // keys g, g + 8
    uint32_t v[4][Geo<D>::VW];   // keys 2c, 2c+1, 2c+8, 2c+9
    float ks, vs;
    uint32_t kz, vz;             // 1024 + zero point as a pair of halves
    bool bad;                    // the block id is out of range: none of these keys exists
};

template <int D>
__device__ __forceinline__ void load_keys(Keys<D> &t, const AttnArgs &a, int32_t page, uint32_t h, uint32_t key_in_block, int g, int c)
{
    t.bad = (uint32_t)page >= a.cache.blocks;
    if (t.bad) {
        page = 0;
        if (threadIdx.x % 32 == 0) atomicCAS(a.bt.status, 0u, STATUS_BAD_BLOCK);
    }
    const uint64_t slot = (uint64_t)(uint32_t)page * a.cache.kv_heads + h;
    const uint2 kq = __ldg(reinterpret_cast<const uint2 *>(a.cache.k_qp_dev + slot)), vq = __ldg(reinterpret_cast<const uint2 *>(a.cache.v_qp_dev + slot));
    t.ks = __uint_as_float(kq.x);
    t.vs = __uint_as_float(vq.x);
    t.kz = pack2(1024.f + (float)(kq.y & 0xFF), 1024.f + (float)(kq.y & 0xFF));
    t.vz = pack2(1024.f + (float)(vq.y & 0xFF), 1024.f + (float)(vq.y & 0xFF));
    const uint64_t base = ((slot << a.bt.log2_bt) + key_in_block) * D;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint8_t *p = a.cache.k_dev + base + (uint64_t)(g + 8 * i) * D;
#pragma unroll
        for (int w = 0; w < Geo<D>::KW; w += 4) {
            constexpr int KW = Geo<D>::KW;
            load_words(t.k[i] + w, p + Geo<D>::k_dim(w, c), KW - w >= 4 ? 4 : KW - w);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint8_t *p = a.cache.v_dev + base + (uint64_t)(2 * c + (i & 1) + 8 * (i >> 1)) * D;
        constexpr int P = D / 128, REST = D - P * 128;
#pragma unroll
        for (int w = 0; w < 4 * P; w += 4) load_words(t.v[i] + w, p + Geo<D>::v_dim(w, g), 4);
        if (REST >= 64) load_words(t.v[i] + 4 * P, p + Geo<D>::v_dim(4 * P, g), 2);
        if (REST == 32 || REST == 96) load_words(t.v[i] + Geo<D>::VW - 1, p + Geo<D>::v_dim(Geo<D>::VW - 1, g), 1);
    }
}

template <int D, int NT>
struct Rows {
    uint32_t q[TERMS][NT][D / 16][2];   // Q^T operand
    float scale[NT][2];                 // softmax scale (base 2) over q's power of two, rows 2c and 2c + 1 of each tile
    int pos[NT][2];                     // position of those rows' tokens; -1: no such row
    float m[NT][2], l[NT][2];
    float o[D / 16][NT][4];
};

template <int D, int NT>
__device__ __forceinline__ void load_rows(Rows<D, NT> &r, const AttnArgs &a, const CacheSeq &s, uint32_t h, uint32_t row0, int g, int c)
{
    using T = typename std::conditional<DT == LTQ_F32, float, uint16_t>::type;
    const T *q = static_cast<const T *>(a.q);
    const uint32_t rows = (uint32_t)s.n * a.group;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const uint32_t row = row0 + nt * 8 + g;
        const bool real = row < rows;
        const uint32_t t = row / a.group;
        const T *p = q + ((uint64_t)s.off + t) * a.ld_q + (uint64_t)(h * a.group + row - t * a.group) * D;
        float x[D / 16][4], most = 0.f;
        bool finite = true;
#pragma unroll
        for (int w = 0; w < D / 16; w++) {
            const int d = Geo<D>::k_dim(w, c);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float v = 0.f;
                if (real) {
                    const T raw = p[d + i];
                    if constexpr (DT == LTQ_F32) v = raw;
                    else if constexpr (DT == LTQ_F16) v = __half2float(__ushort_as_half(raw));
                    else v = __uint_as_float((uint32_t)raw << 16);
                }
                x[w][i] = v;
                finite = finite && fabsf(v) < INFINITY;
                most = fmaxf(most, fabsf(v));
            }
        }
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1) {
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
            finite = __shfl_xor_sync(0xFFFFFFFFu, (int)finite, o) && finite;
        }
        // 2^e with most * 2^e in [2^10, 2^11): halves keep 11 bits of entries down to 2^-24 of the largest
        int e = 0;
        if (most > 0.f && finite) {
            e = 10 - ilogbf(most);
            e = e > 100 ? 100 : e;
        }
        const float f = ldexpf(1.f, e);
        float sc = finite ? a.scale_log2 * ldexpf(1.f, -e) : __int_as_float(0x7FC00000);   // an infinity or NaN: the row becomes NaN
#pragma unroll
        for (int w = 0; w < D / 16; w++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float u = finite ? x[w][2 * i] * f : 0.f, v = finite ? x[w][2 * i + 1] * f : 0.f;
                const uint32_t hi = pack2(u, v);
                r.q[0][nt][w][i] = hi;
                if (TERMS == 2) {
                    const float2 b = unpack2(hi);
                    r.q[TERMS - 1][nt][w][i] = pack2(u - b.x, v - b.y);
                }
            }
        }
        const int pos = real ? s.len - s.n + (int)t : -1;
#pragma unroll
        for (int j = 0; j < 2; j++) {   // rows 2c + j live in lanes with g = 2c + j
            r.scale[nt][j] = __shfl_sync(0xFFFFFFFFu, sc, (2 * c + j) * 4);
            r.pos[nt][j] = __shfl_sync(0xFFFFFFFFu, pos, (2 * c + j) * 4);
            r.m[nt][j] = -INFINITY;
            r.l[nt][j] = 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < D / 16; i++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 4; j++) r.o[i][nt][j] = 0.f;
}

// Scores, softmax and accumulation for 16 keys, the first at position key0.
template <int D, int NT>
__device__ __forceinline__ void take_keys(Rows<D, NT> &r, const Keys<D> &t, int key0, int g)
{
    const uint32_t magic = 0x64646464u;
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[nt][j] = 0.f;
#pragma unroll
    for (int w = 0; w < D / 16; w++) {
        const uint32_t a0 = sub2(prmt(t.k[0][w], magic, 0x4140), t.kz), a2 = sub2(prmt(t.k[0][w], magic, 0x4342), t.kz);
        const uint32_t a1 = sub2(prmt(t.k[1][w], magic, 0x4140), t.kz), a3 = sub2(prmt(t.k[1][w], magic, 0x4342), t.kz);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < TERMS; i++) mma16816(s[nt], a0, a1, a2, a3, r.q[i][nt][w][0], r.q[i][nt][w][1]);
    }
    bool up = false;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < 4; j++) {   // j & 1: row 2c + (j & 1); j >> 1: key g or g + 8
            const int key = key0 + g + 8 * (j >> 1);
            s[nt][j] = (key <= r.pos[nt][j & 1] && !t.bad) ? s[nt][j] * (r.scale[nt][j & 1] * t.ks) : -INFINITY;
            up = up || s[nt][j] > r.m[nt][j & 1] + MAX_STEP;
        }
    if (__any_sync(0xFFFFFFFFu, up)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float mx = fmaxf(s[nt][j], s[nt][j + 2]);
#pragma unroll
                for (int o = 4; o <= 16; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
                mx = fmaxf(mx, r.m[nt][j]);
                const float alpha = r.m[nt][j] == mx ? 1.f : exp2_fast(r.m[nt][j] - mx);   // (both -inf: nothing there yet)
                r.m[nt][j] = mx;
                r.l[nt][j] *= alpha;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    r.o[i][nt][j] *= alpha;
                    r.o[i][nt][j + 2] *= alpha;
                }
            }
    }
    uint32_t p[TERMS][NT][2];
    float vs[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float m = r.m[nt][j & 1];
            s[nt][j] = exp2_fast(s[nt][j] - (m == -INFINITY ? 0.f : m));
            r.l[nt][j & 1] += s[nt][j];
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t hi = pack2(s[nt][2 * i], s[nt][2 * i + 1]);
            p[0][nt][i] = movmatrix(hi);
            if (TERMS == 2) {
                const float2 b = unpack2(hi);
                p[TERMS - 1][nt][i] = movmatrix(pack2(s[nt][2 * i] - b.x, s[nt][2 * i + 1] - b.y));
            }
        }
        // a block whose scale is NaN must not reach rows that see none of its keys (0 * NaN)
#pragma unroll
        for (int j = 0; j < 2; j++) vs[nt][j] = (t.vs == t.vs || (key0 <= r.pos[nt][j] && !t.bad)) ? t.vs : 0.f;
    }
#pragma unroll
    for (int w = 0; w < D / 32; w++) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t sel = half ? 0x7362 : 0x5140;
            const uint32_t x = prmt(t.v[0][w], t.v[1][w], sel), y = prmt(t.v[2][w], t.v[3][w], sel);
            const uint32_t a0 = sub2(prmt(x, magic, 0x4140), t.vz), a1 = sub2(prmt(x, magic, 0x4342), t.vz);
            const uint32_t a2 = sub2(prmt(y, magic, 0x4140), t.vz), a3 = sub2(prmt(y, magic, 0x4342), t.vz);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < TERMS; i++) mma16816(d, a0, a1, a2, a3, p[i][nt][0], p[i][nt][1]);
#pragma unroll
                for (int j = 0; j < 4; j++) r.o[2 * w + half][nt][j] = fmaf(vs[nt][j & 1], d[j], r.o[2 * w + half][nt][j]);
            }
        }
    }
}

template <int D, int NT>
struct Shared {
    float o[WARPS][8 * NT][D + 4];   // + 4: rows start in different banks
    float m[WARPS][8 * NT], l[WARPS][8 * NT];
};

// Grid: (splits * row tiles, kv_heads, sequences).  The keys that a row tile can see are cut into `splits` equal runs of 16-key
// steps, a run into four for the warps; the four results meet in shared memory.
template <int D, int NT>
__global__ void __launch_bounds__(32 * WARPS)
cache_attention_kernel(const AttnArgs a, uint32_t row_tiles)
{
    griddep_launch_dependents();
    griddep_wait();
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Shared<D, NT> &sh = *reinterpret_cast<Shared<D, NT> *>(smem_raw);
    const uint32_t b = blockIdx.z, h = blockIdx.y, split = blockIdx.x / row_tiles, row0 = (blockIdx.x - split * row_tiles) * 8 * NT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const CacheSeq s = cache_seq(a.bt, b);
    const uint32_t rows = s.ok ? (uint32_t)s.n * a.group : 0u;
    if (row0 >= rows) return;
    const uint32_t last = row0 + 8 * NT < rows ? row0 + 8 * NT - 1 : rows - 1;
    const int keys = s.len - s.n + (int)(last / a.group) + 1;             // what the tile's last row sees
    const uint32_t steps = keys > 0 ? ((uint32_t)keys + 15) / 16 : 0u;
    const uint32_t c0 = (uint32_t)((uint64_t)steps * split / a.splits), c1 = (uint32_t)((uint64_t)steps * (split + 1) / a.splits);
    const uint32_t w0 = c0 + (c1 - c0) * warp / WARPS, w1 = c0 + (c1 - c0) * (warp + 1) / WARPS;

    Rows<D, NT> r;
    load_rows<D, NT>(r, a, s, h, row0, g, c);
    if (w0 < w1) {
        const int32_t *table = a.bt.table + (uint64_t)b * a.bt.table_width;
        const int sh16 = a.bt.log2_bt - 4;                    // steps per block, log2
        const uint32_t in_block = (1u << sh16) - 1;
        Keys<D> cur, nxt;
        load_keys<D>(cur, a, __ldg(table + (w0 >> sh16)), h, (w0 & in_block) * 16, g, c);
        int32_t page = w0 + 1 < w1 ? __ldg(table + ((w0 + 1) >> sh16)) : 0;
        for (uint32_t st = w0; st < w1; st++) {
            if (st + 1 < w1) load_keys<D>(nxt, a, page, h, ((st + 1) & in_block) * 16, g, c);
            if (st + 2 < w1) page = __ldg(table + ((st + 2) >> sh16));
            take_keys<D, NT>(r, cur, (int)(st * 16), g);
            cur = nxt;
        }
    }
    // this warp's share -> shared memory
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            float l = r.l[nt][j];
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
            if (g == 0) {
                sh.m[warp][nt * 8 + 2 * c + j] = r.m[nt][j];
                sh.l[warp][nt * 8 + 2 * c + j] = l;
            }
#pragma unroll
            for (int w = 0; w < D / 32; w++) {
                const float4 v = make_float4(r.o[2 * w][nt][j], r.o[2 * w][nt][j + 2], r.o[2 * w + 1][nt][j], r.o[2 * w + 1][nt][j + 2]);
                *reinterpret_cast<float4 *>(&sh.o[warp][nt * 8 + 2 * c + j][Geo<D>::v_dim(w, g)]) = v;
            }
        }
    __syncthreads();
    using T = typename std::conditional<DT == LTQ_F32, float, uint16_t>::type;
    T *out = static_cast<T *>(a.out);
    for (uint32_t i = threadIdx.x; i < 8 * NT * (D / 4); i += 32 * WARPS) {
        const uint32_t rr = i / (D / 4), d = (i - rr * (D / 4)) * 4, row = row0 + rr;
        if (row >= rows) break;
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) m = fmaxf(m, sh.m[w][rr]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float mw = sh.m[w][rr], f = mw == m ? 1.f : exp2_fast(mw - m);
            const float4 v = *reinterpret_cast<const float4 *>(&sh.o[w][rr][d]);
            l = fmaf(f, sh.l[w][rr], l);
            o.x = fmaf(f, v.x, o.x);
            o.y = fmaf(f, v.y, o.y);
            o.z = fmaf(f, v.z, o.z);
            o.w = fmaf(f, v.w, o.w);
        }
        const uint32_t t = row / a.group;
        const uint64_t at = ((uint64_t)s.off + t) * a.q_heads + h * a.group + (row - t * a.group);
        if (a.splits > 1) {
            const uint64_t slot = (uint64_t)split * a.bt.tokens * a.q_heads + at;
            *reinterpret_cast<float4 *>(a.part_o + slot * D + d) = o;
            if (d == 0) a.part_ml[slot] = make_float2(m, l);
        } else {
            const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);   // a row that sees nothing: zeros
            T *p = out + at * D + d;
            const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if constexpr (DT == LTQ_F32) p[k] = y[k];
                else p[k] = (T)token_bits<DT>(y[k]);
            }
        }
    }
}

// Joins the splits: one warp per (new token, query head).
template <int D>
__global__ void __launch_bounds__(256)
cache_attention_join_kernel(const AttnArgs a)
{
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const CacheSeq s = cache_seq(a.bt, blockIdx.y);
    const uint32_t i = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (!s.ok || i >= (uint32_t)s.n * a.q_heads) return;
    const uint64_t at = (uint64_t)s.off * a.q_heads + i, pitch = a.bt.tokens * a.q_heads;
    float m = -INFINITY;
    for (uint32_t k = 0; k < a.splits; k++) m = fmaxf(m, a.part_ml[k * pitch + at].x);
    float l = 0.f;
    float o[(D + 31) / 32];
#pragma unroll
    for (int j = 0; j < D / 32; j++) o[j] = 0.f;
    for (uint32_t k = 0; k < a.splits; k++) {
        const float2 ml = a.part_ml[k * pitch + at];
        const float f = ml.x == m ? 1.f : exp2_fast(ml.x - m);
        l = fmaf(f, ml.y, l);
#pragma unroll
        for (int j = 0; j < D / 32; j++) o[j] = fmaf(f, a.part_o[(k * pitch + at) * D + 32 * j + lane], o[j]);
    }
    const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
    using T = typename std::conditional<DT == LTQ_F32, float, uint16_t>::type;
    T *p = static_cast<T *>(a.out) + at * D;
#pragma unroll
    for (int j = 0; j < D / 32; j++) {
        if constexpr (DT == LTQ_F32) p[32 * j + lane] = o[j] * inv;
        else p[32 * j + lane] = (T)token_bits<DT>(o[j] * inv);
    }
}

template <int D, int NT>
cudaError_t launch_nt(const AttnArgs &a, cudaStream_t stream)
{
    constexpr size_t smem = sizeof(Shared<D, NT>);
    static bool attr_done[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (smem > 48 * 1024 && dev >= 0 && dev < 64 && !attr_done[dev]) {
        e = cudaFuncSetAttribute(cache_attention_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        attr_done[dev] = true;
    }
    const uint32_t row_tiles = (a.bt.max_new * a.group + 8 * NT - 1) / (8 * NT);
    e = launch_chained(cache_attention_kernel<D, NT>, dim3(a.splits * row_tiles, a.cache.kv_heads, a.bt.seqs), dim3(32 * WARPS), smem, stream, a,
                       row_tiles);
    count_launch();
    if (e != cudaSuccess || a.splits == 1) return e;
    e = launch_chained(cache_attention_join_kernel<D>, dim3((a.bt.max_new * a.q_heads + 7) / 8, a.bt.seqs), dim3(256), 0, stream, a);
    count_launch();
    return e;
}

template <int D>
cudaError_t launch_d(const AttnArgs &a, cudaStream_t stream)
{
    if constexpr (D * TERMS <= 128) {
        if (attn_rows_per_tile(DT, D, (uint64_t)a.bt.max_new * a.group) == 16) return launch_nt<D, 2>(a, stream);
    }
    return launch_nt<D, 1>(a, stream);
}

}  // namespace

cudaError_t LTQ_ATTN_LAUNCH(const AttnArgs &a, cudaStream_t stream)
{
    switch (a.cache.head_dim) {
        case 32: return launch_d<32>(a, stream);
        case 64: return launch_d<64>(a, stream);
        case 96: return launch_d<96>(a, stream);
        case 128: return launch_d<128>(a, stream);
        case 192: return launch_d<192>(a, stream);
        case 256: return launch_d<256>(a, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace ltq
