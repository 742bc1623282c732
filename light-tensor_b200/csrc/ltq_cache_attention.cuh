// Attention of a few new tokens over the 8-bit cache, one instantiation per element type of q (the including file defines
// LTQ_ATTN_DT, LTQ_ATTN_LAUNCH and, where the type has a tensor-core form, LTQ_ATTN_JOIN).
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
// The next step's bytes are on their way into registers while a step is computed (4 KB per warp at head_dim 128, 48 KB per SM).
//
// Work is divided evenly whatever the lengths are: the steps of all (sequence, row tile, head) items in a row are cut into
// equal ranges, one per resident warp.  A warp finishes the items that lie inside its range and leaves its part of the one
// or two that reach beyond it in the workspace, for the join kernel.  Warps never wait for one another, so that the start and
// end of one's range passes under the others' reading.  (Ranges per CTA, its warps joined in shared memory: 27 us of the
// 126 us of 64 sequences of 2048 to 8192 tokens went there.)
//
// Past that the kernel is bound by instruction issue, so a step is kept short:
//  * a code b with a zero byte above it IS a half, the subnormal b * 2^-24, which the tensor core multiplies exactly: one byte
//    permute per two codes of K, whose zero points come off the scores, q . (k - z) = q . k - z * sum(q);
//  * V's zero points come off the codes first (1024 + code - (1024 + zero point), exact in halves).  The tensor core cuts off what does
//    not fit a sum, always towards zero: O added up over thousands of steps from positive codes around 128 drifted (256 sequences
//    of 32 000 keys, half: 1.2e-2 off, now 2.9e-4; with 18 000 steps per warp, all that the device's memory holds, 3.8e-4);
//  * q is scaled by a power of two per row so that halves hold it (float q: split into two halves, 22 bits, and so are
//    the probabilities then, K's zero points come off the codes as well, and every product starts from zero and is added up in
//    float: 742 new tokens of 1364 were off by 1.6e-5 otherwise, now by 3e-7);
//  * V's block scales go into the probabilities, so that one accumulator serves all.  What halves have to hold is then the weight
//    exp2(score) * V scale, and its reference is the row's own: m + d, with m the reference of the scores (and of the sum of the
//    probabilities) and 2^d what V's scale adds to the largest weight.  (With the largest V scale in sight as the reference, one
//    loud block that a row gives no weight took the bits of all others: 2^22 times louder, outputs were 2 % off and more.)
//  * both references are kept only approximately: they move when a score exceeds m, or a weight m + d, by more than 8 (base 2), so
//    that almost every step does without a reduction over lanes.  A row's largest weight is 2^6 or more then, not 1: halves end
//    at 2^16, and what they lose below 2^-14 (2^-25 at most) lies further from the largest.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "ltq_cache.cuh"
#include "ltq_ptx.cuh"

namespace ltq {

namespace {

constexpr int DT = LTQ_ATTN_DT;
constexpr int TERMS = DT == LTQ_F32 ? 2 : 1;
constexpr int WARPS = ATTN_WARPS;
constexpr uint32_t AHEAD = 2;     // steps beyond the one on its way into registers that are asked into L2
constexpr float MAX_STEP = 8.f;   // how far a score or a weight may exceed its reference before that moves
constexpr int HEAD = 7;           // a weight at its reference is 2^HEAD: with MAX_STEP above it still a half
constexpr float LARGE = 180.f;    // factors up to this, 2^(HEAD + 0.49), need no look at the weights
constexpr float QUIET = -118.f;   // V scales below 2^this do not lower the reference further, so that 2^(HEAD - d) stays a float
constexpr float LOUD = 1.2676506e30f;   // 2^100: no weight's factor is larger (probabilities that reach it are below 2^-85)

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
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
__device__ __forceinline__ float log2_fast(float x)
{
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float power2(int e) { return __int_as_float((127 + e) << 23); }        // 2^e, -126 <= e <= 127
__device__ __forceinline__ int exponent_of(float p) { return (__float_as_int(p) >> 23) - 127; }   // of a power of two

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

// The pieces (16, 8 and 4 bytes) that a lane holds of one key, for K and for V.
template <int D>
struct Piece {
    static constexpr int K16 = D / 64, K8 = (D % 64) / 32;
    static constexpr int V16 = D / 128, V8 = (D % 128) >= 64, V4 = (D % 64) / 32;
};

// Byte offsets of a lane's first piece of each size within 16 keys, the rest lies at constant distances from them.
template <int D>
struct LaneOffsets {
    uint32_t k16, k8, v16, v8, v4;
    __device__ __forceinline__ LaneOffsets(int lane)
    {
        const int g = lane >> 2, c = lane & 3;
        k16 = g * D + Geo<D>::k_dim(0, c);
        k8 = g * D + Geo<D>::k_dim(Geo<D>::KW - 1, c) - 4;
        v16 = 2 * c * D + Geo<D>::v_dim(0, g);
        v8 = 2 * c * D + Geo<D>::v_dim(4 * Piece<D>::V16, g);
        v4 = 2 * c * D + Geo<D>::v_dim(Geo<D>::VW - 1, g);
    }
};

// What a lane holds of 16 keys, and their block's parameters.
template <int D>
struct Keys {
    uint32_t k[2][Geo<D>::KW];   // keys g, g + 8
    uint32_t v[4][Geo<D>::VW];   // keys 2c, 2c+1, 2c+8, 2c+9
    uint2 k_par, v_par;          // scale, zero point
    bool bad;                    // the block id is out of range: none of these keys exists
};

__device__ __forceinline__ void load16(uint32_t *w, const uint8_t *p)
{
    const uint4 x = __ldg(reinterpret_cast<const uint4 *>(p));
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
}
__device__ __forceinline__ void load8(uint32_t *w, const uint8_t *p)
{
    const uint2 x = __ldg(reinterpret_cast<const uint2 *>(p));
    w[0] = x.x; w[1] = x.y;
}

template <int D>
__device__ __forceinline__ void fetch_keys(Keys<D> &t, const AttnArgs &a, const LaneOffsets<D> &at, int32_t page, uint32_t h, uint32_t key_in_block)
{
    t.bad = (uint32_t)page >= a.cache.blocks;
    if (t.bad) {
        page = 0;
        if (threadIdx.x % 32 == 0) atomicCAS(a.bt.refused, 0u, REFUSED_BLOCK);
    }
    const uint64_t slot = (uint64_t)(uint32_t)page * a.cache.kv_heads + h, base = ((slot << a.bt.log2_bt) + key_in_block) * D;
    t.k_par = __ldg(reinterpret_cast<const uint2 *>(a.cache.k_qp_dev + slot));
    t.v_par = __ldg(reinterpret_cast<const uint2 *>(a.cache.v_qp_dev + slot));
    const uint8_t *k = a.cache.k_dev + base, *v = a.cache.v_dev + base;
#pragma unroll
    for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int j = 0; j < Piece<D>::K16; j++) load16(t.k[i] + 4 * j, k + at.k16 + (8 * i * D + 64 * j));
        if (Piece<D>::K8) load8(t.k[i] + 4 * Piece<D>::K16, k + at.k8 + 8 * i * D);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int key = ((i & 1) + 8 * (i >> 1)) * D;
#pragma unroll
        for (int j = 0; j < Piece<D>::V16; j++) load16(t.v[i] + 4 * j, v + at.v16 + (key + 128 * j));
        if (Piece<D>::V8) load8(t.v[i] + 4 * Piece<D>::V16, v + at.v8 + key);
        if (Piece<D>::V4) t.v[i][Geo<D>::VW - 1] = __ldg(reinterpret_cast<const uint32_t *>(v + at.v4 + key));
    }
}

// Asks 16 keys of a block into L2: one line per lane and round.
template <int D>
__device__ __forceinline__ void ask_keys(const AttnArgs &a, int32_t page, uint32_t h, uint32_t key_in_block, int lane)
{
    if ((uint32_t)page >= a.cache.blocks) return;
    const uint64_t base = ((((uint64_t)(uint32_t)page * a.cache.kv_heads + h) << a.bt.log2_bt) + key_in_block) * D;
    constexpr int LINES = 16 * D / 128;   // of K, and of V
#pragma unroll
    for (int i = 0; i < (2 * LINES + 31) / 32; i++) {
        const int line = i * 32 + lane;
        if (line < 2 * LINES) {
            const uint8_t *p = (line < LINES ? a.cache.k_dev + base + line * 128 : a.cache.v_dev + base + (line - LINES) * 128);
            asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
        }
    }
}

template <int D, int NT>
struct Rows {
    uint32_t q[TERMS][NT][D / 16][2];   // Q^T operand
    float scale[NT][2];                 // softmax scale (base 2) over q's power of two, rows 2c and 2c + 1 of each tile
    float q_sum[NT][2];                 // sum of the row's q, as the operand holds it
    int pos[NT][2];                     // position of those rows' tokens (rows that do not exist see everything, with q = 0)
    int first_pos;                      // the smallest of the warp's
    float m[NT][2], l[NT][2];
    float o[D / 16][NT][4];             // sum of weight * (code - zero point)
    float g[NT][2];                     // 2^(HEAD - d): weight = probability * V scale * g
};
constexpr float CODE = 16777216.f;      // 2^24: a code's half is the code over this
constexpr bool EXACT = TERMS == 2;      // K's codes as the halves code - zero point instead, and sums in float, see above

// Two codes of a word as an operand: bytes `sel` picks of w and, above each, of what makes it a half.  OFF: without the zero point (`zero`:
// 1024 + it, twice).
template <bool OFF>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, uint32_t sel, uint32_t zero)
{
    if (!OFF) return prmt(w, 0, sel);
    const uint32_t x = prmt(w, 0x64646464u, sel);   // 1024 + code
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&x), *reinterpret_cast<const __half2 *>(&zero));
    return *reinterpret_cast<const uint32_t *>(&r);
}

template <int D, int NT>
__device__ __forceinline__ void load_rows(Rows<D, NT> &r, const AttnArgs &a, const CacheSeq &s, uint32_t h, uint32_t row0, int g, int c)
{
    using T = typename std::conditional<DT == LTQ_F32, float, uint16_t>::type;
    using Four = typename std::conditional<DT == LTQ_F32, float4, uint2>::type;
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
            T raw[4] = {0, 0, 0, 0};
            if (real) {
                if (a.q_vec) {
                    *reinterpret_cast<Four *>(raw) = __ldg(reinterpret_cast<const Four *>(p + d));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) raw[i] = p[d + i];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float v;
                if constexpr (DT == LTQ_F32) v = raw[i];
                else if constexpr (DT == LTQ_F16) v = __half2float(__ushort_as_half(raw[i]));
                else v = __uint_as_float((uint32_t)raw[i] << 16);
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
        const float sc = finite ? a.scale_log2 * ldexpf(1.f, -e) : __int_as_float(0x7FC00000);   // an infinity or NaN: the row becomes NaN
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < D / 16; w++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float u = finite ? x[w][2 * i] * f : 0.f, v = finite ? x[w][2 * i + 1] * f : 0.f;
                const uint32_t hi = pack2(u, v);
                const float2 b = unpack2(hi);
                r.q[0][nt][w][i] = hi;
                sum += b.x + b.y;
                if (TERMS == 2) {
                    const uint32_t lo = pack2(u - b.x, v - b.y);
                    const float2 d = unpack2(lo);
                    r.q[TERMS - 1][nt][w][i] = lo;
                    sum += d.x + d.y;
                }
            }
        }
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        const int pos = real ? s.len - s.n + (int)t : 0x7FFFFFFF;
#pragma unroll
        for (int j = 0; j < 2; j++) {   // rows 2c + j live in lanes with g = 2c + j
            r.scale[nt][j] = __shfl_sync(0xFFFFFFFFu, sc, (2 * c + j) * 4);
            r.q_sum[nt][j] = __shfl_sync(0xFFFFFFFFu, sum, (2 * c + j) * 4);
            r.g[nt][j] = power2(HEAD);
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
    int first = 0x7FFFFFFF;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) first = min(first, min(r.pos[nt][0], r.pos[nt][1]));
    r.first_pos = __reduce_min_sync(0xFFFFFFFFu, first);
}

// Scores, softmax and accumulation for 16 keys, the first at position key0.
template <int D, int NT>
__device__ __forceinline__ void take_keys(Rows<D, NT> &r, const Keys<D> &keys, int key0, int g)
{
    const float k_scale = __uint_as_float(keys.k_par.x), v_scale = __uint_as_float(keys.v_par.x);
    const float k_zero = (float)(keys.k_par.y & 0xFF);
    const bool bad = keys.bad;
    const uint32_t k_zero2 = 0x64006400u + (keys.k_par.y & 0xFF) * 0x10001u, v_zero2 = 0x64006400u + (keys.v_par.y & 0xFF) * 0x10001u;
    float acc[NT][2][4];   // two chains: an MMA waits for the one before it on the same accumulator 
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[nt][0][j] = acc[nt][1][j] = 0.f;
#pragma unroll
    for (int w = 0; w < D / 16; w++) {
        const uint32_t a0 = code_pair<EXACT>(keys.k[0][w], 0x4140, k_zero2), a2 = code_pair<EXACT>(keys.k[0][w], 0x4342, k_zero2);
        const uint32_t a1 = code_pair<EXACT>(keys.k[1][w], 0x4140, k_zero2), a3 = code_pair<EXACT>(keys.k[1][w], 0x4342, k_zero2);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            if (EXACT) {
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = TERMS - 1; i >= 0; i--) mma16816(part, a0, a1, a2, a3, r.q[i][nt][w][0], r.q[i][nt][w][1]);
#pragma unroll
                for (int j = 0; j < 4; j++) acc[nt][w & 1][j] += part[j];
            } else {
                mma16816(acc[nt][w & 1], a0, a1, a2, a3, r.q[0][nt][w][0], r.q[0][nt][w][1]);
            }
        }
    }

    // t = score - m.  Of element j: row 2c + (j & 1), key g + 8 * (j >> 1).
    float t[NT][4], sc[NT][2], zo[NT][2];
    const bool masked = bad || key0 + 15 > r.first_pos;
    float top = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const float x = r.scale[nt][j] * k_scale;
            sc[nt][j] = EXACT ? x : x * CODE;
            zo[nt][j] = EXACT ? 0.f : x * (k_zero * r.q_sum[nt][j]);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            acc[nt][0][j] += acc[nt][1][j];
            t[nt][j] = fmaf(acc[nt][0][j], sc[nt][j & 1], -(zo[nt][j & 1] + r.m[nt][j & 1]));
        }
    }
    auto mask = [&](float (&x)[NT][4]) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (bad || key0 + g + 8 * (j >> 1) > r.pos[nt][j & 1]) x[nt][j] = -INFINITY;
    };
    if (masked) mask(t);
    // what makes a probability of a row a weight
    float f[NT][2];
    auto factors = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) f[nt][j] = fminf(v_scale * r.g[nt][j], LOUD);
    };
    factors();
    float loudest = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int j = 0; j < 4; j++) top = fmaxf(top, t[nt][j]);
        loudest = fmaxf(loudest, fmaxf(f[nt][0], f[nt][1]));
    }
    bool move = __any_sync(0xFFFFFFFFu, top > MAX_STEP || loudest > LARGE);   // (also the first time: m is -inf, t +inf)
    if (move && __all_sync(0xFFFFFFFFu, top <= MAX_STEP)) {   // a block louder than what a row's reference stands on: do its weights reach the limit?
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) top = fmaxf(top, fmaxf(t[nt][j], t[nt][j + 2]) + (log2_fast(f[nt][j]) - (float)HEAD));
        move = __any_sync(0xFFFFFFFFu, top > MAX_STEP);
    }
    if (move) {
        const float v_log = fminf(fmaxf(log2_fast(v_scale), QUIET), 128.f);   // (NaN: QUIET)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 4; j++) t[nt][j] = fmaf(acc[nt][0][j], sc[nt][j & 1], -zo[nt][j & 1]);
        if (masked) mask(t);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float here = fmaxf(t[nt][j], t[nt][j + 2]);
#pragma unroll
                for (int o = 4; o <= 16; o <<= 1) here = fmaxf(here, __shfl_xor_sync(0xFFFFFFFFu, here, o));
                const float mx = fmaxf(here, r.m[nt][j]), down = r.m[nt][j] == mx ? 0.f : r.m[nt][j] - mx;   // (both -inf: nothing there yet)
                const float m = mx == -INFINITY ? 0.f : mx;
                const int d = HEAD - exponent_of(r.g[nt][j]);
                int d_new = d;
                if (mx != -INFINITY) d_new = (int)ceilf(fmaxf(down + (float)d, here - mx + v_log));
                const float alpha = exp2_fast(down), beta = exp2_fast(down + (float)(d - d_new));
                t[nt][j] -= m;
                t[nt][j + 2] -= m;
                r.m[nt][j] = mx;
                r.l[nt][j] *= alpha;
                r.g[nt][j] = power2(HEAD - d_new);
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    r.o[i][nt][j] *= beta;
                    r.o[i][nt][j + 2] *= beta;
                }
            }
        factors();
    }
    uint32_t p[TERMS][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            t[nt][j] = exp2_fast(t[nt][j]);
            r.l[nt][j & 1] += t[nt][j];
        }
        float f0 = f[nt][0], f1 = f[nt][1];
        if (!(v_scale < INFINITY)) {   // a block whose scale is NaN reaches the rows that see one of its keys, and no others (0 * NaN)
            f0 = key0 <= r.pos[nt][0] && !bad ? __int_as_float(0x7FC00000) : 0.f;
            f1 = key0 <= r.pos[nt][1] && !bad ? __int_as_float(0x7FC00000) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float x = t[nt][2 * i] * f0, y = t[nt][2 * i + 1] * f1;
            const uint32_t hi = pack2(x, y);
            p[0][nt][i] = movmatrix(hi);
            if (TERMS == 2) {
                const float2 b = unpack2(hi);
                p[TERMS - 1][nt][i] = movmatrix(pack2(x - b.x, y - b.y));
            }
        }
    }
#pragma unroll
    for (int w = 0; w < D / 32; w++) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t sel = half ? 0x7362 : 0x5140;
            const uint32_t x = prmt(keys.v[0][w], keys.v[1][w], sel), y = prmt(keys.v[2][w], keys.v[3][w], sel);
            const uint32_t a0 = code_pair<true>(x, 0x4140, v_zero2), a1 = code_pair<true>(x, 0x4342, v_zero2);
            const uint32_t a2 = code_pair<true>(y, 0x4140, v_zero2), a3 = code_pair<true>(y, 0x4342, v_zero2);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                if (EXACT) {
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = TERMS - 1; i >= 0; i--) mma16816(part, a0, a1, a2, a3, p[i][nt][0], p[i][nt][1]);
#pragma unroll
                    for (int j = 0; j < 4; j++) r.o[2 * w + half][nt][j] += part[j];
                } else {
                    mma16816(r.o[2 * w + half][nt], a0, a1, a2, a3, p[0][nt][0], p[0][nt][1]);
                }
            }
        }
    }
}

// Steps of one (row tile, head) of a sequence: 16 keys each, by its longest row tile, and at least one (rows without keys get
// their zeros that way).  Row tiles of a long run of new tokens see fewer keys than the last one does; their surplus is empty.
__device__ __forceinline__ uint32_t item_steps(const CacheSeq &s) { return s.len > 16 ? ((uint32_t)s.len + 15) / 16 : 1u; }
__device__ __forceinline__ unsigned long long seq_steps(const AttnArgs &a, const CacheSeq &s, uint32_t rows_per_tile)
{
    if (!s.ok || s.n == 0) return 0;
    return (unsigned long long)item_steps(s) * (((uint32_t)s.n * a.group + rows_per_tile - 1) / rows_per_tile) * a.cache.kv_heads;
}
// How many warps take part: none with fewer than MIN_STEPS steps.
__device__ __forceinline__ unsigned long long active_warps(const AttnArgs &a, unsigned long long total)
{
    const unsigned long long most = (total + ATTN_MIN_STEPS - 1) / ATTN_MIN_STEPS, there = (unsigned long long)a.ctas * WARPS;
    return most < there ? most : there;
}

template <int D>
__device__ __forceinline__ void store4(const AttnArgs &a, uint64_t row, int d, float x, float y, float z, float w)
{
    if constexpr (DT == LTQ_F32) {
        float *p = static_cast<float *>(a.out) + row * D + d;
        if (a.out_vec) *reinterpret_cast<float4 *>(p) = make_float4(x, y, z, w);
        else p[0] = x, p[1] = y, p[2] = z, p[3] = w;
    } else {
        uint16_t *p = static_cast<uint16_t *>(a.out) + row * D + d;
        const uint32_t lo = token_bits2<DT>(x, y), hi = token_bits2<DT>(z, w);
        if (a.out_vec) *reinterpret_cast<uint2 *>(p) = make_uint2(lo, hi);
        else p[0] = (uint16_t)lo, p[1] = (uint16_t)(lo >> 16), p[2] = (uint16_t)hi, p[3] = (uint16_t)(hi >> 16);
    }
}

// What a row tile's last row sees, in steps.
__device__ __forceinline__ uint32_t seen_steps(const AttnArgs &a, const CacheSeq &s, uint32_t row0, uint32_t rows_per_tile)
{
    const uint32_t rows = (uint32_t)s.n * a.group, last = row0 + rows_per_tile < rows ? row0 + rows_per_tile - 1 : rows - 1;
    const int keys = s.len - s.n + (int)(last / a.group) + 1;
    return keys > 0 ? ((uint32_t)keys + 15) / 16 : 0u;
}

// One warp takes steps [w0, w1) of one item into `r`.
template <int D, int NT>
__device__ __forceinline__ void take_steps(Rows<D, NT> &r, const AttnArgs &a, uint32_t b, const CacheSeq &s, uint32_t h, uint32_t row0,
                                           uint32_t w0, uint32_t w1)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int32_t *table = a.bt.table + (uint64_t)b * a.bt.table_width;
    const int sh16 = a.bt.log2_bt - 4;                                    // steps per block, log2
    const uint32_t in_block = (1u << sh16) - 1;
    const LaneOffsets<D> at(lane);
    Keys<D> even, odd;
    int32_t page = 0, page_ahead = 0;   // blocks of the steps to be fetched, and to be asked into L2, next
    auto fetch = [&](Keys<D> &into, uint32_t st) {
        if (st < w1) {
            fetch_keys<D>(into, a, at, page, h, (st & in_block) * 16);
            if (st + 1 < w1) page = __ldg(table + ((st + 1) >> sh16));
        }
    };
    auto ask = [&](uint32_t st) {
        if (st < w1) {
            ask_keys<D>(a, page_ahead, h, (st & in_block) * 16, lane);
            if (st + 1 < w1) page_ahead = __ldg(table + ((st + 1) >> sh16));
        }
    };
    if (w0 < w1) page = __ldg(table + (w0 >> sh16));
    if (w0 + 1 < w1) page_ahead = __ldg(table + ((w0 + 1) >> sh16));
    fetch(even, w0);
    for (uint32_t i = 1; i <= AHEAD; i++) ask(w0 + i);
    load_rows<D, NT>(r, a, s, h, row0, g, c);
    for (uint32_t st = w0; st < w1; st += 2) {
        fetch(odd, st + 1);
        ask(st + 1 + AHEAD);
        take_keys<D, NT>(r, even, (int)(st * 16), g);
        if (st + 1 >= w1) break;
        fetch(even, st + 2);
        ask(st + 2 + AHEAD);
        take_keys<D, NT>(r, odd, (int)(st * 16) + 16, g);
    }
}

// One warp's part [first, end) of the steps of one item; the result goes to `out` if the part is the whole item, to workspace
// slot `slot` otherwise.
template <int D, int NT>
__device__ __forceinline__ void do_segment(const AttnArgs &a, uint32_t b, const CacheSeq &s, uint32_t h, uint32_t row0, uint32_t first,
                                           uint32_t end, bool whole, uint32_t slot)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const uint32_t rows = (uint32_t)s.n * a.group, seen = seen_steps(a, s, row0, 8 * NT);
    Rows<D, NT> r;
    take_steps<D, NT>(r, a, b, s, h, row0, first, end < seen ? end : seen);
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < 2; j++) {   // row 2c + j of the tile: its lanes are those with the same c
            float l = r.l[nt][j];
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
            const uint32_t rr = nt * 8 + 2 * c + j, row = row0 + rr;
            if (row >= rows) continue;
            const uint32_t t = row / a.group;
            const uint64_t out_row = ((uint64_t)s.off + t) * a.q_heads + h * a.group + (row - t * a.group);
            const uint64_t place = (uint64_t)slot * 8 * NT + rr;
            const float f = whole ? (l == 0.f ? 0.f : __fdiv_rn(1.f, l)) : 1.f;   // (a row that sees nothing: zeros)
            const float back = power2(-exponent_of(r.g[nt][j]));
#pragma unroll
            for (int w = 0; w < D / 32; w++) {
                auto real = [&](float x) { return x * f * back; };
                const float x0 = real(r.o[2 * w][nt][j]), x1 = real(r.o[2 * w][nt][j + 2]);
                const float x2 = real(r.o[2 * w + 1][nt][j]), x3 = real(r.o[2 * w + 1][nt][j + 2]);
                const int d = Geo<D>::v_dim(w, g);
                if (whole) store4<D>(a, out_row, d, x0, x1, x2, x3);
                else *reinterpret_cast<float4 *>(a.part_o + place * D + d) = make_float4(x0, x1, x2, x3);
            }
            if (!whole && g == 0) a.part_ml[place] = make_float2(r.m[nt][j], l);
        }
}

template <int D, int NT>
__global__ void __launch_bounds__(32 * WARPS, (D * NT * TERMS <= 128 ? 3 : 2))
cache_attention_kernel(const __grid_constant__ AttnArgs a)
{
    griddep_launch_dependents();
    griddep_wait();
    __shared__ unsigned long long before[32 * WARPS], s_total;   // prefix sums of the sequences' steps
    constexpr uint32_t ROWS = 8 * NT;
    // Where this warp's range begins: every thread adds up a run of sequences, the run with the beginning is then walked.
    const uint32_t run = (a.bt.seqs + 32 * WARPS - 1) / (32 * WARPS), b0 = threadIdx.x * run;
    unsigned long long mine = 0;
    for (uint32_t b = b0; b < b0 + run && b < a.bt.seqs; b++) {
        const CacheSeq s = cache_seq(a.bt, b);
        if (!s.ok) atomicCAS(a.bt.refused, 0u, REFUSED_SEQUENCE);
        mine += seq_steps(a, s, ROWS);
    }
    before[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x < 32) {
        unsigned long long v[WARPS], sum = 0;
#pragma unroll
        for (int k = 0; k < WARPS; k++) {
            v[k] = before[threadIdx.x * WARPS + k];
            sum += v[k];
        }
        unsigned long long incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
            if ((int)threadIdx.x >= o) incl += up;
        }
        if (threadIdx.x == 31) s_total = incl;
        unsigned long long excl = incl - sum;
#pragma unroll
        for (int k = 0; k < WARPS; k++) {
            before[threadIdx.x * WARPS + k] = excl;
            excl += v[k];
        }
    }
    __syncthreads();
    // warps are numbered across the CTAs first: a small call spreads over the SMs
    const unsigned long long total = s_total, warps = active_warps(a, total), me = (unsigned long long)(threadIdx.x >> 5) * gridDim.x + blockIdx.x;
    if (me >= warps) return;
    unsigned long long u = me * total / warps;
    const unsigned long long end = (me + 1) * total / warps;
    int lo = 0, hi = 32 * WARPS - 1;   // last run that begins at or before u (runs without steps share their beginning)
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (before[mid] <= u) lo = mid;
        else hi = mid - 1;
    }
    uint32_t b = (uint32_t)lo * run;
    unsigned long long base = before[lo];   // first step of sequence b
    bool first_segment = true;
    while (u < end) {
        const CacheSeq s = cache_seq(a.bt, b);
        const unsigned long long steps_b = seq_steps(a, s, ROWS);
        if (u >= base + steps_b) {
            base += steps_b;
            b++;
            continue;
        }
        const uint32_t steps = item_steps(s);
        while (u < end && u < base + steps_b) {
            const uint64_t item = (u - base) / steps;
            const unsigned long long item0 = base + item * steps;
            const uint32_t tile = (uint32_t)(item / a.cache.kv_heads), h = (uint32_t)(item - (uint64_t)tile * a.cache.kv_heads);
            const uint32_t from = (uint32_t)(u - item0), to = end - item0 < steps ? (uint32_t)(end - item0) : steps;
            const bool whole = from == 0 && to == steps;
            const uint32_t slot = (uint32_t)me * 2 + (first_segment ? 0 : 1);   // a shared item is a warp's first or its last
            if (from == 0 && (threadIdx.x & 31) == 0) {
                // the last warp with a part of the item: the one whose range holds its last step
                const unsigned long long last = ((item0 + steps) * warps + total - 1) / total - 1;
                a.item[((uint64_t)b * a.row_tiles + tile) * a.cache.kv_heads + h] = make_int2((int)slot, (int)last);
            }
            do_segment<D, NT>(a, b, s, h, tile * ROWS, from, to, whole, slot);
            u = item0 + to;
            first_segment = false;
        }
    }
}

// Joins the parts of shared items.  WPR warps share a row (new token and query head): one where there are many rows, eight
// where there are few and a row may have hundreds of parts.
template <int D, int WPR>
__global__ void __launch_bounds__(256)
cache_attention_join_kernel(const __grid_constant__ AttnArgs a, uint32_t rows_per_tile, bool dense)
{
    griddep_launch_dependents();
    griddep_wait();
    constexpr int V = D / 32;   // values per lane
    const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) % WPR;
    const CacheSeq s = cache_seq(a.bt, blockIdx.y);
    const uint32_t i = blockIdx.x * (8 / WPR) + (threadIdx.x >> 5) / WPR;
    if (!s.ok || i >= (uint32_t)s.n * a.q_heads) return;   // (with WPR = 8 the whole CTA)
    const uint32_t t = i / a.q_heads, head = i - t * a.q_heads, h = head / a.group;
    const uint32_t row = t * a.group + (head - h * a.group), tile = row / rows_per_tile, rr = row - tile * rows_per_tile;
    const int2 it = a.item[((uint64_t)blockIdx.y * a.row_tiles + tile) * a.cache.kv_heads + h];
    // Parts are numbered by the warps that made them, two slots each: the first one's part lies in slot it.x, those of the
    // warps behind it in their first slots.  `dense` (the tensor-core form): parts are slots.
    const int first = dense ? it.x : it.x >> 1;
    if (first == it.y) return;   // one warp had it all
    float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
    for (int j = 0; j < V; j++) o[j] = 0.f;
    constexpr int BATCH = WPR == 1 || V > 4 ? 4 : 8;   // parts loaded before the first is used
    for (int k0 = first + w * BATCH; k0 <= it.y; k0 += WPR * BATCH) {
        float2 ml[BATCH];
        float part[BATCH][V];
#pragma unroll
        for (int e = 0; e < BATCH; e++) {
            const int k = k0 + e;
            const uint64_t place = (uint64_t)(dense ? k : (k == first ? it.x : 2 * k)) * rows_per_tile + rr;
            ml[e] = k <= it.y ? a.part_ml[place] : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int j = 0; j < V; j++) part[e][j] = k <= it.y ? a.part_o[place * D + 32 * j + lane] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < BATCH; e++) {
            const float mx = fmaxf(m, ml[e].x), f0 = m == mx ? 1.f : exp2_fast(m - mx), f1 = ml[e].x == mx ? 1.f : exp2_fast(ml[e].x - mx);
            m = mx;
            l = fmaf(f0, l, f1 * ml[e].y);
#pragma unroll
            for (int j = 0; j < V; j++) o[j] = fmaf(f0, o[j], f1 * part[e][j]);
        }
    }
    if (WPR > 1) {
        __shared__ float s_o[WPR][D], s_m[WPR], s_l[WPR];
        if (lane == 0) {
            s_m[w] = m;
            s_l[w] = l;
        }
#pragma unroll
        for (int j = 0; j < V; j++) s_o[w][32 * j + lane] = o[j];
        __syncthreads();
        if (w != 0) return;
#pragma unroll
        for (int k = 1; k < WPR; k++) {
            const float mx = fmaxf(m, s_m[k]), f0 = m == mx ? 1.f : exp2_fast(m - mx), f1 = s_m[k] == mx ? 1.f : exp2_fast(s_m[k] - mx);
            m = mx;
            l = fmaf(f0, l, f1 * s_l[k]);
#pragma unroll
            for (int j = 0; j < V; j++) o[j] = fmaf(f0, o[j], f1 * s_o[k][32 * j + lane]);
        }
    }
    const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
    using T = typename std::conditional<DT == LTQ_F32, float, uint16_t>::type;
    T *p = static_cast<T *>(a.out) + ((uint64_t)s.off * a.q_heads + i) * D;
#pragma unroll
    for (int j = 0; j < V; j++) {
        if constexpr (DT == LTQ_F32) p[32 * j + lane] = o[j] * inv;
        else p[32 * j + lane] = (T)token_bits<DT>(o[j] * inv);
    }
}

// The same for calls of few items and at most a thousand keys or so per CTA: one launch, no workspace.  A cluster of CTAs takes an
// item (row tiles along grid.x, heads grid.y, sequences grid.z), every warp an equal part of its steps; the parts meet in
// shared memory, the CTAs' results through distributed shared memory, each CTA finishing some of the rows.
template <int D, int NT>
__global__ void __launch_bounds__(32 * WARPS, (D * NT * TERMS <= 128 ? 3 : 2))
cache_attention_cluster_kernel(const __grid_constant__ AttnArgs a)
{
    griddep_launch_dependents();
    griddep_wait();
    constexpr uint32_t ROWS = 8 * NT;
    __shared__ __align__(16) float s_o[ROWS][D], s_part[WARPS][ROWS][2];
    __shared__ float s_m[ROWS], s_l[ROWS];
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), size = cluster.num_blocks();
    const uint32_t h = blockIdx.y, b = blockIdx.z, row0 = blockIdx.x / size * ROWS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const CacheSeq s = cache_seq(a.bt, b);
    if (!s.ok && threadIdx.x == 0) atomicCAS(a.bt.refused, 0u, REFUSED_SEQUENCE);
    const uint32_t rows = s.ok ? (uint32_t)s.n * a.group : 0u;
    if (row0 >= rows) return;   // the whole cluster
    const uint32_t steps = seen_steps(a, s, row0, ROWS), parts = size * WARPS, me = rank * WARPS + warp;
    Rows<D, NT> r;
    take_steps<D, NT>(r, a, b, s, h, row0, (uint32_t)((uint64_t)steps * me / parts), (uint32_t)((uint64_t)steps * (me + 1) / parts));
    // the warps' maxima and sums, then their rows one warp after the other into the CTA's
    float l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            l[nt][j] = r.l[nt][j];
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) l[nt][j] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][j], o);
            if (g == 0) {
                s_part[warp][nt * 8 + 2 * c + j][0] = r.m[nt][j];
                s_part[warp][nt * 8 + 2 * c + j][1] = l[nt][j];
            }
        }
    __syncthreads();
    float f[NT][2];   // this warp's weight in the CTA's row
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int rr = nt * 8 + 2 * c + j;
            float m = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) m = fmaxf(m, s_part[w][rr][0]);
#pragma unroll
            for (int w = 0; w < WARPS; w++) sum = fmaf(s_part[w][rr][0] == m ? 1.f : exp2_fast(s_part[w][rr][0] - m), s_part[w][rr][1], sum);
            f[nt][j] = r.m[nt][j] == m ? 1.f : exp2_fast(r.m[nt][j] - m);
            if (warp == 0 && g == 0) {
                s_m[rr] = m;
                s_l[rr] = sum;
            }
        }
    for (int w = 0; w < WARPS; w++) {
        if (warp == w) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float k = f[nt][j] * power2(-exponent_of(r.g[nt][j]));
#pragma unroll
                    for (int i = 0; i < D / 32; i++) {
                        float4 *at = reinterpret_cast<float4 *>(&s_o[nt * 8 + 2 * c + j][Geo<D>::v_dim(i, g)]);
                        float4 v = w == 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : *at;
                        v.x = fmaf(r.o[2 * i][nt][j], k, v.x);
                        v.y = fmaf(r.o[2 * i][nt][j + 2], k, v.y);
                        v.z = fmaf(r.o[2 * i + 1][nt][j], k, v.z);
                        v.w = fmaf(r.o[2 * i + 1][nt][j + 2], k, v.w);
                        *at = v;
                    }
                }
        }
        __syncthreads();
    }
    if (size > 1) cluster.sync();   // every CTA's rows are there
    for (uint32_t k = threadIdx.x; k < ROWS * (D / 4); k += 32 * WARPS) {
        const uint32_t rr = k / (D / 4), d = (k - rr * (D / 4)) * 4, row = row0 + rr;
        if (rr % size != rank || row >= rows) continue;
        float m = -INFINITY, sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t q = 0; q < size; q++) m = fmaxf(m, *cluster.map_shared_rank(&s_m[rr], q));
        for (uint32_t q = 0; q < size; q++) {
            const float mq = *cluster.map_shared_rank(&s_m[rr], q), w = mq == m ? 1.f : exp2_fast(mq - m);
            const float4 v = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(&s_o[rr][d], q));
            sum = fmaf(w, *cluster.map_shared_rank(&s_l[rr], q), sum);
            o.x = fmaf(w, v.x, o.x);
            o.y = fmaf(w, v.y, o.y);
            o.z = fmaf(w, v.z, o.z);
            o.w = fmaf(w, v.w, o.w);
        }
        const uint32_t t = row / a.group;
        const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);   // a row that sees nothing: zeros
        store4<D>(a, ((uint64_t)s.off + t) * a.q_heads + h * a.group + (row - t * a.group), d, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
    if (size > 1) cluster.sync();   // nobody leaves while its shared memory may still be read
}

template <int D>
cudaError_t launch_join(const AttnArgs &a, uint32_t rows_per_tile, bool dense, cudaStream_t stream)
{
    const uint64_t rows = (uint64_t)a.bt.max_new * a.q_heads;   // of one sequence
    count_launch();
    if (rows * a.bt.seqs <= a.few_rows)
        return launch_chained(cache_attention_join_kernel<D, 8>, dim3((unsigned)rows, a.bt.seqs), dim3(256), 0, stream, a, rows_per_tile, dense);
    return launch_chained(cache_attention_join_kernel<D, 1>, dim3((unsigned)((rows + 7) / 8), a.bt.seqs), dim3(256), 0, stream, a, rows_per_tile, dense);
}

template <int D, int NT>
cudaError_t launch_nt(const AttnArgs &a, cudaStream_t stream)
{
    if (a.cluster) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(a.cluster * a.row_tiles, a.cache.kv_heads, a.bt.seqs);
        cfg.blockDim = dim3(32 * WARPS);
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = a.cluster;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = chained_launches_enabled() ? 2 : 1;
        count_launch();
        return cudaLaunchKernelEx(&cfg, cache_attention_cluster_kernel<D, NT>, a);
    }
    cudaError_t e = launch_chained(cache_attention_kernel<D, NT>, dim3(a.ctas), dim3(32 * WARPS), 0, stream, a);
    count_launch();
    if (e != cudaSuccess) return e;
    return launch_join<D>(a, 8 * NT, false, stream);
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

#ifdef LTQ_ATTN_JOIN   // the types that have a tensor-core form
cudaError_t LTQ_ATTN_JOIN(const AttnArgs &a, uint32_t rows_per_tile, cudaStream_t stream)
{
    switch (a.cache.head_dim) {
        case 32: return launch_join<32>(a, rows_per_tile, true, stream);
        case 64: return launch_join<64>(a, rows_per_tile, true, stream);
        case 96: return launch_join<96>(a, rows_per_tile, true, stream);
        case 128: return launch_join<128>(a, rows_per_tile, true, stream);
        case 192: return launch_join<192>(a, rows_per_tile, true, stream);
        case 256: return launch_join<256>(a, rows_per_tile, true, stream);
        default: return cudaErrorInvalidValue;
    }
}
#endif

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
