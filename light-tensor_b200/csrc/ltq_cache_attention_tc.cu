// Attention of many new tokens over the 8-bit cache (prompts and chunks of them) on the 5th-generation tensor cores.
//
// A CTA owns two tiles of 128 rows (new tokens x query heads of one group; one tile for head_dim above 128) of one sequence
// and key/value head and walks the keys in tiles of 64:
//   S [128 x 64]  = Q [128 x D] . K^T        tcgen05.mma kind::f16, both operands in shared memory
//   P             = exp2(S * scales - m)     one thread per row, straight out of tensor memory
//   O [128 x D]  += P [128 x 64] . V         P as the operand in tensor memory, V transposed in shared memory
//
//   softmax      four warps per row tile: thread = row = TMEM lane.  No reduction crosses threads.  The reference maximum m moves
//                only when a score exceeds it by more than 8 (base 2), so that O is hardly ever rescaled.
//   conversion   four warps: codes -> halves, for both row tiles.  A code under 0x64 is the half 1024 + code, minus
//                (1024 + zero point) it is exact.  K is written as rows of keys, V as rows of head dimensions (eight keys'
//                bytes gathered per 16-byte store), both under the 128-byte swizzle the MMA reads; lanes are dealt so that
//                stores spread over the banks.  The next tile's codes are on their way into registers meanwhile.
//   MMA issue    one warp: S of the next tile goes out before O of this one, so that the tensor core works on one row tile while
//                the softmax of the other runs.
// S is double buffered in TMEM and P overwrites it there; K and V have two stages.
//
// Scales: K's block scale multiplies the scores, V's goes into the exponent as log2 of its ratio to a reference (at least twice
// the largest so far, per CTA), the sum of probabilities takes it out again per 16 keys.  q is scaled by a power of two per
// row, so that halves hold it exactly or to 11 bits (half, bfloat16 queries).
//
// Every wait is bounded, see mbar_wait.
#include <cuda_fp16.h>

#include "ltq_cache.cuh"
#include "ltq_ptx.cuh"
#include "ltq_tcgen05.cuh"

namespace ltq {

namespace {

constexpr int TC_ROWS = 128, TC_KEYS = 64;
constexpr float TC_MAX_STEP = 8.f;
constexpr float TC_SMALLEST = 1.17549435e-38f;   // 2^-126
constexpr float TC_MIN_RATIO = 8.6736174e-19f;   // 2^-60: a V scale below the reference by more than this adds nothing

// What the softmax needs of a tile: per 16 keys the K scale, log2 of the V scale's ratio to the reference and its inverse, and
// whether their block does not exist; for the tile the reference and what O so far has to be multiplied with for it.
struct GroupPar {
    float ks, lr, inv;
    uint32_t bad;
};
struct TilePar {
    GroupPar g[4];
    float v_ref, rescale;
    uint32_t any_bad, pad;
};

template <int D>
struct TcGeo {
    static constexpr int RT = D <= 128 ? 2 : 1;                    // row tiles per CTA: TMEM holds O (D columns) and two S (64) of each
    static constexpr int PANELS = (D + 63) / 64;                   // 64 halves = one 128-byte swizzle row
    static constexpr int Q_BYTES = PANELS * TC_ROWS * 128;
    static constexpr int K_BYTES = PANELS * TC_KEYS * 128;
    static constexpr int V_BYTES = D * 128;                        // rows = head dimensions, 64 keys = 128 bytes
    static constexpr int SOFTMAX_WARPS = 4 * RT, MMA_WARP = SOFTMAX_WARPS + 4, THREADS = 32 * (MMA_WARP + 1);
    static constexpr int BARS = 8 + 6 * RT + 1;                    // k_full k_empty v_full v_empty, s_full p_full pv_done per row tile, q_full
    static constexpr size_t SMEM = 1024 + RT * Q_BYTES + 2 * K_BYTES + 2 * V_BYTES + 4 * sizeof(TilePar) + BARS * 8 + 16;
    static __device__ __forceinline__ uint32_t o_col(uint32_t rt) { return rt * 128; }
    static __device__ __forceinline__ uint32_t s_col(uint32_t rt, uint32_t st) { return 256 + rt * 128 + st * TC_KEYS; }
};

__device__ __forceinline__ uint32_t h2sub(uint32_t a, uint32_t b)
{
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t h2pack(float lo, float hi)
{
    const __half2 r = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x)
{
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// kind::f16, D = F32 (1 at bit 4), A = B = F16, both K-major.
__device__ __forceinline__ constexpr uint32_t idesc_f16(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
        "r"(idesc), "r"(accumulate)
        : "memory");
}
// A from tensor memory: 128 lanes x 8 columns of half pairs per 16 keys.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
        "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]), "r"(r[1]),
        "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
        "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int DT>
__device__ __forceinline__ float elem(uint32_t w, int i)   // half i (0, 1) of a word as a float
{
    const uint16_t b = (uint16_t)(i ? w >> 16 : w & 0xFFFF);
    if (DT == LTQ_F16) return __half2float(__ushort_as_half(b));
    return __uint_as_float((uint32_t)b << 16);
}

}  // namespace

// Grid: (kv_heads, sequences, groups of row tiles); those that see most keys come first.
template <int DT, int D>
__global__ void __launch_bounds__(TcGeo<D>::THREADS, 1)
cache_attention_tc_kernel(const __grid_constant__ AttnArgs a)
{
    using G = TcGeo<D>;
    constexpr uint32_t RT = G::RT;
    griddep_launch_dependents();
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), sq = (raw + 1023u) & ~1023u;
    const uint32_t sk = sq + RT * G::Q_BYTES, sv = sk + 2 * G::K_BYTES;
    uint8_t *after = smem_raw + (sv - raw) + 2 * G::V_BYTES;
    TilePar *s_par = reinterpret_cast<TilePar *>(after);     // of four tiles
    uint64_t *bars = reinterpret_cast<uint64_t *>(after + 4 * sizeof(TilePar));
    uint32_t *s_misc = reinterpret_cast<uint32_t *>(bars + G::BARS);   // [0] tmem base, [1] abort flag
    volatile uint32_t *abort_flag = s_misc + 1;
    const uint32_t k_full = smem_u32(bars), k_empty = k_full + 16, v_full = k_full + 32, v_empty = k_full + 48, q_full = k_full + 64;
    const uint32_t s_full = k_full + 72, p_full = s_full + 16 * RT, pv_done = p_full + 16 * RT;   // [row tile][stage]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t *status = a.bt.status;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < 2; i++) {
            mbar_init(k_full + 8 * i, 128);
            mbar_init(k_empty + 8 * i, 1);
            mbar_init(v_full + 8 * i, 128);
            mbar_init(v_empty + 8 * i, 1);
        }
        for (uint32_t i = 0; i < 2 * RT; i++) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 4);
            mbar_init(pv_done + 8 * i, 1);
        }
        mbar_init(q_full, 128 * RT);
        s_misc[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == G::MMA_WARP) {
        tmem_alloc(smem_u32(s_misc), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_wait();
    const uint32_t tmem = s_misc[0];

    const uint32_t h = blockIdx.x, b = blockIdx.y, row0 = (gridDim.z - 1 - blockIdx.z) * (TC_ROWS * RT);
    const CacheSeq s = cache_seq(a.bt, b);
    if (!s.ok && threadIdx.x == 0) atomicCAS(status, 0u, STATUS_BAD_SEQUENCE);
    const uint32_t rows = s.ok ? (uint32_t)s.n * a.group : 0u;
    auto tiles_of = [&](uint32_t rt) -> uint32_t {   // key tiles that row tile rt sees
        const uint32_t first = row0 + rt * TC_ROWS;
        if (first >= rows) return 0u;
        const uint32_t last = first + TC_ROWS < rows ? first + TC_ROWS - 1 : rows - 1;
        const int keys = s.len - s.n + (int)(last / a.group) + 1;
        return keys > 0 ? ((uint32_t)keys + TC_KEYS - 1) / TC_KEYS : 0u;
    };
    const uint32_t tiles0 = tiles_of(0), tiles1 = RT == 2 ? tiles_of(1) : 0u, tiles = tiles0 > tiles1 ? tiles0 : tiles1;
    if (row0 < rows) {
        if (warp < G::SOFTMAX_WARPS) {
            // ---------------- softmax: one row per thread ----------------
            const uint32_t rt = (uint32_t)warp >> 2, mine = rt ? tiles1 : tiles0;
            const uint32_t r = ((uint32_t)warp & 3) * 32 + lane, row = row0 + rt * TC_ROWS + r, t = row / a.group;
            const bool real = row < rows;
            const uint64_t q_row = ((uint64_t)s.off + t) * a.ld_q + (uint64_t)(h * a.group + row - t * a.group) * D;
            const uint16_t *q = static_cast<const uint16_t *>(a.q) + q_row;
            auto eight = [&](int d, uint32_t (&w)[4]) {   // eight neighbouring elements
                if (!real) {
                    w[0] = w[1] = w[2] = w[3] = 0;
                } else if (a.q_vec8) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(q + d));
                    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] = (uint32_t)q[d + 2 * i] | (uint32_t)q[d + 2 * i + 1] << 16;
                }
            };
            float most = 0.f;
            bool finite = true;
#pragma unroll 4
            for (int d = 0; d < D; d += 8) {
                uint32_t w[4];
                eight(d, w);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float v = fabsf(elem<DT>(w[i / 2], i & 1));
                    finite = finite && v < INFINITY;
                    most = fmaxf(most, v);
                }
            }
            int e = 0;   // most * 2^e in [2^10, 2^11)
            if (most > 0.f && finite) {
                e = 10 - ilogbf(most);
                e = e > 100 ? 100 : e;
            }
            const float f = ldexpf(1.f, e);
            const float row_scale = finite ? a.scale_log2 * ldexpf(1.f, -e) : __int_as_float(0x7FC00000);
#pragma unroll 4
            for (int d = 0; d < D; d += 8) {
                uint32_t w[4], p[4];
                eight(d, w);
#pragma unroll
                for (int i = 0; i < 4; i++) p[i] = finite ? h2pack(elem<DT>(w[i], 0) * f, elem<DT>(w[i], 1) * f) : 0u;
                const uint32_t panel = (uint32_t)d / 64, chunk = ((uint32_t)d / 8) & 7;
                sts16(sq + rt * G::Q_BYTES + panel * (TC_ROWS * 128) + r * 128 + ((chunk ^ (r & 7)) << 4), p[0], p[1], p[2], p[3]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(q_full);

            const int pos = real ? s.len - s.n + (int)t : 0x7FFFFFFF;
            const int first_pos = __reduce_min_sync(0xFFFFFFFFu, pos);
            const uint32_t lane_addr = tmem + ((((uint32_t)warp & 3) * 32) << 16), o_addr = lane_addr + G::o_col(rt);
            const uint32_t s_bar = s_full + 16 * rt, p_bar = p_full + 16 * rt, pv_bar = pv_done + 16 * rt;
            float m = -INFINITY, l = 0.f, v_ref = TC_SMALLEST;
            bool ok = true;
            for (uint32_t j = 0; j < mine; j++) {
                const uint32_t st = j & 1, ph = (j >> 1) & 1;
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(s_bar + 8 * st, ph, abort_flag, status, 0xB00u | st));
                if (!ok) break;
                tc_fence_after();
                const uint32_t s_addr = lane_addr + G::s_col(rt, st);
                float x[64];
                auto load_scores = [&]() {
                    uint32_t v0[32], v1[32];
                    tmem_ld32(s_addr, v0);
                    tmem_ld32(s_addr + 32, v1);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        x[i] = __uint_as_float(v0[i]);
                        x[32 + i] = __uint_as_float(v1[i]);
                    }
                };
                load_scores();
                const TilePar &par = s_par[j & 3];
                const int key0 = (int)(j * TC_KEYS);
                const bool masked = par.any_bad || key0 + TC_KEYS - 1 > first_pos;
                v_ref = par.v_ref;
                float alpha = par.rescale;
                // x = score - m + log2(ratio); the largest without the last term
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float ks = row_scale * par.g[k].ks, lr = par.g[k].lr, c = lr - m;
                    float g0 = -INFINITY, g1 = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 16; i++) x[16 * k + i] = fmaf(x[16 * k + i], ks, c);
                    if (masked) {
                        const int see = par.g[k].bad ? -1 : pos - key0 - 16 * k;   // the last key of these that the row sees
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (i > see) x[16 * k + i] = -INFINITY;
                    }
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        g0 = fmaxf(g0, x[16 * k + i]);
                        g1 = fmaxf(g1, x[16 * k + i + 1]);
                    }
                    top = fmaxf(top, fmaxf(g0, g1) - (lr == lr ? lr : 0.f));
                }
                if (__any_sync(0xFFFFFFFFu, top > TC_MAX_STEP)) {
                    // the scores again (they are still in TMEM; with m at -inf the difference says nothing), and a new reference
                    load_scores();
                    float best = -INFINITY;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float ks = row_scale * par.g[k].ks;
                        const int see = par.g[k].bad ? -1 : pos - key0 - 16 * k;
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            x[16 * k + i] = i > see ? -INFINITY : x[16 * k + i] * ks;
                            best = fmaxf(best, x[16 * k + i]);
                        }
                    }
                    const float mx = fmaxf(m, best), down = m == mx ? 1.f : ex2(m - mx), ref = mx == -INFINITY ? 0.f : mx;
                    m = mx;
                    l *= down;
                    alpha *= down;
#pragma unroll
                    for (int i = 0; i < 64; i++) x[i] = x[i] == -INFINITY ? -INFINITY : x[i] + (par.g[i / 16].lr - ref);   // (lr may be NaN)
                }
                if (j > 0 && __any_sync(0xFFFFFFFFu, alpha != 1.f)) {
                    // O so far times alpha: once the MMA that last added to it is done
                    const uint32_t pj = j - 1;
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait(pv_bar + 8 * (pj & 1), (pj >> 1) & 1, abort_flag, status, 0xB10u | (pj & 1)));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int d = 0; d < D; d += 16) {
                        uint32_t o[16];
                        tmem_ld16(o_addr + d, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st16(o_addr + d, o);
                    }
                }
                uint32_t p[32];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    float sum = 0.f, sum1 = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float y0 = ex2(x[16 * k + i]), y1 = ex2(x[16 * k + i + 1]);
                        sum += y0;
                        sum1 += y1;
                        p[8 * k + i / 2] = h2pack(y0, y1);
                    }
                    l = fmaf(sum + sum1, par.g[k].inv, l);
                }
                tmem_st32(s_addr, p);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_bar + 8 * st);
            }
            if (ok && mine > 0) {
                const uint32_t pj = mine - 1;
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(pv_bar + 8 * (pj & 1), (pj >> 1) & 1, abort_flag, status, 0xB20u | (pj & 1)));
                tc_fence_after();
            }
            if (ok) {
                const float inv = l == 0.f ? 0.f : __fdiv_rn(v_ref, l);   // a row that sees nothing: zeros
                uint16_t *dst = static_cast<uint16_t *>(a.out) + (((uint64_t)s.off + t) * a.q_heads + h * a.group + (row - t * a.group)) * D;
#pragma unroll 1
                for (int d = 0; d < D; d += 32) {
                    uint32_t o[32];
                    if (mine > 0) {
                        tmem_ld32(o_addr + d, o);
                        tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = 0;
                    }
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) w[i] = token_bits2<DT>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
                    if (real) {
                        if (a.out_vec8) {
#pragma unroll
                            for (int i = 0; i < 4; i++) reinterpret_cast<uint4 *>(dst + d)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i++) dst[d + i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
                        }
                    }
                }
            }
        } else if (warp < G::MMA_WARP) {
            // ---------------- conversion ----------------
            const int tid = threadIdx.x - 32 * G::SOFTMAX_WARPS;
            const int32_t *table = a.bt.table + (uint64_t)b * a.bt.table_width;
            const uint32_t in_block = (1u << a.bt.log2_bt) - 1;
            const uint32_t last_key = tiles * TC_KEYS - 1 < (uint32_t)s.len - 1 ? tiles * TC_KEYS - 1 : (uint32_t)s.len - 1;
            // K: lanes 0..7 of a group take eight keys, so that their stores meet eight different banks; V likewise eight groups of keys
            constexpr int KC = D / 16, K_UNITS = TC_KEYS * KC, K_PER = (K_UNITS + 127) / 128;   // 16-byte pieces of a tile's K
            constexpr int V_UNITS = 8 * (D / 8), V_PER = (V_UNITS + 127) / 128;                   // 8 keys x 8 head dimensions of its V
            struct Codes {
                uint4 k[K_PER];
                uint2 v[V_PER][8];
                uint32_t kz[K_PER], vz[V_PER];
            };
            // the slot (block and head) that holds a key; keys behind the sequence's last read its block (masked later)
            auto page_of = [&](uint32_t key) { return __ldg(table + ((key < last_key ? key : last_key) >> a.bt.log2_bt)); };
            auto slot_of = [&](int32_t page) { return (uint64_t)((uint32_t)page < a.cache.blocks ? (uint32_t)page : 0u) * a.cache.kv_heads + h; };
            auto k_key = [&](int i) { return (uint32_t)(((i * 128 + tid) & 7) | ((i * 128 + tid) / (8 * KC)) << 3); };
            auto k_chunk = [&](int i) { return (uint32_t)((i * 128 + tid) / 8 % KC); };
            auto v_group = [&](int i) { return (uint32_t)((i * 128 + tid) & 7); };
            auto v_dim = [&](int i) { return (uint32_t)((i * 128 + tid) / 8 * 8); };
            int32_t k_page[K_PER], v_page[V_PER], g_page = 0;   // block ids of the tile to be loaded next
            auto pages = [&](uint32_t j) {
#pragma unroll
                for (int i = 0; i < K_PER; i++) k_page[i] = page_of(j * TC_KEYS + k_key(i));
#pragma unroll
                for (int i = 0; i < V_PER; i++) v_page[i] = page_of(j * TC_KEYS + v_group(i) * 8);
                if (tid < 32) g_page = page_of(j * TC_KEYS + (tid & 3) * 16);
            };
            auto load = [&](Codes &c, uint32_t j) {
#pragma unroll
                for (int i = 0; i < K_PER; i++) {
                    if (K_UNITS % 128 == 0 || i * 128 + tid < K_UNITS) {
                        const uint64_t slot = slot_of(k_page[i]);
                        const uint32_t key = j * TC_KEYS + k_key(i);
                        c.k[i] = __ldg(reinterpret_cast<const uint4 *>(a.cache.k_dev + ((slot << a.bt.log2_bt) + (key & in_block)) * D + k_chunk(i) * 16));
                        c.kz[i] = __ldg(&a.cache.k_qp_dev[slot].zero_point);
                    }
                }
#pragma unroll
                for (int i = 0; i < V_PER; i++) {
                    if (V_UNITS % 128 == 0 || i * 128 + tid < V_UNITS) {
                        const uint64_t slot = slot_of(v_page[i]);
                        const uint32_t key = j * TC_KEYS + v_group(i) * 8;
                        const uint8_t *p = a.cache.v_dev + ((slot << a.bt.log2_bt) + (key & in_block)) * D + v_dim(i);
#pragma unroll
                        for (int k = 0; k < 8; k++) c.v[i][k] = __ldg(reinterpret_cast<const uint2 *>(p + k * D));
                        c.vz[i] = __ldg(&a.cache.v_qp_dev[slot].zero_point);
                    }
                }
            };
            float g_ks = 0.f, g_vs = 0.f, v_ref = TC_SMALLEST;   // first converting warp: lane i & 3 looks after group i
            bool g_bad = false;
            auto load_params = [&]() {
                if (tid < 32) {
                    const uint64_t slot = slot_of(g_page);
                    g_bad = (uint32_t)g_page >= a.cache.blocks;
                    g_ks = __ldg(&a.cache.k_qp_dev[slot].scale);
                    g_vs = __ldg(&a.cache.v_qp_dev[slot].scale);
                    if (g_bad && tid < 4) atomicCAS(status, 0u, STATUS_BAD_BLOCK);
                }
            };
            const uint32_t magic = 0x64646464u;
            // tile j from `cur`; the codes of tile j + 1 go into `nxt` meanwhile
            auto convert = [&](uint32_t j, Codes &cur, Codes &nxt) -> bool {
                const uint32_t st = j & 1;
                if (tid < 32) {   // four tiles deep: this place was last read for tile j - 4
                    float top = g_vs;
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));   // (NaN is passed over)
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                    float rescale = 1.f;
                    if (top > v_ref) {
                        const float next = top < 1e38f ? 2.f * top : top;
                        rescale = v_ref * __fdividef(1.f, next);
                        v_ref = next;
                    }
                    const float ratio = __fdiv_rn(g_vs, v_ref), x = fmaxf(ratio, TC_MIN_RATIO);
                    const bool nan = ratio != ratio;
                    const uint32_t any = __ballot_sync(0xFFFFFFFFu, g_bad);
                    TilePar &p = s_par[j & 3];
                    if (tid < 4) p.g[tid] = GroupPar{g_ks, nan ? ratio : lg2(x), nan ? 1.f : __fdividef(1.f, x), g_bad ? 1u : 0u};
                    if (tid == 0) {
                        p.v_ref = v_ref;
                        p.rescale = rescale;
                        p.any_bad = any;
                    }
                }
                if (j + 1 < tiles) {
                    load_params();
                    load(nxt, j + 1);
                    if (j + 2 < tiles) pages(j + 2);
                }
                if (j >= 2 && !mbar_wait(k_empty + 8 * st, ((j - 2) >> 1) & 1, abort_flag, status, 0xB30u | st)) return false;
#pragma unroll
                for (int i = 0; i < K_PER; i++) {
                    if (K_UNITS % 128 == 0 || i * 128 + tid < K_UNITS) {
                        const uint32_t key = k_key(i), ch = k_chunk(i), z = 0x64006400u + cur.kz[i] * 0x10001u;
                        const uint32_t w[4] = {cur.k[i].x, cur.k[i].y, cur.k[i].z, cur.k[i].w};
                        uint32_t x[8];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            x[2 * k] = h2sub(__byte_perm(w[k], magic, 0x4140), z);
                            x[2 * k + 1] = h2sub(__byte_perm(w[k], magic, 0x4342), z);
                        }
                        const uint32_t row = sk + st * G::K_BYTES + (ch / 4) * (TC_KEYS * 128) + key * 128, c0 = (ch & 3) * 2;
                        sts16(row + ((c0 ^ (key & 7)) << 4), x[0], x[1], x[2], x[3]);
                        sts16(row + (((c0 + 1) ^ (key & 7)) << 4), x[4], x[5], x[6], x[7]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(k_full + 8 * st);
                if (j >= 2 && !mbar_wait(v_empty + 8 * st, ((j - 2) >> 1) & 1, abort_flag, status, 0xB40u | st)) return false;
#pragma unroll
                for (int i = 0; i < V_PER; i++) {
                    if (V_UNITS % 128 == 0 || i * 128 + tid < V_UNITS) {
                        const uint32_t g = v_group(i), d0 = v_dim(i), z = 0x64006400u + cur.vz[i] * 0x10001u;
#pragma unroll
                        for (int half = 0; half < 2; half++) {   // head dimensions d0 + 4 * half + 0..3
                            uint32_t lo[4], hi[4];                 // key pairs 2k, 2k+1: {d, d+1} and {d+2, d+3} interleaved
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const uint32_t u = half ? cur.v[i][2 * k].y : cur.v[i][2 * k].x, v = half ? cur.v[i][2 * k + 1].y : cur.v[i][2 * k + 1].x;
                                lo[k] = __byte_perm(u, v, 0x5140);
                                hi[k] = __byte_perm(u, v, 0x7362);
                            }
#pragma unroll
                            for (int d = 0; d < 4; d++) {
                                uint32_t x[4];
#pragma unroll
                                for (int k = 0; k < 4; k++) x[k] = h2sub(__byte_perm(d < 2 ? lo[k] : hi[k], magic, d & 1 ? 0x4342 : 0x4140), z);
                                const uint32_t dd = d0 + 4 * half + d;
                                sts16(sv + st * G::V_BYTES + dd * 128 + ((g ^ (dd & 7)) << 4), x[0], x[1], x[2], x[3]);
                            }
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(v_full + 8 * st);
                return true;
            };
            Codes even, odd;
            if (tiles > 0) {
                pages(0);
                load_params();
                load(even, 0);
                if (tiles > 1) pages(1);
            }
            for (uint32_t j = 0; j < tiles; j += 2) {
                if (!convert(j, even, odd)) break;
                if (j + 1 >= tiles || !convert(j + 1, odd, even)) break;
            }
        } else {
            // ---------------- MMA issue: the whole warp runs the loop, one elected lane issues ----------------
            constexpr uint32_t id_qk = idesc_f16(TC_ROWS, TC_KEYS), id_pv = idesc_f16(TC_ROWS, D);
            auto wait = [&](uint32_t bar, uint32_t phase, uint32_t code) {
                return __all_sync(0xFFFFFFFFu, mbar_wait(bar, phase, abort_flag, status, code));
            };
            bool ok = tiles > 0 && wait(q_full, 0, 0xB50u);
            for (uint32_t j = 0; ok && j <= tiles; j++) {
                if (j < tiles) {
                    const uint32_t st = j & 1, ph = (j >> 1) & 1;
                    ok = wait(k_full + 8 * st, ph, 0xB60u | st);
                    const uint64_t kd = make_smem_desc(sk + st * G::K_BYTES);
                    for (uint32_t rt = 0; ok && rt < RT; rt++) {
                        if (j >= (rt ? tiles1 : tiles0)) continue;
                        // this S buffer holds P of tile j - 2 until the MMA that reads it is done
                        if (j >= 2) ok = wait(pv_done + 16 * rt + 8 * st, ((j - 2) >> 1) & 1, 0xB70u | st);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t qd = make_smem_desc(sq + rt * G::Q_BYTES);
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < D / 16; k++)
                                mma_ss(tmem + G::s_col(rt, st), qd + (uint64_t)((k / 4) * (TC_ROWS * 128 / 16) + 2 * (k & 3)),
                                       kd + (uint64_t)((k / 4) * (TC_KEYS * 128 / 16) + 2 * (k & 3)), id_qk, k != 0);
                            umma_commit(s_full + 16 * rt + 8 * st);
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    if (elect_one()) umma_commit(k_empty + 8 * st);
                    __syncwarp();
                }
                if (j >= 1) {
                    const uint32_t p = j - 1, st = p & 1, ph = (p >> 1) & 1;
                    ok = wait(v_full + 8 * st, ph, 0xB80u | st);
                    const uint64_t vd = make_smem_desc(sv + st * G::V_BYTES);
                    for (uint32_t rt = 0; ok && rt < RT; rt++) {
                        if (p >= (rt ? tiles1 : tiles0)) continue;
                        ok = wait(p_full + 16 * rt + 8 * st, ph, 0xB90u | st);
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < TC_KEYS / 16; k++)
                                mma_ts(tmem + G::o_col(rt), tmem + G::s_col(rt, st) + 8 * k, vd + 2u * k, id_pv, p != 0 || k != 0);
                            umma_commit(pv_done + 16 * rt + 8 * st);
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    if (elect_one()) umma_commit(v_empty + 8 * st);
                    __syncwarp();
                }
            }
        }
    }
    // Teardown: nobody leaves before every role is done with TMEM and shared memory.
    tc_fence_before();
    __syncthreads();
    if (warp == G::MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

namespace {

template <int DT, int D>
cudaError_t launch_tc(const AttnArgs &a, cudaStream_t stream)
{
    static bool attr_done[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!attr_done[dev]) {
        e = cudaFuncSetAttribute(cache_attention_tc_kernel<DT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)TcGeo<D>::SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(cache_attention_tc_kernel<DT, D>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return e;
        attr_done[dev] = true;
    }
    constexpr uint32_t PER = TC_ROWS * TcGeo<D>::RT;
    const uint32_t tiles = (a.bt.max_new * a.group + PER - 1) / PER;
    count_launch();
    return launch_chained(cache_attention_tc_kernel<DT, D>, dim3(a.cache.kv_heads, a.bt.seqs, tiles), dim3(TcGeo<D>::THREADS), TcGeo<D>::SMEM, stream, a);
}

template <int DT>
cudaError_t launch_tc_d(const AttnArgs &a, cudaStream_t stream)
{
    switch (a.cache.head_dim) {
        case 32: return launch_tc<DT, 32>(a, stream);
        case 64: return launch_tc<DT, 64>(a, stream);
        case 96: return launch_tc<DT, 96>(a, stream);
        case 128: return launch_tc<DT, 128>(a, stream);
        case 192: return launch_tc<DT, 192>(a, stream);
        case 256: return launch_tc<DT, 256>(a, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace

cudaError_t launch_attention_tc(const AttnArgs &a, int dtype, cudaStream_t stream)
{
    return dtype == LTQ_F16 ? launch_tc_d<LTQ_F16>(a, stream) : launch_tc_d<LTQ_BF16>(a, stream);
}

}  // namespace ltq
