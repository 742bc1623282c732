// Attention of many new tokens over the 8-bit cache (prompts and chunks of them) on the 5th-generation tensor cores.
//
// A CTA owns two tiles of 128 rows (new tokens x query heads of one group) of one sequence and key/value head and walks the
// keys in tiles of 64 (head_dim above 128: one row tile; tensor memory holds O and two S of every row):
//   S [128 x keys]  = Q [128 x D] . K^T        tcgen05.mma kind::f16, both operands in shared memory
//   P               = exp2(S * scales - m)     one thread per row, straight out of tensor memory
//   O [128 x D]    += P [128 x keys] . V       P as the operand in tensor memory (over S), V transposed in shared memory
//
//   softmax      four warps per row tile: thread = row = TMEM lane.  No reduction crosses threads.  The reference maximum m moves
//                only when a tile's probabilities add up to more than 2^12, so that O is hardly ever rescaled and no maximum is
//                taken on the way; P waits in registers until that is known.
//   conversion   four warps for K, four for V: codes -> halves, for both row tiles.  K's codes become subnormal halves, code * 2^-24, by
//                a byte permute alone, their zero points come off the scores (times the sum of q).  V's get 0x64 above them,
//                the half 1024 + code, minus (1024 + zero point), exact.  K is written as rows of keys, V as rows of head dimensions
//                (eight keys' bytes gathered per 16-byte store), both under the 128-byte swizzle the MMA reads; lanes are
//                dealt so that stores spread over the banks.  The next half tile's codes are on their way into registers meanwhile.
//   MMA issue    one warp per row tile, so that each goes its own way: while one row tile is in its softmax, the tensor core has
//                the other's products.
// S has two buffers, so that the next tile's is there when a softmax is done; P overwrites it.  (Measured on 2 x 1500 new tokens
// behind up to 4500, 32 query and 8 key/value heads of 128: one warp issuing for both row tiles was busy 2300 of 3250 cycles a
// tile, 372 us; tiles of 128 keys with one S buffer leave the softmax waiting for the two products in between, 474 us.)
// The warps' registers are divided by need (setmaxnreg).
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

constexpr int TC_ROWS = 128;
constexpr float TC_MAX_SUM = 4096.f;
constexpr float TC_SMALLEST = 1.17549435e-38f;   // 2^-126
constexpr float TC_MIN_RATIO = 8.6736174e-19f;   // 2^-60: a V scale below the reference by more than this adds nothing
constexpr float TC_CODE = 16777216.f;            // 2^24: a K code's half is the code over this

// What the softmax needs of 16 keys: K scale times 2^24, K scale times zero point, log2 of the V scale's ratio to the reference and
// the ratio's inverse.
struct GroupPar {
    float ks, kzs, lr, inv;
};

template <int D>
struct TcGeo {
    static constexpr int RT = D <= 128 ? 2 : 1;                    // row tiles per CTA
    static constexpr int KEYS = 64, GROUPS = KEYS / 16;
    static constexpr int PARTS = RT == 2 ? 1 : 2, PART = KEYS / PARTS;   // a tile is converted in so many parts
    static constexpr int SB = 2;                                   // S buffers per row tile
    static constexpr int PANELS = (D + 63) / 64;                   // 64 halves = one 128-byte swizzle row
    static constexpr int Q_BYTES = PANELS * TC_ROWS * 128;
    static constexpr int K_BYTES = PANELS * KEYS * 128;
    static constexpr int V_BYTES = D * 128;                        // rows = head dimensions, 64 keys = 128 bytes
    static constexpr int THREADS = 128 * (RT + 3);                 // warpgroups: softmax per row tile, K, V, MMA issue
    // Registers per thread: as launched (640 or 512 threads), and after setmaxnreg, which may only raise with .inc, lower with .dec,
    // and hands out no more than the block was launched with.
    static constexpr int REGS = RT == 2 ? 96 : 128;
    static constexpr int REGS_SOFTMAX = RT == 2 ? 136 : 200, REGS_CONVERT = RT == 2 ? 80 : 128, REGS_MMA = RT == 2 ? 48 : 56;
    static_assert(RT * REGS_SOFTMAX + 2 * REGS_CONVERT + REGS_MMA == (RT + 3) * REGS, "register shares");
    static_assert(REGS_SOFTMAX >= REGS && REGS_CONVERT <= REGS && REGS_MMA <= REGS, "register shares");
    static constexpr int BARS = 8 + RT * (2 * SB + SB) + 1;        // k_full k_empty v_full v_empty; s_full p_full pv_done per row tile; q_full
    struct TilePar {
        GroupPar g[GROUPS];
        float v_ref, rescale;   // the reference, and what O so far has to be multiplied with for it
        uint32_t bad, pad;      // bit i: group i's block does not exist
    };
    static constexpr size_t SMEM = 1024 + RT * Q_BYTES + 2 * K_BYTES + 2 * V_BYTES + 8 * sizeof(TilePar) + BARS * 8 + 16;
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static __device__ __forceinline__ uint32_t o_col(uint32_t rt) { return rt * 128; }
    static __device__ __forceinline__ uint32_t s_col(uint32_t rt, uint32_t sb) { return 256 + rt * 128 + sb * 64; }
};

// Two floats at a time.
__device__ __forceinline__ uint64_t pair(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <int N>
__device__ __forceinline__ void regs_up()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

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

// Grid: (kv_heads * splits, sequences, groups of row tiles); those that see most keys come first.  Where the groups do not fill
// the device, `splits` CTAs share one's keys and leave their parts in the workspace for the join kernel.
template <int DT, int D>
__global__ void __launch_bounds__(TcGeo<D>::THREADS, 1)
cache_attention_tc_kernel(const __grid_constant__ AttnArgs a)
{
    using G = TcGeo<D>;
    using TilePar = typename G::TilePar;
    constexpr uint32_t RT = G::RT, SB = G::SB;
    griddep_launch_dependents();
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), sq = (raw + 1023u) & ~1023u;
    const uint32_t sk = sq + RT * G::Q_BYTES, sv = sk + 2 * G::K_BYTES;
    uint8_t *after = smem_raw + (sv - raw) + 2 * G::V_BYTES;
    TilePar *s_par = reinterpret_cast<TilePar *>(after);     // of eight tiles
    uint64_t *bars = reinterpret_cast<uint64_t *>(after + 8 * sizeof(TilePar));
    uint32_t *s_misc = reinterpret_cast<uint32_t *>(bars + G::BARS);   // [0] tmem base, [1] abort flag
    volatile uint32_t *abort_flag = s_misc + 1;
    const uint32_t k_full = smem_u32(bars), k_empty = k_full + 16, v_full = k_full + 32, v_empty = k_full + 48, q_full = k_full + 64;
    const uint32_t s_full = k_full + 72, p_full = s_full + 8 * SB * RT, pv_done = p_full + 8 * SB * RT;   // [row tile][S buffer]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t wg = (uint32_t)warp >> 2;
    uint32_t *status = a.bt.status;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < 2; i++) {
            mbar_init(k_full + 8 * i, 128);
            mbar_init(k_empty + 8 * i, RT);
            mbar_init(v_full + 8 * i, 128);
            mbar_init(v_empty + 8 * i, RT);
        }
        for (uint32_t i = 0; i < SB * RT; i++) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 4);
            mbar_init(pv_done + 8 * i, 1);
        }
        mbar_init(q_full, 128 * RT);
        s_misc[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 0) {
        tmem_alloc(smem_u32(s_misc), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_wait();
    const uint32_t tmem = s_misc[0];

    const uint32_t split = blockIdx.x / a.cache.kv_heads, h = blockIdx.x - split * a.cache.kv_heads, b = blockIdx.y;
    const uint32_t group = gridDim.z - 1 - blockIdx.z, row0 = group * (TC_ROWS * RT);
    const CacheSeq s = cache_seq(a.bt, b);
    if (!s.ok && threadIdx.x == 0) atomicCAS(status, 0u, STATUS_BAD_SEQUENCE);
    const uint32_t rows = s.ok ? (uint32_t)s.n * a.group : 0u;
    auto tiles_of = [&](uint32_t rt) -> uint32_t {   // key tiles that row tile rt sees
        const uint32_t first = row0 + rt * TC_ROWS;
        if (first >= rows) return 0u;
        const uint32_t last = first + TC_ROWS < rows ? first + TC_ROWS - 1 : rows - 1;
        const int keys = s.len - s.n + (int)(last / a.group) + 1;
        return keys > 0 ? ((uint32_t)keys + G::KEYS - 1) / G::KEYS : 0u;
    };
    const uint32_t all0 = tiles_of(0), all1 = RT == 2 ? tiles_of(RT - 1) : 0u, all = all0 > all1 ? all0 : all1;
    // this CTA's tiles: [tile0, tile0 + tiles), of which the row tiles see the first tiles0 and tiles1
    const uint32_t tile0 = (uint32_t)((uint64_t)all * split / a.splits), tiles = (uint32_t)((uint64_t)all * (split + 1) / a.splits) - tile0;
    auto part_of = [&](uint32_t n) { return n <= tile0 ? 0u : (n - tile0 < tiles ? n - tile0 : tiles); };
    const uint32_t tiles0 = part_of(all0), tiles1 = part_of(all1);
    const uint32_t place = ((b * gridDim.z + group) * a.cache.kv_heads + h) * a.splits;   // workspace slot of split 0
    if (a.splits > 1 && split == 0 && row0 < rows && threadIdx.x == 0)
        a.item[((uint64_t)b * gridDim.z + group) * a.cache.kv_heads + h] = make_int2((int)place, (int)(place + a.splits - 1));

    if (wg < RT) {
        // ---------------- softmax: one row per thread ----------------
        regs_up<G::REGS_SOFTMAX>();
        const uint32_t rt = wg, mine = rt ? tiles1 : tiles0;
        const uint32_t r = ((uint32_t)warp & 3) * 32 + lane, row = row0 + rt * TC_ROWS + r, t = row / a.group;
        const bool real = row < rows;
        const uint16_t *q = static_cast<const uint16_t *>(a.q) + ((uint64_t)s.off + t) * a.ld_q + (uint64_t)(h * a.group + row - t * a.group) * D;
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
        uint32_t qw[D / 8][4];   // the whole row: one memory latency
#pragma unroll
        for (int d = 0; d < D / 8; d++) eight(8 * d, qw[d]);
        float most = 0.f;
        bool finite = true;
#pragma unroll
        for (int d = 0; d < D / 8; d++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = fabsf(elem<DT>(qw[d][i / 2], i & 1));
                finite = finite && v < INFINITY;
                most = fmaxf(most, v);
            }
        int e = 0;   // most * 2^e in [2^10, 2^11)
        if (most > 0.f && finite) {
            e = 10 - ilogbf(most);
            e = e > 100 ? 100 : e;
        }
        const float f = ldexpf(1.f, e);
        const float row_scale = finite ? a.scale_log2 * ldexpf(1.f, -e) : __int_as_float(0x7FC00000);
        float q_sum = 0.f;
#pragma unroll
        for (int d = 0; d < D / 8; d++) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                w[i] = finite ? h2pack(elem<DT>(qw[d][i], 0) * f, elem<DT>(qw[d][i], 1) * f) : 0u;
                const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                q_sum += x.x + x.y;
            }
            sts16(sq + rt * G::Q_BYTES + (d / 8) * (TC_ROWS * 128) + r * 128 + (((d & 7) ^ (r & 7)) << 4), w[0], w[1], w[2], w[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(q_full);

        const float zero_scale = row_scale * q_sum;
        const int pos = real ? s.len - s.n + (int)t : 0x7FFFFFFF;
        const int first_pos = __reduce_min_sync(0xFFFFFFFFu, pos);
        const uint32_t lane_addr = tmem + ((((uint32_t)warp & 3) * 32) << 16), o_addr = lane_addr + G::o_col(rt);
        const uint32_t s_bar = s_full + 8 * SB * rt, p_bar = p_full + 8 * SB * rt, pv_bar = pv_done + 8 * SB * rt;
        float m = -INFINITY, l = 0.f, v_ref = TC_SMALLEST;
        bool ok = true;
        for (uint32_t j = 0; j < mine; j++) {
            const uint32_t sb = j % SB, ph = (j / SB) & 1;
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(s_bar + 8 * sb, ph, abort_flag, status, 0xB00u | sb));
            if (!ok) break;
            tc_fence_after();
            const uint32_t s_addr = lane_addr + G::s_col(rt, sb);
            const TilePar &par = s_par[j & 7];
            uint32_t x[2][32];
            auto load_scores = [&]() {
                tmem_ld32(s_addr, x[0]);
                tmem_ld32(s_addr + 32, x[1]);
            };
            load_scores();   // (the tile's parameters are read while they are on their way)
            GroupPar g[G::GROUPS];
#pragma unroll
            for (int k = 0; k < G::GROUPS; k++) g[k] = par.g[k];
            const int key0 = (int)((tile0 + j) * G::KEYS);
            const uint32_t bad = par.bad;
            const bool masked = bad || key0 + G::KEYS - 1 > first_pos;
            v_ref = par.v_ref;
            float alpha = par.rescale, sum = 0.f;
            uint32_t p[G::KEYS / 2];
            // P of the tile under the reference `ref`, and the sum of its probabilities
            auto probabilities = [&](float ref) {
                tmem_ld_wait();
                uint64_t add[G::GROUPS];
#pragma unroll
                for (int k = 0; k < G::GROUPS; k++) {
                    const float ks = row_scale * g[k].ks, base = g[k].lr - fmaf(zero_scale, g[k].kzs, ref);
                    const uint64_t ks2 = pair(ks, ks), base2 = pair(base, base);
                    float2 y[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int c = 16 * k + 2 * i;
                        y[i] = unpair(fma2(pair(__uint_as_float(x[c / 32][c % 32]), __uint_as_float(x[c / 32][c % 32 + 1])), ks2, base2));
                    }
                    if (masked) {
                        const int see = bad >> k & 1 ? -1 : pos - key0 - 16 * k;   // the last key of these that the row sees
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            if (2 * i > see) y[i].x = -INFINITY;
                            if (2 * i + 1 > see) y[i].y = -INFINITY;
                        }
                    }
                    add[k] = 0;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        y[i].x = ex2(y[i].x);
                        y[i].y = ex2(y[i].y);
                        add[k] = i == 0 ? pair(y[i].x, y[i].y) : add2(add[k], pair(y[i].x, y[i].y));
                        p[8 * k + i] = h2pack(y[i].x, y[i].y);
                    }
                }
                sum = 0.f;
#pragma unroll
                for (int k = 0; k < G::GROUPS; k++) {
                    const float2 s2 = unpair(add[k]);
                    sum = fmaf(s2.x + s2.y, g[k].inv, sum);
                }
            };
            probabilities(m);   // (with m at -inf everything visible is inf, and so is the sum)
            if (__any_sync(0xFFFFFFFFu, sum > TC_MAX_SUM)) {
                load_scores();
                tmem_ld_wait();
                float best = -INFINITY;
#pragma unroll
                for (int k = 0; k < G::GROUPS; k++) {
                    const float ks = row_scale * g[k].ks, base = -zero_scale * g[k].kzs;
                    const int see = bad >> k & 1 ? -1 : pos - key0 - 16 * k;
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int c = 16 * k + i;
                        best = i > see ? best : fmaxf(best, fmaf(__uint_as_float(x[c / 32][c % 32]), ks, base));
                    }
                }
                const float mx = fmaxf(m, best), down = m == mx ? 1.f : ex2(m - mx);
                m = mx;
                l *= down;
                alpha *= down;
                probabilities(m == -INFINITY ? 0.f : m);
            }
            l += sum;
            if (j > 0 && __any_sync(0xFFFFFFFFu, alpha != 1.f)) {
                // O so far times alpha: once the MMA that last added to it is done
                const uint32_t pj = j - 1;
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(pv_bar + 8 * (pj % SB), (pj / SB) & 1, abort_flag, status, 0xB10u | (pj % SB)));
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
            tmem_st32(s_addr, p);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_bar + 8 * sb);
        }
        if (ok && mine > 0) {
            const uint32_t pj = mine - 1;
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(pv_bar + 8 * (pj % SB), (pj / SB) & 1, abort_flag, status, 0xB20u | (pj % SB)));
            tc_fence_after();
        }
        if (ok && a.splits > 1) {
            const uint64_t at = (uint64_t)(place + split) * (TC_ROWS * RT) + rt * TC_ROWS + r;
            if (real) a.part_ml[at] = make_float2(m, l);
            float4 *dst = reinterpret_cast<float4 *>(a.part_o + at * D);
#pragma unroll 1
            for (int d = 0; d < D; d += 16) {
                uint32_t o[16];
                if (mine > 0) {
                    tmem_ld16(o_addr + d, o);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (real)
                        dst[d / 4 + i] = mine > 0 ? make_float4(__uint_as_float(o[4 * i]) * v_ref, __uint_as_float(o[4 * i + 1]) * v_ref,
                                                                __uint_as_float(o[4 * i + 2]) * v_ref, __uint_as_float(o[4 * i + 3]) * v_ref)
                                                  : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        } else if (ok) {
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
    } else if (wg < RT + 2) {
        // ---------------- conversion ----------------
        if constexpr (G::REGS_CONVERT < G::REGS) regs_down<G::REGS_CONVERT>();
        const int tid = threadIdx.x & 127;
        const int32_t *table = a.bt.table + (uint64_t)b * a.bt.table_width;
        const uint32_t in_block = (1u << a.bt.log2_bt) - 1, parts = G::PARTS * tiles;
        const uint32_t begin = tile0 * G::KEYS, end = (tile0 + tiles) * G::KEYS, last_key = end < (uint32_t)s.len ? end - 1 : (uint32_t)s.len - 1;
        // the block that holds a key; keys behind the sequence's last read its block (masked later)
        auto page_of = [&](uint32_t key) { return __ldg(table + ((key < last_key ? key : last_key) >> a.bt.log2_bt)); };
        auto slot_of = [&](int32_t page) { return (uint64_t)((uint32_t)page < a.cache.blocks ? (uint32_t)page : 0u) * a.cache.kv_heads + h; };
        if (wg == RT) {
            // K: 16-byte pieces; lanes 0..7 of a group take eight keys, so that their stores meet eight different banks
            constexpr int KC = D / 16, PER = G::PART * KC / 128;
            static_assert(PER * 128 == G::PART * KC, "pieces");
            auto key_of = [&](int i) { return (uint32_t)(((i * 128 + tid) & 7) | ((i * 128 + tid) / (8 * KC)) << 3); };
            auto piece_of = [&](int i) { return (uint32_t)((i * 128 + tid) / 8 % KC); };
            int32_t page[PER];
            auto pages = [&](uint32_t hf) {
#pragma unroll
                for (int i = 0; i < PER; i++) page[i] = page_of(begin + hf * G::PART + key_of(i));
            };
            auto load = [&](uint4 (&c)[PER], uint32_t hf) {
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const uint32_t key = begin + hf * G::PART + key_of(i);
                    c[i] = __ldg(reinterpret_cast<const uint4 *>(a.cache.k_dev + ((slot_of(page[i]) << a.bt.log2_bt) + (key & in_block)) * D + piece_of(i) * 16));
                }
            };
            // first warp: lane i % GROUPS looks after a tile's group i
            int32_t g_page = 0;
            float v_ref = TC_SMALLEST;
            if (warp % 4 == 0 && tiles > 0) g_page = page_of(begin + (lane % G::GROUPS) * 16);
            auto params = [&](uint32_t j) {   // of tile j, in the place of tile j - 8: S of tile j - 3 is done, so P of tile j - 5 was
                const uint64_t slot = slot_of(g_page);
                const bool bad = (uint32_t)g_page >= a.cache.blocks;
                const ltq_qparams kq = a.cache.k_qp_dev[slot];
                const float vs = a.cache.v_qp_dev[slot].scale;
                if (j + 1 < tiles) g_page = page_of(begin + (j + 1) * G::KEYS + (lane % G::GROUPS) * 16);
                if (bad && lane < G::GROUPS) atomicCAS(status, 0u, STATUS_BAD_BLOCK);
                float top = vs;   // (NaN is passed over)
#pragma unroll
                for (int o = 1; o < G::GROUPS; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                float rescale = 1.f;
                if (top > v_ref) {
                    const float next = top < 1e38f ? 2.f * top : top;
                    rescale = v_ref * __fdividef(1.f, next);
                    v_ref = next;
                }
                const float ratio = __fdiv_rn(vs, v_ref), x = fmaxf(ratio, TC_MIN_RATIO);
                const bool nan = ratio != ratio;
                const uint32_t any = __ballot_sync(0xFFFFFFFFu, bad) & ((1u << G::GROUPS) - 1);
                TilePar &p = s_par[j & 7];
                if (lane < G::GROUPS)
                    p.g[lane] = GroupPar{kq.scale * TC_CODE, kq.scale * (float)kq.zero_point, nan ? ratio : lg2(x), nan ? 1.f : __fdividef(1.f, x)};
                if (lane == 0) {
                    p.v_ref = v_ref;
                    p.rescale = rescale;
                    p.bad = any;
                }
            };
            auto convert = [&](uint32_t hf, uint4 (&cur)[PER], uint4 (&nxt)[PER]) -> bool {
                const uint32_t j = hf / G::PARTS, st = j & 1;
                if (hf + 1 < parts) load(nxt, hf + 1);
                if (hf + 2 < parts) pages(hf + 2);
                if (hf % G::PARTS == 0) {
                    if (warp % 4 == 0) params(j);
                    if (j >= 2 && !mbar_wait(k_empty + 8 * st, ((j - 2) >> 1) & 1, abort_flag, status, 0xB30u | st)) return false;
                }
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const uint32_t key = hf % G::PARTS * G::PART + key_of(i), ch = piece_of(i), w[4] = {cur[i].x, cur[i].y, cur[i].z, cur[i].w};
                    uint32_t x[8];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        x[2 * k] = __byte_perm(w[k], 0, 0x4140);
                        x[2 * k + 1] = __byte_perm(w[k], 0, 0x4342);
                    }
                    const uint32_t at = sk + st * G::K_BYTES + (ch / 4) * (G::KEYS * 128) + key * 128, c0 = (ch & 3) * 2;
                    sts16(at + ((c0 ^ (key & 7)) << 4), x[0], x[1], x[2], x[3]);
                    sts16(at + (((c0 + 1) ^ (key & 7)) << 4), x[4], x[5], x[6], x[7]);
                }
                if (hf % G::PARTS == G::PARTS - 1) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_arrive(k_full + 8 * st);
                }
                return true;
            };
            uint4 even[PER], odd[PER];
            if (tiles > 0) {
                pages(0);
                load(even, 0);
                pages(1);
            }
            for (uint32_t hf = 0; hf < parts; hf += 2)
                if (!convert(hf, even, odd) || hf + 1 >= parts || !convert(hf + 1, odd, even)) break;
        } else {
            // V: units of 8 keys x 8 head dimensions; neighbouring lanes take neighbouring groups of keys, for the banks again
            constexpr int KG = G::PART / 8, UNITS = KG * (D / 8), PER = (UNITS + 127) / 128;
            static_assert(PER == 1, "units");
            const bool busy = UNITS == 128 || tid < UNITS;
            const uint32_t kg = (uint32_t)tid % KG, d0 = (uint32_t)tid / KG * 8;
            int32_t page = 0;
            struct Codes {
                uint2 c[8];
                uint32_t z;
            };
            auto load = [&](Codes &c, uint32_t hf) {
                if (!busy) return;
                const uint64_t slot = slot_of(page);
                const uint32_t key = begin + hf * G::PART + kg * 8;
                const uint8_t *p = a.cache.v_dev + ((slot << a.bt.log2_bt) + (key & in_block)) * D + d0;
#pragma unroll
                for (int k = 0; k < 8; k++) c.c[k] = __ldg(reinterpret_cast<const uint2 *>(p + k * D));
                c.z = __ldg(&a.cache.v_qp_dev[slot].zero_point);
            };
            const uint32_t magic = 0x64646464u;
            auto convert = [&](uint32_t hf, Codes &cur, Codes &nxt) -> bool {
                const uint32_t j = hf / G::PARTS, st = j & 1;
                if (hf + 1 < parts) load(nxt, hf + 1);
                if (hf + 2 < parts) page = page_of(begin + (hf + 2) * G::PART + kg * 8);
                if (hf % G::PARTS == 0 && j >= 2 && !mbar_wait(v_empty + 8 * st, ((j - 2) >> 1) & 1, abort_flag, status, 0xB40u | st)) return false;
                if (busy) {
                    const uint32_t z = 0x64006400u + cur.z * 0x10001u;
                    const uint32_t key = hf % G::PARTS * G::PART + kg * 8, chunk = key / 8;
                        const uint32_t at = sv + st * G::V_BYTES;
#pragma unroll
                    for (int half = 0; half < 2; half++) {   // head dimensions d0 + 4 * half + 0..3
                        uint32_t lo[4], hi[4];                 // key pairs 2k, 2k+1: {d, d+1} and {d+2, d+3} interleaved
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint32_t u = half ? cur.c[2 * k].y : cur.c[2 * k].x, v = half ? cur.c[2 * k + 1].y : cur.c[2 * k + 1].x;
                            lo[k] = __byte_perm(u, v, 0x5140);
                            hi[k] = __byte_perm(u, v, 0x7362);
                        }
#pragma unroll
                        for (int d = 0; d < 4; d++) {
                            uint32_t x[4];
#pragma unroll
                            for (int k = 0; k < 4; k++) x[k] = h2sub(__byte_perm(d < 2 ? lo[k] : hi[k], magic, d & 1 ? 0x4342 : 0x4140), z);
                            const uint32_t dd = d0 + 4 * half + d;
                            sts16(at + dd * 128 + ((chunk ^ (dd & 7)) << 4), x[0], x[1], x[2], x[3]);
                        }
                    }
                }
                if (hf % G::PARTS == G::PARTS - 1) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_arrive(v_full + 8 * st);
                }
                return true;
            };
            Codes even, odd;
            if (tiles > 0) {
                page = page_of(begin + kg * 8);
                load(even, 0);
                page = page_of(begin + G::PART + kg * 8);
            }
            for (uint32_t hf = 0; hf < parts; hf += 2)
                if (!convert(hf, even, odd) || hf + 1 >= parts || !convert(hf + 1, odd, even)) break;
        }
    } else {
        // ---------------- MMA issue: a warp per row tile runs the loop, one elected lane issues ----------------
        regs_down<G::REGS_MMA>();
        constexpr uint32_t id_qk = idesc_f16(TC_ROWS, G::KEYS), id_pv = idesc_f16(TC_ROWS, D);
        const uint32_t rt = (uint32_t)warp & 3;
        if (rt < RT) {
            const uint32_t mine = rt ? tiles1 : tiles0;
            const uint32_t s_bar = s_full + 8 * SB * rt, p_bar = p_full + 8 * SB * rt, pv_bar = pv_done + 8 * SB * rt;
            auto wait = [&](uint32_t bar, uint32_t phase, uint32_t code) {
                return __all_sync(0xFFFFFFFFu, mbar_wait(bar, phase, abort_flag, status, code));
            };
            const uint64_t qd = make_smem_desc(sq + rt * G::Q_BYTES);
            // S of tile j; its buffer holds P of tile j - SB until the MMA that reads it is done
            auto scores = [&](uint32_t j) -> bool {
                const uint32_t st = j & 1, sb = j % SB;
                if (!wait(k_full + 8 * st, (j >> 1) & 1, 0xB60u | st)) return false;
                if (j >= SB && !wait(pv_bar + 8 * sb, ((j - SB) / SB) & 1, 0xB70u | sb)) return false;
                tc_fence_after();
                const uint64_t kd = make_smem_desc(sk + st * G::K_BYTES);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < D / 16; k++)
                        mma_ss(tmem + G::s_col(rt, sb), qd + (uint64_t)((k / 4) * (TC_ROWS * 128 / 16) + 2 * (k & 3)),
                               kd + (uint64_t)((k / 4) * (G::KEYS * 128 / 16) + 2 * (k & 3)), id_qk, k != 0);
                    umma_commit(s_bar + 8 * sb);
                    umma_commit(k_empty + 8 * st);
                }
                __syncwarp();
                return true;
            };
            auto output = [&](uint32_t j) -> bool {
                const uint32_t st = j & 1, sb = j % SB;
                if (!wait(v_full + 8 * st, (j >> 1) & 1, 0xB80u | st) || !wait(p_bar + 8 * sb, (j / SB) & 1, 0xB90u | sb)) return false;
                tc_fence_after();
                const uint64_t vd = make_smem_desc(sv + st * G::V_BYTES);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < G::KEYS / 16; k++)
                        mma_ts(tmem + G::o_col(rt), tmem + G::s_col(rt, sb) + 8 * k, vd + 2u * k, id_pv,
                               j != 0 || k != 0);
                    umma_commit(pv_bar + 8 * sb);
                    umma_commit(v_empty + 8 * st);
                }
                __syncwarp();
                return true;
            };
            bool ok = tiles > 0 && wait(q_full, 0, 0xB50u);
            if (SB == 1) {
                for (uint32_t j = 0; ok && j < mine; j++) ok = scores(j) && output(j);
            } else {   // S of the next tile before O of this one
                if (ok && mine > 0) ok = scores(0);
                for (uint32_t j = 0; ok && j < mine; j++) ok = (j + 1 >= mine || scores(j + 1)) && output(j);
            }
            // tiles that only the other row tile sees: their stages are not held up here
            for (uint32_t j = mine; ok && j < tiles; j++) {
                const uint32_t st = j & 1;
                ok = wait(k_full + 8 * st, (j >> 1) & 1, 0xBA0u | st) && wait(v_full + 8 * st, (j >> 1) & 1, 0xBB0u | st);
                if (ok && lane == 0) {
                    mbar_arrive(k_empty + 8 * st);
                    mbar_arrive(v_empty + 8 * st);
                }
                __syncwarp();
            }
        }
    }
    // Teardown: nobody leaves before every role is done with TMEM and shared memory.
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
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
    count_launch();
    e = launch_chained(cache_attention_tc_kernel<DT, D>, dim3(a.cache.kv_heads * a.splits, a.bt.seqs, a.row_tiles), dim3(TcGeo<D>::THREADS), TcGeo<D>::SMEM, stream, a);
    return e != cudaSuccess || a.splits == 1 ? e : (DT == LTQ_F16 ? launch_attention_join_f16 : launch_attention_join_bf16)(a, TC_ROWS * TcGeo<D>::RT, stream);
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

uint32_t attn_tc_rows(uint32_t head_dim) { return head_dim <= 128 ? 2 * TC_ROWS : TC_ROWS; }

cudaError_t launch_attention_tc(const AttnArgs &a, int dtype, cudaStream_t stream)
{
    return dtype == LTQ_F16 ? launch_tc_d<LTQ_F16>(a, stream) : launch_tc_d<LTQ_BF16>(a, stream);
}

}  // namespace ltq
