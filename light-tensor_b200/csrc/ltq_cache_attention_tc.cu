// Attention of many new tokens over the 8-bit cache (prompts and chunks of them) on the 5th-generation tensor cores.
//
// A CTA owns two tiles of 128 rows (new tokens x query heads of one group) of one sequence and key/value head and walks the
// keys in tiles of 64 (head_dim above 128: one row tile; tensor memory holds O and two S of every row):
//   S [128 x keys]  = Q [128 x D] . K^T        tcgen05.mma kind::f16, both operands in shared memory
//   P               = exp2(S * scales - m)     one thread per row, straight out of tensor memory
//   O [128 x D]    += P [128 x keys] . V       P as the operand in tensor memory (over S), V transposed in shared memory
//
//   copies       one warp: a tile's codes by bulk copies into a ring, up to four parts ahead.
//   conversion   four warps for K, four for V: codes -> halves, for both row tiles.  K's codes become subnormal halves, code * 2^-24, by
//                a byte permute alone, their zero points come off the scores (times the sum of q).  V's get 0x64 above them,
//                the half 1024 + code, minus (1024 + zero point), exact.  K is written as rows of keys, V as rows of head dimensions
//                (eight keys' bytes gathered per 16-byte store), both under the 128-byte swizzle the MMA reads; lanes are
//                dealt so that loads and stores spread over the banks.
//   MMA issue    one warp per row tile, so that each goes its own way: S of a tile goes out before O of the one in front.
//   softmax      two warpgroups per row tile take the tiles in turn, one per S buffer: thread = row = TMEM lane, so that no reduction
//                crosses threads.  The reference m moves only when a tile's weights add up to more than 2^15, from 2^3 for the
//                largest, O is hardly ever rescaled and no maximum is taken on the way.  m is an integer: what two tiles in a row, which
//                two warps have at the same time, have to agree on is a power of two.  A tile with masked keys or a new
//                maximum goes a careful way of its own, from the scores that are still in tensor memory.
//   parameters   one warp: the scales and zero points of every 16 keys.
//
// Measured on 1500 and 1109 new tokens behind up to 4500, 32 query and 8 key/value heads of 128 (230 us, 109 us at the tensor cores'
// measured rate).  A tile takes about 2000 cycles; its MMAs take 1300 of them (48 each for S, where Q's 4 KB per 16 of D come
// through the shared memory port, 64 for O; nothing else slows them down, but every access to tensor memory waits about 90
// cycles for a gap between them, whatever its width), its exponentials 1024, its instructions about 1400 issue slots.
//  * one softmax warpgroup per row tile: 299 us (its chain of latencies is the bound)
//  * codes loaded by the converting warps themselves: 330 us (load latency per tile)
//  * masks as selects on the common way: 247 us
//  * tiles of 128 keys, one S buffer: 375 us; the two row tiles issued by one warp: slower by a fifth
//  * the tiles divided evenly over persistent CTAs, with a join: 289 us (each piece of a group costs about 15 000 cycles)
// The warps' registers are divided by need (setmaxnreg).
//
// Scales: K's block scale multiplies the scores.  V's goes into the exponent as its logarithm, so that P holds weights, exp2(score) * V
// scale, and m is the reference of a row's own weights (with the largest V scale in sight as the reference, one loud block that a
// row gives no weight took the bits of all others: 2^22 times louder, outputs were 2 % off and more).  The sum of the probabilities
// is the sum of the weights of every 16 keys over their V scale, under the same reference; where a tile's V scales are so
// far below the loudest that such a weight could vanish and its probability not, the careful way takes the probabilities themselves.
// q is scaled by a power of two per row, so that halves hold it exactly or to 11 bits (half, bfloat16 queries).
//
// Every wait is bounded, see mbar_wait.
#include <cuda_fp16.h>

#include "ltq_cache.cuh"
#include "ltq_ptx.cuh"
#include "ltq_tcgen05.cuh"

namespace ltq {

namespace {

constexpr int TC_ROWS = 128;
constexpr float TC_MAX_SUM = 32768.f;   // a weight is below it, and a half
constexpr float TC_HEAD = 3.f;          // a row's largest weight is 2^(TC_HEAD - 1) to 2^TC_HEAD when the reference is taken from it
constexpr float TC_SMALLEST = 1.17549435e-38f;   // 2^-126
// Weights down to 2^-126 are floats.  The sum of probabilities is taken from them where no V scale of a tile is below the loudest
// so far by more than 2^TC_SPREAD (what is lost then is below 2^-30 of the sum) or below 2^TC_QUIET (its inverse, 2^15 times and more,
// has to be a float); a V scale below that one does not lower the reference further.
constexpr float TC_SPREAD = 96.f, TC_QUIET = -100.f;
constexpr float TC_CODE = 16777216.f;            // 2^24: a K code's half is the code over this

// What the softmax needs of 16 keys: K scale times 2^24, K scale times zero point, log2 of the V scale and 2^-that.
struct GroupPar {
    float ks, kzs, lv, inv;
};

template <int D>
struct TcGeo {
    static constexpr int RT = D <= 128 ? 2 : 1;                    // row tiles per CTA
    static constexpr int KEYS = 64, GROUPS = KEYS / 16;
    static constexpr int PARTS = RT == 2 ? 1 : 2, PART = KEYS / PARTS;   // a tile is fetched and converted in so many parts
    static constexpr int RAW = RT == 2 ? 4 : 2;                    // parts whose codes are on their way or waiting
    static constexpr int V_GROUP = 8 * D + 16;                     // eight keys of V, 16 bytes apart: reads of a column spread over the banks
    static constexpr int RAW_BYTES = PART * D + PART / 8 * V_GROUP - 16;
    static constexpr int SB = 2;                                   // S buffers per row tile
    static constexpr int PANELS = (D + 63) / 64;                   // 64 halves = one 128-byte swizzle row
    static constexpr int Q_BYTES = PANELS * TC_ROWS * 128;
    static constexpr int K_BYTES = PANELS * KEYS * 128;
    static constexpr int V_BYTES = D * 128;                        // rows = head dimensions, 64 keys = 128 bytes
    static constexpr int SW = RT * SB;                             // softmax warpgroups: one per row tile and S buffer
    static constexpr int THREADS = 128 * (SW + 3);                 // warpgroups: softmax, K, V, MMA issue
    // Registers per thread: as launched (896 or 640 threads), and after setmaxnreg, which may only raise with .inc, lower with .dec,
    // and hands out no more than the block was launched with.
    static constexpr int REGS = RT == 2 ? 72 : 96;
    static constexpr int REGS_SOFTMAX = RT == 2 ? 88 : 136, REGS_CONVERT = RT == 2 ? 48 : 80, REGS_MMA = RT == 2 ? 56 : 48;
    static_assert(SW * REGS_SOFTMAX + 2 * REGS_CONVERT + REGS_MMA == (SW + 3) * REGS, "register shares");
    static_assert(REGS_SOFTMAX >= REGS && REGS_CONVERT <= REGS && REGS_MMA <= REGS, "register shares");
    static constexpr int BARS = 9 + RT * 3 * SB + SW * 4 + 2 * RAW;   // k_full k_empty v_full v_empty q_full; s_full p_full pv_done; m_done; raw_full raw_empty
    struct TilePar {
        GroupPar g[GROUPS];
        uint32_t bad, wide;     // bit i: group i's block does not exist; 1: V scales too far below the loudest for the common way
        uint32_t pad[2];
    };
    static constexpr size_t SMEM = 1024 + RT * Q_BYTES + 2 * K_BYTES + 2 * V_BYTES + RAW * RAW_BYTES + 8 * sizeof(TilePar) + SW * TC_ROWS * 4 + (BARS + BARS % 2) * 8 + RAW * 16 + 16;
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
__device__ __forceinline__ float times2(float x, float e)   // x * 2^e, where 2^e alone may not be a float
{
    return x * ex2(0.5f * e) * ex2(0.5f * e);
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
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
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
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), sq = (raw + 1023u) & ~1023u;
    const uint32_t sk = sq + RT * G::Q_BYTES, sv = sk + 2 * G::K_BYTES;
    uint8_t *codes = smem_raw + (sv - raw) + 2 * G::V_BYTES, *after = codes + G::RAW * G::RAW_BYTES;   // a part: K, then V in groups of eight keys
    TilePar *s_par = reinterpret_cast<TilePar *>(after);     // of eight tiles
    float *s_m = reinterpret_cast<float *>(after + 8 * sizeof(TilePar));   // [row tile][S buffer][row]: the reference maximum
    uint64_t *bars = reinterpret_cast<uint64_t *>(s_m + G::SW * TC_ROWS);
    uint32_t(*s_zero)[4] = reinterpret_cast<uint32_t(*)[4]>(bars + G::BARS + G::BARS % 2);   // zero points of a part's V, per 16 keys
    uint32_t *s_misc = reinterpret_cast<uint32_t *>(s_zero + G::RAW);   // [0] tmem base, [1] abort flag, [2] another one, [3] the group
    volatile uint32_t *abort_flag = s_misc + 1;
    const uint32_t k_full = smem_u32(bars), k_empty = k_full + 16, v_full = k_full + 32, v_empty = k_full + 48, q_full = k_full + 64;
    const uint32_t s_full = k_full + 72, p_full = s_full + 8 * SB * RT, pv_done = p_full + 8 * SB * RT,   // [row tile][S buffer]
                   m_done = pv_done + 8 * SB * RT,                                                           // [row tile][S buffer][warp]
                   raw_full = m_done + 8 * 4 * G::SW, raw_empty = raw_full + 8 * G::RAW;
    const int warp = __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;   // (known to be uniform)
    const uint32_t wg = (uint32_t)warp >> 2;
    uint32_t *status = a.bt.status;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < 2; i++) {
            mbar_init(k_full + 8 * i, 129);
            mbar_init(k_empty + 8 * i, RT);
            mbar_init(v_full + 8 * i, 128);
            mbar_init(v_empty + 8 * i, RT);
        }
        for (uint32_t i = 0; i < SB * RT; i++) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 4);
            mbar_init(pv_done + 8 * i, 1);
        }
        for (uint32_t i = 0; i < G::SW * 4; i++) mbar_init(m_done + 8 * i, 1);
        for (uint32_t i = 0; i < (uint32_t)G::RAW; i++) {
            mbar_init(raw_full + 8 * i, 1);
            mbar_init(raw_empty + 8 * i, 8);
        }
        mbar_init(q_full, 128 * G::SW);
        s_misc[1] = s_misc[2] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 0) {
        tmem_alloc(smem_u32(s_misc), 512);
        tmem_relinquish();
        griddep_launch_dependents();   // not before: see there
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_wait();
    const uint32_t tmem = s_misc[0];

    auto tiles_to = [&](const CacheSeq &s, uint32_t row) -> uint32_t {   // key tiles that a sequence's rows up to this one see
        const int keys = s.len - s.n + (int)(row / a.group) + 1;
        return keys > 0 ? ((uint32_t)keys + G::KEYS - 1) / G::KEYS : 0u;
    };
    // This CTA's group of row tiles.  Where there is more than the device takes at once the groups go by the tiles they see, most first
    // (the case above: 271 us in the grid's order, 247 us by tiles, both before the last step).
    const uint32_t split = blockIdx.x / a.cache.kv_heads, h = blockIdx.x - split * a.cache.kv_heads, pairs = gridDim.y * gridDim.z;
    uint32_t b = blockIdx.y, group = gridDim.z - 1 - blockIdx.z;
    if (pairs * gridDim.x > a.ctas && pairs <= G::THREADS) {
        uint32_t *s_weight = reinterpret_cast<uint32_t *>(smem_raw);   // (nothing else is there yet)
        const uint32_t mine_b = threadIdx.x % gridDim.y, mine_group = threadIdx.x / gridDim.y;
        uint32_t weight = 0;   // tiles, plus one for the group itself
        if (threadIdx.x < pairs) {
            const CacheSeq s = cache_seq(a.bt, mine_b);
            const uint32_t rows = s.ok ? (uint32_t)s.n * a.group : 0u, first = mine_group * (TC_ROWS * RT);
            if (first < rows) weight = 1 + tiles_to(s, (first + TC_ROWS * RT < rows ? first + TC_ROWS * RT : rows) - 1);
        }
        s_weight[threadIdx.x] = weight;
        __syncthreads();
        if (threadIdx.x < pairs) {
            uint32_t rank = 0;
            for (uint32_t i = 0; i < pairs; i++) rank += s_weight[i] > weight || (s_weight[i] == weight && i < threadIdx.x);
            if (rank == blockIdx.y + blockIdx.z * gridDim.y) s_misc[3] = threadIdx.x;
        }
        __syncthreads();
        b = s_misc[3] % gridDim.y;
        group = s_misc[3] / gridDim.y;
    }
    const uint32_t row0 = group * (TC_ROWS * RT);
    const CacheSeq s = cache_seq(a.bt, b);
    if (!s.ok && threadIdx.x == 0) atomicCAS(a.bt.refused, 0u, REFUSED_SEQUENCE);
    const uint32_t rows = s.ok ? (uint32_t)s.n * a.group : 0u;
    auto tiles_of = [&](uint32_t rt) -> uint32_t {   // key tiles that row tile rt sees
        const uint32_t first = row0 + rt * TC_ROWS;
        return first >= rows ? 0u : tiles_to(s, (first + TC_ROWS < rows ? first + TC_ROWS : rows) - 1);
    };
    const uint32_t all0 = tiles_of(0), all1 = RT == 2 ? tiles_of(RT - 1) : 0u, all = all0 > all1 ? all0 : all1;
    // this CTA's tiles: [tile0, tile0 + tiles), of which the row tiles see the first tiles0 and tiles1
    const uint32_t tile0 = (uint32_t)((uint64_t)all * split / a.splits), tiles = (uint32_t)((uint64_t)all * (split + 1) / a.splits) - tile0;
    auto part_of = [&](uint32_t n) { return n <= tile0 ? 0u : (n - tile0 < tiles ? n - tile0 : tiles); };
    const uint32_t tiles0 = part_of(all0), tiles1 = part_of(all1);
    const uint32_t place = ((b * gridDim.z + group) * a.cache.kv_heads + h) * a.splits;   // workspace slot of split 0
    if (a.splits > 1 && split == 0 && row0 < rows && threadIdx.x == 0)
        a.item[((uint64_t)b * gridDim.z + group) * a.cache.kv_heads + h] = make_int2((int)place, (int)(place + a.splits - 1));

    const int32_t *table = a.bt.table + (uint64_t)b * a.bt.table_width;
    const uint32_t in_block = (1u << a.bt.log2_bt) - 1, parts = G::PARTS * tiles;
    const uint32_t begin = tile0 * G::KEYS, end = (tile0 + tiles) * G::KEYS, last_key = end < (uint32_t)s.len ? end - 1 : (uint32_t)s.len - 1;
    // the block that holds a key; keys behind the sequence's last read its block (masked later)
    auto page_of = [&](uint32_t key) { return __ldg(table + ((key < last_key ? key : last_key) >> a.bt.log2_bt)); };
    auto slot_of = [&](int32_t page) { return (uint64_t)((uint32_t)page < a.cache.blocks ? (uint32_t)page : 0u) * a.cache.kv_heads + h; };

    if (wg < G::SW) {
        // ---------------- softmax: one row per thread, this warpgroup's half of the tiles ----------------
        regs_up<G::REGS_SOFTMAX>();
        const uint32_t rt = wg / SB, sb = wg % SB, quarter = (uint32_t)warp & 3, mine = rt ? tiles1 : tiles0;
        const uint32_t r = quarter * 32 + lane, row = row0 + rt * TC_ROWS + r, t = row / a.group;
        const bool real = row < rows;
        auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + rt * 4 + quarter) : "memory"); };             // with the rows' other warp
        auto meet_all = [&]() { asm volatile("bar.sync %0, 256;" ::"r"(1 + RT * 4 + rt) : "memory"); };   // the row tile's warps
        // 16 rows of q per warp, whole rows at a time: a power of two on each, so that halves hold it.
        float2 *const row_par = reinterpret_cast<float2 *>(s_m) + rt * TC_ROWS;
        {
            constexpr int LANES = D <= 32 ? 4 : (D <= 64 ? 8 : (D <= 128 ? 16 : 32)), PASSES = LANES / 2;   // lanes per row, eight elements each
            const int at = lane % LANES;
            const bool has = at < D / 8;
            uint32_t qw[PASSES][4];   // one memory latency
            auto row_of = [&](int i) { return (sb * 4 + quarter) * 16 + (uint32_t)(i * (32 / LANES) + lane / LANES); };
#pragma unroll
            for (int i = 0; i < PASSES; i++) {
                const uint32_t qr = row0 + rt * TC_ROWS + row_of(i), qt = qr / a.group;
                const uint16_t *q = static_cast<const uint16_t *>(a.q) + ((uint64_t)s.off + qt) * a.ld_q + (uint64_t)(h * a.group + qr - qt * a.group) * D + 8 * at;
                qw[i][0] = qw[i][1] = qw[i][2] = qw[i][3] = 0;
                if (qr < rows && has) {
                    if (a.q_vec8) {
                        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(q));
                        qw[i][0] = v.x; qw[i][1] = v.y; qw[i][2] = v.z; qw[i][3] = v.w;
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; k++) qw[i][k] = (uint32_t)q[2 * k] | (uint32_t)q[2 * k + 1] << 16;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < PASSES; i++) {
                // the largest magnitude, by its bits: both types' order like integers
                uint32_t top = 0;
#pragma unroll
                for (int k = 0; k < 4; k++) top = __vmaxu2(top, qw[i][k] & 0x7FFF7FFFu);
#pragma unroll
                for (int o = 1; o < LANES; o <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                top = top >> 16 > (top & 0xFFFFu) ? top >> 16 : top & 0xFFFFu;
                const bool finite = top < (DT == LTQ_F16 ? 0x7C00u : 0x7F80u);
                const int size = (int)(__float_as_uint(elem<DT>(top, 0)) >> 23) - 127;   // its exponent
                const int e = size < -90 ? 100 : 10 - size;   // most * 2^e in [2^10, 2^11), where that is a float
                const float f = __uint_as_float((uint32_t)(127 + e) << 23);
                float q_sum = 0.f;
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    w[k] = finite ? h2pack(elem<DT>(qw[i][k], 0) * f, elem<DT>(qw[i][k], 1) * f) : 0u;
                    const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
                    q_sum += x.x + x.y;
                }
#pragma unroll
                for (int o = 1; o < LANES; o <<= 1) q_sum += __shfl_xor_sync(0xFFFFFFFFu, q_sum, o);
                const uint32_t qr = row_of(i);
                if (has) sts16(sq + rt * G::Q_BYTES + (at / 8) * (TC_ROWS * 128) + qr * 128 + (((at & 7) ^ (qr & 7)) << 4), w[0], w[1], w[2], w[3]);
                if (at == 0) {
                    const float row_scale = finite ? a.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23) : __int_as_float(0x7FC00000);
                    row_par[qr] = make_float2(row_scale, row_scale * q_sum);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(q_full);
        }
        meet_all();
        const float row_scale = row_par[r].x, zero_scale = row_par[r].y;
        meet_all();   // (what follows takes the place)
        const int pos = real ? s.len - s.n + (int)t : 0x7FFFFFFF;
        const int first_pos = __reduce_min_sync(0xFFFFFFFFu, pos);
        const uint32_t lane_addr = tmem + ((quarter * 32) << 16), o_addr = lane_addr + G::o_col(rt), s_addr = lane_addr + G::s_col(rt, sb);
        const uint32_t s_bar = s_full + 8 * wg, p_bar = p_full + 8 * wg, pv_bar = pv_done + 8 * SB * rt;
        const uint32_t m_bar = m_done + 8 * (wg * 4 + quarter), m_other = m_done + 8 * ((wg ^ 1) * 4 + quarter);
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (uint32_t j = sb; j < mine; j += SB) {
            const uint32_t ph = (j / SB) & 1;
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(s_bar, ph, abort_flag, status, 0xE00u | sb));
            if (!ok) break;
            tc_fence_after();
            const TilePar &par = s_par[j & 7];
            const int key0 = (int)((tile0 + j) * G::KEYS);
            auto last_seen = [&](int k) { return par.bad >> k & 1 ? -1 : pos - key0 - 16 * k; };   // the last key of group k that the row sees
            uint32_t p[G::KEYS / 2];
            // The common way: everything is seen, and the reference stays.  Else the careful way, from the scores as they still are.
            bool careful = par.bad || par.wide || key0 + G::KEYS - 1 > first_pos;
            if (!careful) {
                float sum = 0.f, weight = 0.f;
#pragma unroll
                for (int c = 0; c < G::KEYS / 32; c++) {   // 32 keys at a time
                    uint32_t x[32];
                    tmem_ld32(s_addr + 32 * c, x);
                    GroupPar g[2];
#pragma unroll
                    for (int k = 0; k < 2; k++) g[k] = par.g[2 * c + k];
                    tmem_ld_wait();
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const float ks = row_scale * g[k].ks, base = g[k].lv - fmaf(zero_scale, g[k].kzs, m);
                        const uint64_t ks2 = pair(ks, ks), base2 = pair(base, base);
                        float2 y[8];
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            y[i] = unpair(fma2(pair(__uint_as_float(x[16 * k + 2 * i]), __uint_as_float(x[16 * k + 2 * i + 1])), ks2, base2));
                        uint64_t add[2];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            y[i].x = ex2(y[i].x);
                            y[i].y = ex2(y[i].y);
                            add[i & 1] = i < 2 ? pair(y[i].x, y[i].y) : add2(add[i & 1], pair(y[i].x, y[i].y));
                            p[16 * c + 8 * k + i] = h2pack(y[i].x, y[i].y);
                        }
                        const float2 s2 = unpair(add2(add[0], add[1]));
                        weight += s2.x + s2.y;
                        sum = fmaf(s2.x + s2.y, g[k].inv, sum);
                    }
                }
                careful = __any_sync(0xFFFFFFFFu, weight > TC_MAX_SUM);   // (with m at -inf everything is inf, and so is the sum)
                if (!careful) l += sum;
            }
            if (careful) {   // the largest weight first
                float best = -INFINITY;
#pragma unroll 1
                for (int k = 0; k < G::GROUPS; k++) {
                    uint32_t x[16];
                    tmem_ld16(s_addr + 16 * k, x);
                    const float ks = row_scale * par.g[k].ks, base = fmaxf(par.g[k].lv, TC_QUIET) - zero_scale * par.g[k].kzs;
                    const int see = last_seen(k);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; i++) best = i > see ? best : fmaxf(best, fmaf(__uint_as_float(x[i]), ks, base));
                }
                const float mx = fmaxf(m, ceilf(best) - TC_HEAD);
                if (m != mx) l = times2(l, m - mx);
                m = mx;
            }
            // The tile in front has its reference by now: the larger one holds for both.
            float alpha = 1.f;
            if (j > 0) {
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(m_other, ((j - 1) / SB) & 1, abort_flag, status, 0xE40u | sb));
                if (!ok) break;
                const float before = s_m[(wg ^ 1) * TC_ROWS + r], mx = fmaxf(m, before);
                if (__any_sync(0xFFFFFFFFu, m < before)) {
                    const float down = m == mx ? 1.f : ex2(m - mx);
                    if (m != mx) l = times2(l, m - mx);
                    if (!careful) {
                        const __half2 by = __float2half2_rn(down);   // a power of two
#pragma unroll
                        for (int i = 0; i < G::KEYS / 2; i++) *reinterpret_cast<__half2 *>(&p[i]) = __hmul2(*reinterpret_cast<__half2 *>(&p[i]), by);
                    }
                }
                if (before != mx) alpha = ex2(before - mx);
                m = mx;
            }
            s_m[wg * TC_ROWS + r] = m;
            __syncwarp();
            if (lane == 0) mbar_arrive(m_bar);
            if (__any_sync(0xFFFFFFFFu, alpha != 1.f)) {
                // O so far times alpha: once the MMA that last added to it is done (S of the tile in front is, so the one before that was)
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(pv_bar + 8 * (sb ^ 1), ((j - 1) / SB) & 1, abort_flag, status, 0xE10u | sb));
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
            if (!careful) {
                tmem_st32(s_addr, p);
            } else {
                const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll 1
                for (int k = 0; k < G::GROUPS; k++) {   // P takes the place of scores that are in registers already
                    uint32_t x[16], w[8];
                    tmem_ld16(s_addr + 16 * k, x);
                    const GroupPar g = par.g[k];
                    const float ks = row_scale * g.ks, score = -fmaf(zero_scale, g.kzs, ref), base = g.lv + score;
                    const int see = last_seen(k);
                    float sum = 0.f;
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float y0 = 2 * i > see ? 0.f : ex2(fmaf(__uint_as_float(x[2 * i]), ks, base));
                        const float y1 = 2 * i + 1 > see ? 0.f : ex2(fmaf(__uint_as_float(x[2 * i + 1]), ks, base));
                        sum += y0 + y1;
                        w[i] = h2pack(y0, y1);
                    }
                    if (!par.wide) {
                        l = fmaf(sum, g.inv, l);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i++) l += i > see ? 0.f : ex2(fmaf(__uint_as_float(x[i]), ks, score));
                    }
                    tmem_st8(s_addr + 8 * k, w);
                }
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_bar);
        }
        // The last tile's reference holds for all.
        if (ok && mine > 0) {
            const uint32_t last = mine - 1, lb = last % SB, ph = (last / SB) & 1;
            if (lb != sb) {
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(m_other, ph, abort_flag, status, 0xE20u | sb));
                const float mx = s_m[(wg ^ 1) * TC_ROWS + r];
                if (m != mx) l = times2(l, m - mx);
                m = mx;
            }
            ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait(pv_bar + 8 * lb, ph, abort_flag, status, 0xE28u | sb));
            tc_fence_after();
        }
        meet();
        s_m[wg * TC_ROWS + r] = l;
        meet();
        l += s_m[(wg ^ 1) * TC_ROWS + r];
        // this warpgroup's half of the head dimensions
        if (ok && a.splits > 1) {
            // the join works on sums near 1: their exponent goes into the reference, and off O
            const uint64_t at = (uint64_t)(place + split) * (TC_ROWS * RT) + rt * TC_ROWS + r;
            const int e = (int)((__float_as_uint(l) >> 23) & 0xFF) - 127, el = e < -126 ? -126 : (e > 126 ? 126 : e);
            const float back = __uint_as_float((uint32_t)(127 - el) << 23);
            if (real && sb == 0) a.part_ml[at] = make_float2(m + (float)el, l * back);
            float4 *dst = reinterpret_cast<float4 *>(a.part_o + at * D);
#pragma unroll 1
            for (int d = sb * (D / 2); d < (int)(sb + 1) * (D / 2); d += 16) {
                uint32_t o[16];
                if (mine > 0) {
                    tmem_ld16(o_addr + d, o);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (real)
                        dst[d / 4 + i] = mine > 0 ? make_float4(__uint_as_float(o[4 * i]) * back, __uint_as_float(o[4 * i + 1]) * back,
                                                                __uint_as_float(o[4 * i + 2]) * back, __uint_as_float(o[4 * i + 3]) * back)
                                                  : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        } else if (ok) {
            const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);   // a row that sees nothing: zeros
            uint16_t *dst = static_cast<uint16_t *>(a.out) + (((uint64_t)s.off + t) * a.q_heads + h * a.group + (row - t * a.group)) * D;
#pragma unroll 1
            for (int d = sb * (D / 2); d < (int)(sb + 1) * (D / 2); d += 16) {
                uint32_t o[16];
                if (mine > 0) {
                    tmem_ld16(o_addr + d, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] = 0;
                }
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; i++) w[i] = token_bits2<DT>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
                if (real) {
                    if (a.out_vec8) {
#pragma unroll
                        for (int i = 0; i < 2; i++) reinterpret_cast<uint4 *>(dst + d)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i++) dst[d + i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
                    }
                }
            }
        }
    } else if (wg < G::SW + 2) {
        // ---------------- conversion ----------------
        if constexpr (G::REGS_CONVERT < G::REGS) regs_down<G::REGS_CONVERT>();
        const int tid = threadIdx.x & 127;
        auto take = [&](uint32_t hf) {   // part hf of the codes is there
            return __all_sync(0xFFFFFFFFu, mbar_wait(raw_full + 8 * (hf % G::RAW), hf / G::RAW & 1, abort_flag, status, 0xE50u | hf % G::RAW));
        };
        auto give = [&](uint32_t hf) {
            __syncwarp();
            if (lane == 0) mbar_arrive(raw_empty + 8 * (hf % G::RAW));
        };
        if (wg == G::SW) {
            // K: 16-byte pieces, those of a row to neighbouring lanes; odd groups of four write their second half first (other banks)
            constexpr int KC = D / 16, PER = G::PART * KC / 128;
            static_assert(PER * 128 == G::PART * KC, "pieces");
#pragma unroll 1
            for (uint32_t hf = 0; hf < parts; hf++) {
                const uint32_t j = hf / G::PARTS, st = j & 1;
                if (!take(hf)) break;
                if (hf % G::PARTS == 0 && j >= 2 &&
                    !__all_sync(0xFFFFFFFFu, mbar_wait(k_empty + 8 * st, ((j - 2) >> 1) & 1, abort_flag, status, 0xE30u | st))) break;
                const uint4 *src = reinterpret_cast<const uint4 *>(codes + hf % G::RAW * G::RAW_BYTES) + tid;
                uint4 w[PER];
#pragma unroll
                for (int i = 0; i < PER; i++) w[i] = src[i * 128];
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const uint32_t u = (uint32_t)(i * 128 + tid) / KC, ch = (uint32_t)(i * 128 + tid) % KC, key = hf % G::PARTS * G::PART + u;
                    const bool second = ch & 4;
                    const uint32_t w0 = second ? w[i].z : w[i].x, w1 = second ? w[i].w : w[i].y, w2 = second ? w[i].x : w[i].z, w3 = second ? w[i].y : w[i].w;
                    const uint32_t at = sk + st * G::K_BYTES + (ch / 4) * (G::KEYS * 128) + key * 128, c0 = ((ch & 3) * 2 + second) ^ (key & 7);
                    sts16(at + (c0 << 4), __byte_perm(w0, 0, 0x4140), __byte_perm(w0, 0, 0x4342), __byte_perm(w1, 0, 0x4140), __byte_perm(w1, 0, 0x4342));
                    sts16(at + ((c0 ^ 1) << 4), __byte_perm(w2, 0, 0x4140), __byte_perm(w2, 0, 0x4342), __byte_perm(w3, 0, 0x4140), __byte_perm(w3, 0, 0x4342));
                }
                give(hf);
                if (hf % G::PARTS == G::PARTS - 1) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_arrive(k_full + 8 * st);
                }
            }
        } else {
            // V: units of 8 keys x 8 head dimensions; neighbouring lanes take neighbouring groups of keys
            constexpr int KG = G::PART / 8, UNITS = KG * (D / 8);
            static_assert(UNITS <= 128, "units");
            const bool busy = UNITS == 128 || tid < UNITS;
            const uint32_t kg = (uint32_t)tid % KG, d0 = (uint32_t)tid / KG * 8;
            const uint32_t magic = 0x64646464u;
#pragma unroll 1
            for (uint32_t hf = 0; hf < parts; hf++) {
                const uint32_t j = hf / G::PARTS, st = j & 1;
                if (!take(hf)) break;
                if (hf % G::PARTS == 0 && j >= 2 &&
                    !__all_sync(0xFFFFFFFFu, mbar_wait(v_empty + 8 * st, ((j - 2) >> 1) & 1, abort_flag, status, 0xE48u | st))) break;
                if (busy) {
                    const uint8_t *src = codes + hf % G::RAW * G::RAW_BYTES + G::PART * D + kg * G::V_GROUP + d0;
                    uint2 c[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) c[k] = *reinterpret_cast<const uint2 *>(src + k * D);
                    const uint32_t z = 0x64006400u + s_zero[hf % G::RAW][kg / 2] * 0x10001u;
                    const uint32_t chunk = (hf % G::PARTS * G::PART + kg * 8) / 8, at = sv + st * G::V_BYTES;
#pragma unroll
                    for (int half = 0; half < 2; half++) {   // head dimensions d0 + 4 * half + 0..3
                        uint32_t lo[4], hi[4];                 // key pairs 2k, 2k+1: {d, d+1} and {d+2, d+3} interleaved
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint32_t u = half ? c[2 * k].y : c[2 * k].x, v = half ? c[2 * k + 1].y : c[2 * k + 1].x;
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
                give(hf);
                if (hf % G::PARTS == G::PARTS - 1) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_arrive(v_full + 8 * st);
                }
            }
        }
    } else {
        // ---------------- MMA issue: a warp per row tile runs the loop, one elected lane issues ----------------
        regs_down<G::REGS_MMA>();
        constexpr uint32_t id_qk = idesc_f16(TC_ROWS, G::KEYS), id_pv = idesc_f16(TC_ROWS, D);
        const uint32_t rt = (uint32_t)warp & 3;
        if (rt == 2) {
            // The codes: a lane copies a block's share of K in the part (at most four), lane 8 + g eight keys of V.
            const uint32_t piece = G::PART <= in_block ? (uint32_t)G::PART : in_block + 1;   // keys of K per copy
            const bool k_lane = lane < G::PART / piece, v_lane = lane >= 8 && lane < 8 + G::PART / 8;
            const uint32_t first = k_lane ? lane * piece : (v_lane ? (lane - 8) * 8 : 0u);
            auto page_at = [&](uint32_t hf) { return page_of(begin + hf * G::PART + first); };
            auto zero_at = [&](int32_t page) { return (uint32_t)a.cache.v_qp_dev[slot_of(page)].zero_point; };
            int32_t page = 0, next = 0;
            uint32_t zero = 0, hf = 0;
            if (parts > 0) {
                page = page_at(0);
                zero = zero_at(page);
            }
            if (parts > 1) next = page_at(1);
            for (; hf < parts; hf++) {
                const uint32_t st = hf % G::RAW, bar = raw_full + 8 * st;
                if (!__all_sync(0xFFFFFFFFu, hf < (uint32_t)G::RAW || mbar_wait(raw_empty + 8 * st, (hf / G::RAW - 1) & 1, abort_flag, status, 0xE58u | st))) break;
                if (v_lane && lane % 2 == 0) s_zero[st][(lane - 8) / 2] = zero;
                __syncwarp();
                if (lane == 0) mbar_expect_tx(bar, G::PART * D * 2);
                __syncwarp();
                const uint64_t at = ((slot_of(page) << a.bt.log2_bt) + ((begin + hf * G::PART + first) & in_block)) * D;
                const uint32_t dst = smem_u32(codes) + st * G::RAW_BYTES;
                if (k_lane) bulk_load_1d(dst + first * D, a.cache.k_dev + at, piece * D, bar);
                if (v_lane) bulk_load_1d(dst + G::PART * D + (lane - 8) * G::V_GROUP, a.cache.v_dev + at, 8 * D, bar);
                page = next;
                if (hf + 1 < parts) zero = zero_at(page);
                if (hf + 2 < parts) next = page_at(hf + 2);
            }
            // given up: the copies still under way have to land before the block ends (a second, bounded wait)
            if (hf < parts)
                for (uint32_t i = hf > (uint32_t)G::RAW ? hf - G::RAW : 0u; i < hf; i++)
                    mbar_wait(raw_full + 8 * (i % G::RAW), i / G::RAW & 1, s_misc + 2, status, 0xE5Cu);
        } else if (rt == 3) {
            // what the softmax needs of every tile: lane i % GROUPS looks after its group i
            float loudest = -INFINITY;   // log2 of V's largest scale so far
            auto page_at = [&](uint32_t j) { return page_of(begin + j * G::KEYS + (lane % G::GROUPS) * 16); };
            int32_t page = tiles > 0 ? page_at(0) : 0;
            ltq_qparams kq{};
            float vs = 0.f;
            bool bad = false;
            auto fetch = [&]() {   // of the tile whose page is here
                const uint64_t slot = slot_of(page);
                bad = (uint32_t)page >= a.cache.blocks;
                kq = a.cache.k_qp_dev[slot];
                vs = a.cache.v_qp_dev[slot].scale;
            };
            if (tiles > 0) fetch();
            if (tiles > 1) page = page_at(1);
            for (uint32_t j = 0; j < tiles; j++) {
                // in the place of tile j - 8: S of tile j - 2 is done, so P of tile j - 4 was
                const uint32_t st = j & 1;
                if (!__all_sync(0xFFFFFFFFu, j < 2 || mbar_wait(k_empty + 8 * st, ((j - 2) >> 1) & 1, abort_flag, status, 0xE38u | st))) break;
                if (bad && lane < G::GROUPS) atomicCAS(a.bt.refused, 0u, REFUSED_BLOCK);
                // log2 of the scale, from its exponent where it has one; an infinity is as good as a NaN
                const float mantissa = __uint_as_float((__float_as_uint(vs) & 0x7FFFFFu) | 0x3F800000u);
                float lv = vs < TC_SMALLEST ? lg2(vs) : (float)((int)(__float_as_uint(vs) >> 23) - 127) + lg2(mantissa);
                if (!(vs < INFINITY)) lv = __int_as_float(0x7FC00000);
                if (bad) lv = 0.f;   // (nothing of it is seen)
                float top = bad || lv != lv ? -INFINITY : lv, low = bad || lv != lv ? INFINITY : lv;
#pragma unroll
                for (int o = 1; o < G::GROUPS; o <<= 1) {
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                    low = fminf(low, __shfl_xor_sync(0xFFFFFFFFu, low, o));
                }
                loudest = fmaxf(loudest, top);
                const uint32_t any = __ballot_sync(0xFFFFFFFFu, bad) & ((1u << G::GROUPS) - 1);
                TilePar &p = s_par[j & 7];
                if (lane < G::GROUPS) {
                    float inv;   // (as far as lv is rounded it is so on both sides; not flushed to zero, as ex2 would)
                    asm("ex2.approx.f32 %0, %1;" : "=f"(inv) : "f"(-lv));
                    p.g[lane] = GroupPar{kq.scale * TC_CODE, kq.scale * (float)kq.zero_point, lv, lv != lv ? 1.f : inv};
                }
                if (lane == 0) {
                    p.bad = any;
                    p.wide = low < fmaxf(loudest - TC_SPREAD, TC_QUIET);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(k_full + 8 * st);
                if (j + 1 < tiles) fetch();
                if (j + 2 < tiles) page = page_at(j + 2);
            }
        } else if (rt < RT) {
            const uint32_t mine = rt ? tiles1 : tiles0;
            const uint32_t s_bar = s_full + 8 * SB * rt, p_bar = p_full + 8 * SB * rt, pv_bar = pv_done + 8 * SB * rt;
            auto wait = [&](uint32_t bar, uint32_t phase, uint32_t code) {
                return __all_sync(0xFFFFFFFFu, mbar_wait(bar, phase, abort_flag, status, code));
            };
            const uint64_t qd = make_smem_desc(sq + rt * G::Q_BYTES);
            // S of tile j; its buffer holds P of tile j - SB until the MMA that reads it is done
            auto scores = [&](uint32_t j) -> bool {
                const uint32_t st = j & 1, sb = j % SB;
                if (!wait(k_full + 8 * st, (j >> 1) & 1, 0xE60u | st)) return false;
                if (j >= SB && !wait(pv_bar + 8 * sb, ((j - SB) / SB) & 1, 0xE70u | sb)) return false;
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
                if (!wait(v_full + 8 * st, (j >> 1) & 1, 0xE80u | st) || !wait(p_bar + 8 * sb, (j / SB) & 1, 0xE90u | sb)) return false;
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
            bool ok = tiles > 0 && wait(q_full, 0, 0xEC0u);
            // S of the next tile before O of this one
            if (ok && mine > 0) ok = scores(0);
            for (uint32_t j = 0; ok && j < mine; j++) ok = (j + 1 >= mine || scores(j + 1)) && output(j);
            // tiles that only the other row tile sees: their stages are not held up here
            for (uint32_t j = mine; ok && j < tiles; j++) {
                const uint32_t st = j & 1;
                ok = wait(k_full + 8 * st, (j >> 1) & 1, 0xEA0u | st) && wait(v_full + 8 * st, (j >> 1) & 1, 0xEB0u | st);
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
