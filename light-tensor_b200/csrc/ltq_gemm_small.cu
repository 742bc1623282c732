// uint8 x uint8 product with parameters per token and channel for calls of a decode batch's size: more rows than the weight-streaming
// kernel takes (16), too few output tiles to occupy the device with 128-deep steps through all of K.
//
// What bounds such a call is neither memory nor the tensor cores but what one SM's copies and MMAs cost one by one: with one
// 128-byte line of K per step (a copy of 128 activation rows and one of the tile's weight rows, four MMAs on one accumulator)
// a step took 400 cycles whatever the width was, 16 columns or 128, 17 tokens or 128 (K = 4096: 10 us on 16 SMs as on 64).  So
//  * a copy brings several lines (as in the weight-streaming kernel, {128-byte line, row, line along K}: a copy below 16 KB costs
//    as much as one of 16 KB) and of the activations only the rows there are, in groups of eight; the MMA's remaining rows
//    are computed from whatever lies behind them and never read;
//  * four warps issue MMAs, each one 32-byte K step of every line into an accumulator of its own; the epilogue adds the four up
//    (int32, exact in any order);
//  * where the tiles leave SMs idle a cluster of 2 or 4 CTAs shares a tile, each taking a part of K.  Every CTA finishes a slice
//    of the tile's columns: it gets the others' partial sums of its slice through distributed shared memory;
//  * the tile width is a run-time multiple of 16, chosen so that the tiles fill the device in whole rounds;
//  * one tile per CTA: nothing is double buffered and the ring takes what shared memory there is;
//  * the first weight boxes are on their way before the kernel in front (the activation quantise) has finished.
// Warps 0..3 issue, 4..7 are the epilogue (thread = row), 8 loads.  Every mbarrier wait is bounded.
#include <cuda.h>

#include "ltq_gemm_small.cuh"
#include "ltq_tcgen05.cuh"
#include "ltq_tokens.cuh"

namespace ltq {

namespace {

constexpr int SM_M = 128, SM_BK = 128, SM_THREADS = 288, SM_ACC = 4, SM_MAX_STAGES = 8, SM_MAX_BN = 128;
constexpr size_t SM_SMEM_LIMIT = 226 * 1024;

struct SmallLayout {
    uint32_t a_rows, stages, stage_bytes;
    size_t smem;
};
// Ring, then the partial sums received from the other CTAs of the cluster, the column terms and barriers.  The ring also serves as
// the staging area of unaligned output rows.  An MMA reads 128 rows from the start of an activation line tile whatever it
// holds: up to 16 KB behind the last one belong to the block.
SmallLayout small_layout(const SmallPlan &p, uint64_t M)
{
    SmallLayout l;
    l.a_rows = M < SM_M ? (uint32_t)(M + 7) / 8 * 8 : SM_M;
    l.stage_bytes = p.lines * (l.a_rows + p.bn) * SM_BK;
    const size_t fixed = 1024 + (size_t)(p.split - 1) * SM_M * (p.bn / p.split) * 4 + SM_MAX_BN * 16 + 256;
    const size_t over = (size_t)(SM_M - l.a_rows) * SM_BK;
    const size_t fit = (SM_SMEM_LIMIT - fixed - over) / l.stage_bytes;
    l.stages = (uint32_t)(fit < SM_MAX_STAGES ? fit : SM_MAX_STAGES);
    size_t ring = (size_t)l.stages * l.stage_bytes;
    const size_t staging = (size_t)4 * 32 * (p.bn / p.split + 1) * 4;
    l.smem = fixed + over + (ring > staging ? ring : staging);
    return l;
}

__device__ __forceinline__ uint32_t in_cta(uint32_t smem_addr, uint32_t rank)   // the same place in another CTA of the cluster
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_cluster16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}

}  // namespace

// Grid: tiles * split, clusters of `split` along x; OUT: OUT_TOKENS + ltq_dtype.
template <int OUT>
__global__ void __launch_bounds__(SM_THREADS, 1)
gemm_small_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, uint32_t M, uint32_t N, uint32_t K,
                  uint32_t bn, uint32_t split, uint32_t lines, uint32_t a_rows, uint32_t stages, uint32_t ring_bytes, Epilogue epi, void *__restrict__ out, uint32_t *status)
{
    constexpr int DT = OUT - OUT_TOKENS;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), ring = (raw + 1023u) & ~1023u, slice = bn / split;
    const uint32_t a_bytes = lines * a_rows * SM_BK, b_bytes = lines * bn * SM_BK, stage_bytes = a_bytes + b_bytes;
    uint8_t *after = smem_raw + (ring - raw) + ring_bytes;
    uint32_t *recv = reinterpret_cast<uint32_t *>(after);                     // [split - 1][slice / 8][128 rows][8]
    uint4 *s_col = reinterpret_cast<uint4 *>(after + (split - 1) * SM_M * slice * 4);
    uint64_t *bars = reinterpret_cast<uint64_t *>(s_col + SM_MAX_BN);         // full[8] empty[8] done
    uint32_t *s_misc = reinterpret_cast<uint32_t *>(bars + 2 * SM_MAX_STAGES + 1);
    volatile uint32_t *abort_flag = s_misc + 1;
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * SM_MAX_STAGES, done = empty0 + 8 * SM_MAX_STAGES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = split == 1 ? 0u : cluster_ctarank(), tile = blockIdx.x / split;
    const uint32_t tiles_n = (N + bn - 1) / bn, m0 = (tile / tiles_n) * SM_M, n0 = (tile % tiles_n) * bn;
    const uint32_t blocks = (K + lines * SM_BK - 1) / (lines * SM_BK), kb0 = (uint32_t)((uint64_t)blocks * rank / split),
                   kb1 = (uint32_t)((uint64_t)blocks * (rank + 1) / split);

    // Block `kb` of `lines` lines, all rows of the box: a 3-D copy, or a 2-D one of a single line (K not a multiple of 128: what is
    // behind the end arrives as zeros either way).
    auto load = [&](uint32_t dst, const CUtensorMap *map, uint32_t bar, uint32_t kb, uint32_t row) {
        if (lines > 1) tma_load_3d(dst, map, bar, 0, (int32_t)row, (int32_t)(kb * lines));
        else tma_load_2d(dst, map, bar, (int32_t)(kb * SM_BK), (int32_t)row);
    };

    if (threadIdx.x == 256) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
        for (uint32_t i = 0; i < stages; i++) {
            mbar_init(full0 + 8 * i, 1);
            mbar_init(empty0 + 8 * i, SM_ACC);
        }
        mbar_init(done, SM_ACC);
        s_misc[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        // Weights do not depend on the kernel in front (without early_weights there is none to wait for): the ring's worth goes out now,
        // the activation boxes follow behind the dependency and make the stages' one arrival.
        const uint32_t head = kb1 - kb0 < stages ? kb1 - kb0 : stages;
        for (uint32_t i = 0; i < head; i++) {
            mbar_expect_tx_only(full0 + 8 * i, b_bytes);
            load(ring + i * stage_bytes + a_bytes, &map_b, full0 + 8 * i, kb0 + i, n0);
        }
        griddep_wait();
        for (uint32_t i = 0; i < head; i++) {
            mbar_expect_tx(full0 + 8 * i, a_bytes);
            load(ring + i * stage_bytes, &map_a, full0 + 8 * i, kb0 + i, m0);
        }
    }
    if (warp == 0) {
        tmem_alloc(smem_u32(s_misc), SM_ACC * SM_MAX_BN);
        tmem_relinquish();
        griddep_launch_dependents();   // not before: see there
    }
    tc_fence_before();
    __syncthreads();
    if (split > 1) cluster_arrive();   // every CTA of the cluster runs once this phase is over: waited for before its memory is written
    tc_fence_after();
    const uint32_t tmem = s_misc[0];

    if (warp == 8) {
        // ---------------- TMA producer (the ring is filled already) ----------------
        if (lane == 0) {
            uint32_t st = 0, ph = 0;
            for (uint32_t kb = kb0 + stages; kb < kb1; kb++) {
                if (!mbar_wait(empty0 + 8 * st, ph, abort_flag, status, 0xF00u | st)) break;
                mbar_expect_tx(full0 + 8 * st, stage_bytes);
                load(ring + st * stage_bytes, &map_a, full0 + 8 * st, kb, m0);
                load(ring + st * stage_bytes + a_bytes, &map_b, full0 + 8 * st, kb, n0);
                if (++st == stages) { st = 0; ph ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp < SM_ACC) {
        // ---------------- MMA issue: K step `warp` of every block ----------------
        const uint32_t idesc = make_idesc_i8(SM_M, (int)bn), acc = tmem + (uint32_t)warp * SM_MAX_BN;
        uint32_t st = 0, ph = 0;
        bool ok = true;
        for (uint32_t kb = kb0; kb < kb1; kb++) {
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(full0 + 8 * st, ph, abort_flag, status, 0xF10u | st));
            if (!ok) break;
            tc_fence_after();
            const uint64_t a_desc = make_smem_desc(ring + st * stage_bytes) + 2u * warp;
            const uint64_t b_desc = make_smem_desc(ring + st * stage_bytes + a_bytes) + 2u * warp;
            if (elect_one()) {
                for (uint32_t l = 0; l < lines; l++)
                    umma_i8(acc, a_desc + (uint64_t)(l * a_rows * (SM_BK / 16)), b_desc + (uint64_t)(l * bn * (SM_BK / 16)), idesc,
                            kb != kb0 || l != 0 ? 1u : 0u);
                umma_commit(empty0 + 8 * st);
            }
            __syncwarp();
            if (++st == stages) { st = 0; ph ^= 1; }
        }
        if (ok && elect_one()) umma_commit(done);
        __syncwarp();
    }
    const uint32_t q = (uint32_t)warp & 3u, r = q * 32 + lane, et = threadIdx.x - 128;
    const uint32_t lane_addr = tmem + ((q * 32u) << 16);
    const bool epilogue = warp >= 4 && warp < 8;
    // eight columns of this thread's row, the four accumulators added up
    auto sums = [&](uint32_t col, uint32_t (&v)[8]) {
        uint32_t w1[8], w2[8], w3[8];
        tmem_ld8(lane_addr + col, v);
        tmem_ld8(lane_addr + SM_MAX_BN + col, w1);
        tmem_ld8(lane_addr + 2 * SM_MAX_BN + col, w2);
        tmem_ld8(lane_addr + 3 * SM_MAX_BN + col, w3);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] += w1[k] + w2[k] + w3[k];
    };
    bool ok = true;
    if (epilogue) {
        // ---------------- epilogue, first half: the other CTAs' slices go to them ----------------
        griddep_wait();   // token parameters and sums come from the kernel in front
        for (uint32_t j = et; j < slice; j += 128) {
            const uint32_t gj = n0 + rank * slice + j;
            s_col[j] = gj < N ? token_col(epi, gj) : make_uint4(0, 0, 0, 0);
        }
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(done, 0, abort_flag, status, 0xF20u));
        if (split > 1) cluster_wait();
        if (ok) {
            tc_fence_after();
            for (uint32_t to = 0; to < split; to++) {
                if (to == rank) continue;
                // in CTA `to`: the part of this one, numbered among the senders in order
                const uint32_t base = in_cta(smem_u32(recv) + (rank < to ? rank : rank - 1) * SM_M * slice * 4, to);
                for (uint32_t u = 0; u < slice / 8; u++) {
                    uint32_t v[8];
                    sums(to * slice + 8 * u, v);
                    const uint32_t at = base + (u * SM_M + r) * 32;
                    st_cluster16(at, v[0], v[1], v[2], v[3]);
                    st_cluster16(at + 16, v[4], v[5], v[6], v[7]);
                }
            }
        }
    }
    if (!epilogue && split > 1) {
        __syncwarp();
        cluster_wait();
    }
    __syncthreads();                 // column terms, and every role is done with the ring
    if (split > 1) cluster_sync();   // the partial sums have arrived everywhere (and nobody's shared memory goes before that)
    if (epilogue && ok) {
        // ---------------- second half: own slice ----------------
        const bool relu = epi.flags & LTQ_FLAG_RELU;
        const uint64_t ldc = epilogue_pitch(epi, N);
        constexpr uint32_t ESZ = DT == LTQ_F32 ? 4 : 2;
        const bool vec_ok = epilogue_vec_ok(epi, out, N, ESZ);
        const uint32_t row = m0 + r, c0 = n0 + rank * slice;
        const TokenRow tr = row < M ? token_row(epi, row) : TokenRow{0, 0, 0.f};
        float *stage = reinterpret_cast<float *>(smem_raw + (ring - raw)) + q * 32 * (slice + 1);   // [32 rows][slice + 1], unaligned output only
        for (uint32_t u = 0; u < slice / 8; u++) {
            uint32_t v[8];
            sums(rank * slice + 8 * u, v);
            for (uint32_t from = 0; from + 1 < split; from++) {
                const uint4 *p = reinterpret_cast<const uint4 *>(recv + (((uint64_t)from * (slice / 8) + u) * SM_M + r) * 8);
                const uint4 a = p[0], b = p[1];
                v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
                v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
            }
            const uint32_t c = c0 + 8 * u;
            if (vec_ok) {
                if (row < M && c < N) token_chunk<OUT, 8>(v, tr, s_col + 8 * u, relu, out, row * ldc + c, true, N - c < 8 ? (int)(N - c) : 8);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) stage[lane * (slice + 1) + 8 * u + k] = token_value(v[k], tr, s_col[8 * u + k], relu);
            }
        }
        if (!vec_ok) {
            // rows that do not start on 16-byte boundaries: a warp writes them one after the other, lanes side by side
            __syncwarp();
            const uint32_t rows = M > m0 + q * 32 ? (M - m0 - q * 32 < 32 ? M - m0 - q * 32 : 32) : 0;
            for (uint32_t j = lane; j < slice && c0 + j < N; j += 32) {
                const uint64_t o = (uint64_t)(m0 + q * 32) * ldc + c0 + j;
#pragma unroll 8
                for (uint32_t i = 0; i < 32; i++) {
                    const float y = stage[i * (slice + 1) + j];
                    if (i >= rows) continue;
                    if (DT == LTQ_F32) static_cast<float *>(out)[o + i * ldc] = y;
                    else static_cast<uint16_t *>(out)[o + i * ldc] = (uint16_t)token_bits<DT>(y);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8 && lane == 0 && *abort_flag) {
        // after a timeout copies may still be landing in this CTA's shared memory: hold it for a bounded 2 ms
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 2000000ull) __nanosleep(1000);
    }
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, SM_ACC * SM_MAX_BN);
    }
}

SmallPlan small_plan(uint64_t M, uint64_t N, uint64_t K, int sms)
{
    // Cost of a choice in cycles: rounds of CTAs x (launch and latencies, the epilogue per column, the exchange, and a CTA's copies at
    // 150 cycles per 16 KB and no less per copy).  Fitted to sweeps at 32, 77 and 128 tokens, K = 4096; microseconds at 77 tokens as
    // columns/split/lines: N = 1024: 64/1/2 8.6, 64/4/2 7.5, 32/1/4 6.7, 16/1/4 6.2, 128/4/2 10.4; N = 4096: 32/1/4 7.7, 64/1/2 8.8,
    // 128/4/2 12.1, 16/1/4 (two rounds) 12.8; N = 11008: 80/1/2 12.3, 128/1/2 14.3, 64/1/2 (two rounds) 19.1.
    SmallPlan best{0, 0, 0, 0};
    double least = 0;
    const uint64_t tm = (M + SM_M - 1) / SM_M, rows = M < SM_M ? (M + 7) / 8 * 8 : SM_M;
    for (uint32_t split = 1; split <= 4; split *= 2) {
        const uint32_t unit = split < 2 ? 16 : 8 * split;
        for (uint32_t bn = unit; bn <= SM_MAX_BN; bn += unit) {
            uint32_t lines = 1;
            if (K % SM_BK == 0) lines = (rows + bn) * SM_BK * 4 <= 40 * 1024 ? 4 : 2;
            const uint64_t blocks = (K + lines * SM_BK - 1) / (lines * SM_BK);
            if (split > 1 && blocks < 2 * split) continue;
            const uint64_t ctas = tm * ((N + bn - 1) / bn) * split, rounds = (ctas + sms - 1) / sms;
            const double a = (double)(lines * rows * SM_BK), b = (double)(lines * bn * SM_BK);
            const double step = ((a > 16384 ? a : 16384) + (b > 16384 ? b : 16384)) * 150 / 16384;
            const double cost = (double)rounds * (8000 + 60 * (double)(bn / split) + (split > 1 ? 2500 + 25 * (double)bn : 0) +
                                                  (double)((blocks + split - 1) / split) * step);
            if (best.split == 0 || cost < least) {
                best = SmallPlan{bn, split, lines, (uint32_t)rounds};
                least = cost;
            }
        }
    }
    return best;
}

int small_maps(const SmallPlan &p, const uint8_t *A, uint64_t M, uint64_t K, TcOperandMap *map_a, const uint8_t *B, uint64_t N, TcOperandMap *map_b)
{
    const int rows = (int)(M < SM_M ? (M + 7) / 8 * 8 : SM_M), lines = p.lines > 1 ? (int)p.lines : 0;
    int e = 0;
    if (lines) {
        e = tc_make_map_lines(map_a, A, M, K, rows, lines);
        if (e == 0 && !map_b->matches(B, N, K, (int)p.bn, lines)) e = tc_make_map_lines(map_b, B, N, K, (int)p.bn, lines);
    } else {
        e = tc_make_map(map_a, A, M, K, rows);
        if (e == 0 && !map_b->matches(B, N, K, (int)p.bn, 0)) e = tc_make_map(map_b, B, N, K, (int)p.bn);
    }
    return e;
}

namespace {

template <int OUT>
cudaError_t launch_small(const CUtensorMap &ma, const CUtensorMap &mb, const SmallPlan &p, uint64_t M, uint64_t N, uint64_t K, const Epilogue &epi,
                         void *out, uint32_t *status, cudaStream_t stream, bool early_weights)
{
    static bool attr_done[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!attr_done[dev]) {
        e = cudaFuncSetAttribute(gemm_small_kernel<OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SM_SMEM_LIMIT);
        if (e != cudaSuccess) return e;
        attr_done[dev] = true;
    }
    const SmallLayout l = small_layout(p, M);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((M + SM_M - 1) / SM_M) * ((N + p.bn - 1) / p.bn) * p.split));
    cfg.blockDim = dim3(SM_THREADS);
    cfg.dynamicSmemBytes = l.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (p.split > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = p.split;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        n++;
    }
    if (early_weights && chained_launches_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        n++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    e = cudaLaunchKernelEx(&cfg, gemm_small_kernel<OUT>, ma, mb, (uint32_t)M, (uint32_t)N, (uint32_t)K, p.bn, p.split, p.lines, l.a_rows, l.stages,
                           (uint32_t)(l.smem - (1024 + (size_t)(p.split - 1) * SM_M * (p.bn / p.split) * 4 + SM_MAX_BN * 16 + 256)) / 16 * 16, epi, out, status);
    count_launch();
    note_kernel("gemm_small_kernel<%s> (%u columns, K in %u, %u lines)", out_mode_name(OUT), p.bn, p.split, p.lines);
    return e;
}

}  // namespace

cudaError_t launch_gemm_small(const TcOperandMap &map_a, const TcOperandMap &map_b, const SmallPlan &p, uint64_t M, uint64_t N, uint64_t K,
                              const Epilogue &epi, void *out, uint32_t *status, cudaStream_t stream, bool early_weights)
{
    const CUtensorMap &ma = *reinterpret_cast<const CUtensorMap *>(map_a.opaque);
    const CUtensorMap &mb = *reinterpret_cast<const CUtensorMap *>(map_b.opaque);
    switch (epi.out_mode) {
        case OUT_TOKENS + LTQ_F32: return launch_small<OUT_TOKENS + LTQ_F32>(ma, mb, p, M, N, K, epi, out, status, stream, early_weights);
        case OUT_TOKENS + LTQ_F16: return launch_small<OUT_TOKENS + LTQ_F16>(ma, mb, p, M, N, K, epi, out, status, stream, early_weights);
        default: return launch_small<OUT_TOKENS + LTQ_BF16>(ma, mb, p, M, N, K, epi, out, status, stream, early_weights);
    }
}

}  // namespace ltq
