// Operators with quantisation parameters per row ("token") and per output column ("channel"): element types, the epilogue
// that turns raw uint8 x uint8 dot products into float / half / bfloat16 outputs, and the launchers of ltq_tokens.cu.
//
//   y[i,j] = float( sum_k (a[i,k] - za[i]) (w[j,k] - zw[j]) ) * sa[i] * sw[j] (+ bias[j])
//
// The sum is exact in 32-bit integers (K <= TOKENS_MAX_K):
//   raw + za[i] * (K*zw[j] - wsum[j]) - zw[j] * asum[i]
// so an element costs two integer multiply-adds, one conversion, two multiplications and one addition.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ltq_common.cuh"

namespace ltq {

constexpr int OUT_TOKENS = 3;   // Epilogue::out_mode and the kernels' OUT argument: OUT_TOKENS + ltq_dtype
__host__ __device__ constexpr bool out_is_tokens(int out) { return out >= OUT_TOKENS; }
inline uint64_t dtype_size(int dtype) { return dtype == LTQ_F32 ? 4 : 2; }
inline const char *dtype_name(int dtype) { return dtype == LTQ_F32 ? "f32" : (dtype == LTQ_F16 ? "f16" : "bf16"); }
inline bool dtype_ok(int dtype) { return dtype == LTQ_F32 || dtype == LTQ_F16 || dtype == LTQ_BF16; }

// |a - za| and |w - zw| reach 255 when a zero point sits at an end of the range: up to this many terms fit an int32.
constexpr uint64_t TOKENS_MAX_K = 0x7FFFFFFFull / (255 * 255);

struct TokenRow {
    int32_t za;
    uint32_t neg_asum;
    float sa;
};
__device__ __forceinline__ TokenRow token_row(const Epilogue &e, uint64_t i)
{
    const ltq_qparams qp = e.qp_rows[i];
    return TokenRow{(int32_t)qp.zero_point, (uint32_t)(-e.asum[i]), qp.scale};
}
// Column part, 16 bytes: K*zw - wsum, zw, sw, bias.
__device__ __forceinline__ uint4 token_col(const Epilogue &e, uint64_t j)
{
    const ltq_qparams qp = e.qp_cols[j];
    return make_uint4(e.K * (uint32_t)qp.zero_point - (uint32_t)e.bsum[j], (uint32_t)qp.zero_point, __float_as_uint(qp.scale),
                      e.fbias ? __float_as_uint(e.fbias[j]) : 0u);
}
// (adding a bias of +0 to a product of -0 gives +0: the two compare equal)
__device__ __forceinline__ float token_value(uint32_t raw, const TokenRow &r, const uint4 &c, bool relu)
{
    const int32_t acc = (int32_t)(raw + (uint32_t)r.za * c.x + c.y * r.neg_asum);
    const float y = __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(acc), r.sa), __uint_as_float(c.z)), __uint_as_float(c.w));
    return relu && y < 0.f ? 0.f : y;   // (a NaN stays: a token whose input was not finite shows in its whole row)
}

// Rounds to the output type (nearest even; beyond half's range an infinity), the bits in the low half of a word.
template <int DT>
__device__ __forceinline__ uint32_t token_bits(float y)
{
    if (DT == LTQ_F32) return __float_as_uint(y);
    if (DT == LTQ_F16) return (uint32_t)__half_as_ushort(__float2half_rn(y));
    return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(y));
}
template <int DT>
__device__ __forceinline__ uint32_t token_bits2(float lo, float hi)
{
    if (DT == LTQ_F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// One chunk of W consecutive accumulator columns of one row, `valid` of them inside the matrix: converted and stored at
// element offset `off` of `out`.  16-byte stores when vec_ok (row starts and the chunk are 16-byte aligned).
template <int OUT, int W>
__device__ __forceinline__ void token_chunk(const uint32_t (&v)[W], const TokenRow &r, const uint4 *col_smem, bool relu, void *out,
                                            uint64_t off, bool vec_ok, int valid)
{
    constexpr int DT = OUT - OUT_TOKENS, ESZ = DT == LTQ_F32 ? 4 : 2, PER16 = 16 / ESZ;
    uint8_t *dst = static_cast<uint8_t *>(out) + off * ESZ;
#pragma unroll
    for (int g = 0; g < W / PER16; g++) {
        float y[PER16];
#pragma unroll
        for (int k = 0; k < PER16; k++) y[k] = token_value(v[g * PER16 + k], r, col_smem[g * PER16 + k], relu);
        if (vec_ok && (g + 1) * PER16 <= valid) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; k++) w[k] = DT == LTQ_F32 ? __float_as_uint(y[k]) : token_bits2<DT>(y[2 * k % PER16], y[(2 * k + 1) % PER16]);
            *reinterpret_cast<uint4 *>(dst + 16 * g) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int k = 0; k < PER16; k++) {
                if (g * PER16 + k >= valid) continue;
                if (DT == LTQ_F32) reinterpret_cast<float *>(dst)[g * PER16 + k] = y[k];
                else reinterpret_cast<uint16_t *>(dst)[g * PER16 + k] = (uint16_t)token_bits<DT>(y[k]);
            }
        }
    }
}

// Output rows that do not start on 16-byte boundaries.  In the accumulator layout a thread owns a row, and storing it element by
// element makes every store instruction touch 32 rows (4099 columns of 1024 rows: 48 us against 17 us for 4096).  A warp parks 16
// columns of its 32 rows in shared memory instead and writes them row by row, two rows at a time, lanes side by side.
struct TokenStage {
    static constexpr int PITCH = 17;   // odd: neither side meets a bank twice
    static constexpr int BYTES_PER_WARP = 32 * PITCH * 4;

    // W accumulator columns of the warp's 32 rows, `valid` of them inside the matrix, element (0, 0) at offset `off`; the first `rows`
    // rows exist.  Called by the whole warp.
    template <int OUT, int W>
    static __device__ __forceinline__ void chunk(float *stage, const uint32_t (&v)[W], const TokenRow &r, const uint4 *col_smem, bool relu,
                                                 void *out, uint64_t off, uint64_t ldc, int rows, int valid)
    {
        constexpr int DT = OUT - OUT_TOKENS;
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int b = 0; b < W; b += 16) {
#pragma unroll
            for (int k = 0; k < 16; k++) stage[lane * PITCH + k] = token_value(v[b + k], r, col_smem[b + k], relu);
            __syncwarp();
            const int c = lane & 15;
#pragma unroll 4
            for (int i = lane >> 4; i < 32; i += 2) {
                const float y = stage[i * PITCH + c];
                if (i < rows && b + c < valid) {
                    const uint64_t o = off + (uint64_t)i * ldc + b + c;
                    if (DT == LTQ_F32) static_cast<float *>(out)[o] = y;
                    else static_cast<uint16_t *>(out)[o] = (uint16_t)token_bits<DT>(y);
                }
            }
            __syncwarp();
        }
    }
};

// x [rows, cols] of `dtype`, rows ld_x elements apart -> q uint8, rows q_pitch bytes apart (columns [cols, q_pitch) become 0),
// qp [rows], sums [rows] (or nullptr).
cudaError_t launch_quantize_tokens(const void *x, int dtype, uint64_t rows, uint64_t cols, uint64_t ld_x, uint8_t *q, uint64_t q_pitch,
                                   ltq_qparams *qp, int32_t *sums, int sms, cudaStream_t stream);
cudaError_t launch_dequantize_tokens(void *x, int dtype, uint64_t ld_x, const uint8_t *q, const ltq_qparams *qp, uint64_t rows,
                                     uint64_t cols, int sms, cudaStream_t stream);

}  // namespace ltq
