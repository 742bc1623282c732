// Quantise / dequantise with parameters per row ("token"): the framework's GetMinMax -> ComputeQuantizationParams -> Quantize
// (l-ten/utils.cpp:198-286) applied to every row of a float / half / bfloat16 matrix on its own, in one pass.
//
//   lo = min(0, min x), hi = max(0, max x), scale = (hi - lo) / 255, zero = round(0 - lo / scale),
//   q = Quantize(x, {scale, zero})                                              (every step rounded to float, as there)
//
// What the per-tensor functions leave undefined is defined here, because a batch of tokens meets it: a row of zeros (or of
// values so small that the scale would be subnormal) gets the scale 2^-126; a row whose range overflows gets
// hi / 255 - lo / 255; a row that holds an infinity or a NaN gets the scale NaN and codes 0, so that whatever is computed
// from it is NaN in that row and nowhere else.
#include "ltq_ptx.cuh"
#include "ltq_quant.cuh"
#include "ltq_tokens.cuh"

namespace ltq {

namespace {

constexpr int CTA = 256;
constexpr float SMALLEST_SCALE = 1.17549435e-38f;   // 2^-126

struct RowParams {
    float scale, zpf, inv;
    bool finite;
};
__device__ __forceinline__ RowParams row_params(float lo, float hi)
{
    RowParams p;
    p.finite = fabsf(lo) < INFINITY && fabsf(hi) < INFINITY;   // false for NaN
    float scale = __fdiv_rn(__fsub_rn(hi, lo), 255.f);
    if (scale == INFINITY) scale = __fsub_rn(__fdiv_rn(hi, 255.f), __fdiv_rn(lo, 255.f));
    scale = fmaxf(scale, SMALLEST_SCALE);
    p.scale = p.finite ? scale : __int_as_float(0x7FC00000);
    p.zpf = p.finite ? roundf(__fsub_rn(0.f, __fdiv_rn(lo, scale))) : 0.f;
    p.inv = quant_screen_inv(scale);
    return p;
}
__device__ __forceinline__ ltq_qparams stored_params(const RowParams &p)
{
    ltq_qparams qp;
    qp.scale = p.scale;
    qp.zero_point = (uint8_t)(int)p.zpf;
    return qp;
}
// The 8 bytes at once (the padding bytes of the struct become 0).
__device__ __forceinline__ void put_params(ltq_qparams *dst, const RowParams &p)
{
    if (((uintptr_t)dst & 7) == 0) *reinterpret_cast<uint2 *>(dst) = make_uint2(__float_as_uint(p.scale), (uint32_t)(int)p.zpf);
    else *dst = stored_params(p);
}

__device__ __forceinline__ float min_nan(float a, float b)
{
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Per element type: 16-byte vectors, a running {min, max} that a NaN sticks to (starting from 0: the range holds it), and
// the conversion of four neighbours to float.
template <int DT>
struct Elem;
template <>
struct Elem<LTQ_F32> {
    using T = float;
    static constexpr int PER16 = 4;
    struct Range {
        float lo = 0.f, hi = 0.f;
        __device__ __forceinline__ void take(const uint4 &v)
        {
            const float a = __uint_as_float(v.x), b = __uint_as_float(v.y), c = __uint_as_float(v.z), d = __uint_as_float(v.w);
            lo = min_nan(min_nan(lo, min_nan(a, b)), min_nan(c, d));
            hi = max_nan(max_nan(hi, max_nan(a, b)), max_nan(c, d));
        }
        __device__ __forceinline__ float low() const { return lo; }
        __device__ __forceinline__ float high() const { return hi; }
    };
    static __device__ __forceinline__ float4 four(const uint4 &v, int)
    {
        return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
    }
    static __device__ __forceinline__ float one(float x) { return x; }
    static __device__ __forceinline__ float out(float v) { return v; }
};
template <>
struct Elem<LTQ_F16> {
    using T = __half;
    static constexpr int PER16 = 8;
    struct Range {
        __half2 lo = __float2half2_rn(0.f), hi = lo;
        __device__ __forceinline__ void take(const uint4 &v)
        {
            const __half2 *p = reinterpret_cast<const __half2 *>(&v);
            lo = __hmin2_nan(__hmin2_nan(lo, __hmin2_nan(p[0], p[1])), __hmin2_nan(p[2], p[3]));
            hi = __hmax2_nan(__hmax2_nan(hi, __hmax2_nan(p[0], p[1])), __hmax2_nan(p[2], p[3]));
        }
        __device__ __forceinline__ float low() const { return min_nan(__low2float(lo), __high2float(lo)); }
        __device__ __forceinline__ float high() const { return max_nan(__low2float(hi), __high2float(hi)); }
    };
    static __device__ __forceinline__ float4 four(const uint4 &v, int h)
    {
        const __half2 *p = reinterpret_cast<const __half2 *>(&v) + 2 * h;
        const float2 a = __half22float2(p[0]), b = __half22float2(p[1]);
        return make_float4(a.x, a.y, b.x, b.y);
    }
    static __device__ __forceinline__ float one(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half out(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<LTQ_BF16> {
    using T = __nv_bfloat16;
    static constexpr int PER16 = 8;
    struct Range {
        __nv_bfloat162 lo = __float2bfloat162_rn(0.f), hi = lo;
        __device__ __forceinline__ void take(const uint4 &v)
        {
            const __nv_bfloat162 *p = reinterpret_cast<const __nv_bfloat162 *>(&v);
            lo = __hmin2_nan(__hmin2_nan(lo, __hmin2_nan(p[0], p[1])), __hmin2_nan(p[2], p[3]));
            hi = __hmax2_nan(__hmax2_nan(hi, __hmax2_nan(p[0], p[1])), __hmax2_nan(p[2], p[3]));
        }
        __device__ __forceinline__ float low() const { return min_nan(__low2float(lo), __high2float(lo)); }
        __device__ __forceinline__ float high() const { return max_nan(__low2float(hi), __high2float(hi)); }
    };
    static __device__ __forceinline__ float4 four(const uint4 &v, int h)
    {
        const uint32_t a = h ? v.z : v.x, b = h ? v.w : v.y;   // a bfloat16 is the upper half of a float
        return make_float4(__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u), __uint_as_float(b << 16),
                           __uint_as_float(b & 0xFFFF0000u));
    }
    static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 out(float v) { return __float2bfloat16_rn(v); }
};

}  // namespace

// TPR threads share a row (32: a warp per row, 256: the CTA) and keep it in registers, NV 16-byte vectors each, between the
// reduction and the quantisation: every input byte is read once.  Rows start 16-byte aligned (x) and 8-byte aligned (q).
// Bound by HBM (cols * (element + 1) + 12 bytes per row).
template <int DT, int TPR, int NV>
__global__ void __launch_bounds__(CTA)
quantize_tokens_kernel(const typename Elem<DT>::T *__restrict__ x, uint64_t rows, uint32_t cols, uint64_t ld_x, uint8_t *__restrict__ q,
                       uint32_t q_pitch, ltq_qparams *__restrict__ qp, int32_t *__restrict__ sums)
{
    griddep_launch_dependents();
    griddep_wait();
    using E = Elem<DT>;
    constexpr int PER16 = E::PER16, ROWS = CTA / TPR;
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const uint32_t nvec = cols / PER16;
    __shared__ float s_lo[8], s_hi[8];
    __shared__ RowParams s_par;
    __shared__ int32_t s_sum[8];
    for (uint64_t row = (uint64_t)blockIdx.x * ROWS + sub; row < rows; row += (uint64_t)gridDim.x * ROWS) {
        const uint4 *xv = reinterpret_cast<const uint4 *>(x + row * ld_x);
        uint4 v[NV];
        typename E::Range range;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const uint32_t i = (uint32_t)j * TPR + lane;
            v[j] = i < nvec ? __ldcs(xv + i) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < NV; j++) range.take(v[j]);
        float lo = range.low(), hi = range.high();
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            lo = min_nan(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
            hi = max_nan(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
        }
        RowParams p;
        if (TPR == 32) {
            p = row_params(lo, hi);
        } else {
            const int w = threadIdx.x >> 5;
            if ((threadIdx.x & 31) == 0) {
                s_lo[w] = lo;
                s_hi[w] = hi;
            }
            __syncthreads();
            if (w == 0) {   // one warp derives the parameters (three divisions); the others wait for them
                lo = s_lo[lane & 7];
                hi = s_hi[lane & 7];
#pragma unroll
                for (int o = 4; o; o >>= 1) {
                    lo = min_nan(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
                    hi = max_nan(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
                }
                p = row_params(lo, hi);
                if (lane == 0) s_par = p;
            }
            __syncthreads();
            p = s_par;
        }
        uint8_t *qr = q + row * q_pitch;
        uint32_t s = 0;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const uint32_t i = (uint32_t)j * TPR + lane;
            if (i < nvec) {
                uint32_t a = p.finite ? quant4_u8(E::four(v[j], 0), p.scale, p.zpf, p.inv) : 0u;
                s = __dp4a(a, 0x01010101u, s);
                if (PER16 == 8) {
                    const uint32_t b = p.finite ? quant4_u8(E::four(v[j], 1), p.scale, p.zpf, p.inv) : 0u;
                    s = __dp4a(b, 0x01010101u, s);
                    reinterpret_cast<uint2 *>(qr)[i] = make_uint2(a, b);
                } else {
                    reinterpret_cast<uint32_t *>(qr)[i] = a;
                }
            }
        }
        for (uint32_t i = cols + lane; i < q_pitch; i += TPR) qr[i] = 0;
        s = __reduce_add_sync(0xFFFFFFFFu, s);
        if (TPR == 32) {
            if (lane == 0) {
                put_params(qp + row, p);
                if (sums) sums[row] = (int32_t)s;
            }
        } else {
            if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = (int32_t)s;
            __syncthreads();
            if (threadIdx.x == 0) {
                put_params(qp + row, p);
                int32_t t = 0;
                for (int w = 0; w < 8; w++) t += s_sum[w];
                if (sums) sums[row] = t;
            }
        }
    }
}

// Any width, pitch and alignment: element by element, the row read twice (the second time out of L1 / L2).
template <int DT, int TPR>
__global__ void __launch_bounds__(CTA)
quantize_tokens_any_kernel(const typename Elem<DT>::T *__restrict__ x, uint64_t rows, uint64_t cols, uint64_t ld_x, uint8_t *__restrict__ q,
                           uint64_t q_pitch, ltq_qparams *__restrict__ qp, int32_t *__restrict__ sums)
{
    griddep_launch_dependents();
    griddep_wait();
    using E = Elem<DT>;
    constexpr int ROWS = CTA / TPR;
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    __shared__ float s_lo[8], s_hi[8];
    __shared__ int32_t s_sum[8];
    for (uint64_t row = (uint64_t)blockIdx.x * ROWS + sub; row < rows; row += (uint64_t)gridDim.x * ROWS) {
        const typename E::T *xr = x + row * ld_x;
        float lo = 0.f, hi = 0.f;
        for (uint64_t i = lane; i < cols; i += TPR) {
            const float v = E::one(xr[i]);
            lo = min_nan(lo, v);
            hi = max_nan(hi, v);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            lo = min_nan(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
            hi = max_nan(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
        }
        if (TPR != 32) {
            if ((threadIdx.x & 31) == 0) {
                s_lo[threadIdx.x >> 5] = lo;
                s_hi[threadIdx.x >> 5] = hi;
            }
            __syncthreads();
            lo = s_lo[0];
            hi = s_hi[0];
            for (int w = 1; w < 8; w++) {
                lo = min_nan(lo, s_lo[w]);
                hi = max_nan(hi, s_hi[w]);
            }
        }
        const RowParams p = row_params(lo, hi);
        uint8_t *qr = q + row * q_pitch;
        uint32_t s = 0;
        for (uint64_t i = lane; i < cols; i += TPR) {
            const uint32_t a = p.finite ? quant_u8(E::one(xr[i]), p.scale, p.zpf, p.inv) : 0u;
            s += a;
            qr[i] = (uint8_t)a;
        }
        for (uint64_t i = cols + lane; i < q_pitch; i += TPR) qr[i] = 0;
        s = __reduce_add_sync(0xFFFFFFFFu, s);
        if (TPR == 32) {
            if (lane == 0) {
                put_params(qp + row, p);
                if (sums) sums[row] = (int32_t)s;
            }
        } else {
            if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = (int32_t)s;
            __syncthreads();
            if (threadIdx.x == 0) {
                put_params(qp + row, p);
                int32_t t = 0;
                for (int w = 0; w < 8; w++) t += s_sum[w];
                if (sums) sums[row] = t;
            }
        }
    }
}

namespace {

template <int DT, int TPR, int NV>
cudaError_t launch_vec(const void *x, uint64_t rows, uint64_t cols, uint64_t ld_x, uint8_t *q, uint64_t q_pitch, ltq_qparams *qp,
                       int32_t *sums, int sms, cudaStream_t stream)
{
    const uint64_t per = CTA / TPR, want = (rows + per - 1) / per, cap = (uint64_t)sms * 8;
    return launch_chained(quantize_tokens_kernel<DT, TPR, NV>, dim3((unsigned)(want < cap ? want : cap)), dim3(CTA), 0, stream,
                          static_cast<const typename Elem<DT>::T *>(x), rows, (uint32_t)cols, ld_x, q, (uint32_t)q_pitch, qp, sums);
}

template <int DT>
cudaError_t launch_quantize_dt(const void *x, uint64_t rows, uint64_t cols, uint64_t ld_x, uint8_t *q, uint64_t q_pitch, ltq_qparams *qp,
                               int32_t *sums, int sms, cudaStream_t stream)
{
    constexpr uint64_t P = Elem<DT>::PER16;
    const bool aligned = cols % P == 0 && ld_x % P == 0 && q_pitch % P == 0 && (((uintptr_t)x & 15) == 0) && (((uintptr_t)q & (P - 1)) == 0);
    if (aligned && cols <= 256 * 8 * P) {
        if (cols <= 32 * 4 * P) return launch_vec<DT, 32, 4>(x, rows, cols, ld_x, q, q_pitch, qp, sums, sms, stream);
        if (cols <= 256 * 1 * P) return launch_vec<DT, 256, 1>(x, rows, cols, ld_x, q, q_pitch, qp, sums, sms, stream);
        if (cols <= 256 * 2 * P) return launch_vec<DT, 256, 2>(x, rows, cols, ld_x, q, q_pitch, qp, sums, sms, stream);
        if (cols <= 256 * 4 * P) return launch_vec<DT, 256, 4>(x, rows, cols, ld_x, q, q_pitch, qp, sums, sms, stream);
        return launch_vec<DT, 256, 8>(x, rows, cols, ld_x, q, q_pitch, qp, sums, sms, stream);
    }
    const uint64_t cap = (uint64_t)sms * 8;
    if (cols <= 1024) {
        const uint64_t want = (rows + 7) / 8;
        return launch_chained(quantize_tokens_any_kernel<DT, 32>, dim3((unsigned)(want < cap ? want : cap)), dim3(CTA), 0, stream,
                              static_cast<const typename Elem<DT>::T *>(x), rows, cols, ld_x, q, q_pitch, qp, sums);
    }
    return launch_chained(quantize_tokens_any_kernel<DT, 256>, dim3((unsigned)(rows < cap ? rows : cap)), dim3(CTA), 0, stream,
                          static_cast<const typename Elem<DT>::T *>(x), rows, cols, ld_x, q, q_pitch, qp, sums);
}

}  // namespace

cudaError_t launch_quantize_tokens(const void *x, int dtype, uint64_t rows, uint64_t cols, uint64_t ld_x, uint8_t *q, uint64_t q_pitch,
                                   ltq_qparams *qp, int32_t *sums, int sms, cudaStream_t stream)
{
    count_launch();
    if (dtype == LTQ_F32) return launch_quantize_dt<LTQ_F32>(x, rows, cols, ld_x, q, q_pitch, qp, sums, sms, stream);
    if (dtype == LTQ_F16) return launch_quantize_dt<LTQ_F16>(x, rows, cols, ld_x, q, q_pitch, qp, sums, sms, stream);
    return launch_quantize_dt<LTQ_BF16>(x, rows, cols, ld_x, q, q_pitch, qp, sums, sms, stream);
}

// ---- dequantise ---------------------------------------------------------------------------------------------------------
// value = scale * (q - zero), rounded to float and then to the output type.  A warp takes 32 x 16 codes of one row at a time.
template <int DT>
__global__ void __launch_bounds__(CTA)
dequantize_tokens_kernel(typename Elem<DT>::T *__restrict__ x, uint64_t ld_x, const uint8_t *__restrict__ q, const ltq_qparams *__restrict__ qp,
                         uint64_t rows, uint64_t cols, uint32_t pieces, bool vec)
{
    griddep_launch_dependents();
    griddep_wait();
    using E = Elem<DT>;
    const int lane = threadIdx.x & 31;
    const uint64_t nwarps = ((uint64_t)gridDim.x * CTA) >> 5;
    for (uint64_t w = ((uint64_t)blockIdx.x * CTA + threadIdx.x) >> 5; w < rows * pieces; w += nwarps) {
        const uint64_t row = w / pieces, c0 = (w - row * pieces) * 512;
        const float scale = qp[row].scale;
        const int zp = (int)qp[row].zero_point;
        const uint8_t *qr = q + row * cols;
        typename E::T *xr = x + row * ld_x;
        if (vec) {
            const uint64_t c = c0 + (uint64_t)lane * 16;
            if (c >= cols) continue;
            const uint4 p = __ldcs(reinterpret_cast<const uint4 *>(qr + c));
            const uint32_t word[4] = {p.x, p.y, p.z, p.w};
            uint32_t res[16 * sizeof(typename E::T) / 4];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float a = __fmul_rn(scale, (float)((int)((word[i / 4] >> (8 * (i % 4))) & 0xFF) - zp));
                const float b = __fmul_rn(scale, (float)((int)((word[i / 4] >> (8 * (i % 4) + 8)) & 0xFF) - zp));
                if (DT == LTQ_F32) {
                    res[i] = __float_as_uint(a);
                    res[i + 1] = __float_as_uint(b);
                } else {
                    res[i / 2] = token_bits2<DT>(a, b);
                }
            }
            uint4 *dst = reinterpret_cast<uint4 *>(xr + c);
#pragma unroll
            for (int i = 0; i < (int)sizeof(typename E::T); i++) dst[i] = make_uint4(res[4 * i], res[4 * i + 1], res[4 * i + 2], res[4 * i + 3]);
        } else {
            for (uint64_t c = c0 + lane; c < c0 + 512 && c < cols; c += 32) xr[c] = E::out(__fmul_rn(scale, (float)((int)qr[c] - zp)));
        }
    }
}

namespace {

template <int DT>
cudaError_t launch_dequantize_dt(void *x, uint64_t ld_x, const uint8_t *q, const ltq_qparams *qp, uint64_t rows, uint64_t cols, int sms,
                                 cudaStream_t stream)
{
    const uint64_t pieces = (cols + 511) / 512, want = (rows * pieces + 7) / 8, cap = (uint64_t)sms * 8;
    const bool vec = cols % 16 == 0 && ld_x % 8 == 0 && (ld_x * sizeof(typename Elem<DT>::T)) % 16 == 0 && (((uintptr_t)x | (uintptr_t)q) & 15) == 0;
    return launch_chained(dequantize_tokens_kernel<DT>, dim3((unsigned)(want < cap ? want : cap)), dim3(CTA), 0, stream,
                          static_cast<typename Elem<DT>::T *>(x), ld_x, q, qp, rows, cols, (uint32_t)pieces, vec);
}

}  // namespace

cudaError_t launch_dequantize_tokens(void *x, int dtype, uint64_t ld_x, const uint8_t *q, const ltq_qparams *qp, uint64_t rows, uint64_t cols,
                                     int sms, cudaStream_t stream)
{
    count_launch();
    if (dtype == LTQ_F32) return launch_dequantize_dt<LTQ_F32>(x, ld_x, q, qp, rows, cols, sms, stream);
    if (dtype == LTQ_F16) return launch_dequantize_dt<LTQ_F16>(x, ld_x, q, qp, rows, cols, sms, stream);
    return launch_dequantize_dt<LTQ_BF16>(x, ld_x, q, qp, rows, cols, sms, stream);
}

}  // namespace ltq
