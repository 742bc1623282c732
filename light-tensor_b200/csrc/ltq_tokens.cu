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
    p.inv = quant_row_inv(scale);
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

namespace {

// {min, max} over the lanes of a warp.
__device__ __forceinline__ void warp_range(float &lo, float &hi)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
    }
}

// Parameters of a row that TPR threads share: every warp's range in, the row's parameters out.  (TPR > 32: TPR is the CTA.)
template <int TPR>
__device__ __forceinline__ RowParams shared_params(float lo, float hi)
{
    warp_range(lo, hi);
    if (TPR == 32) return row_params(lo, hi);
    __shared__ float s_lo[TPR / 32], s_hi[TPR / 32];
    __shared__ RowParams s_par;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if (lane == 0) {
        s_lo[w] = lo;
        s_hi[w] = hi;
    }
    __syncthreads();
    if (w == 0) {   // one warp derives the parameters (three divisions); the others wait for them
        lo = s_lo[lane % (TPR / 32)];
        hi = s_hi[lane % (TPR / 32)];
        warp_range(lo, hi);
        if (lane == 0) s_par = row_params(lo, hi);
    }
    __syncthreads();
    return s_par;
}

// Writes the row's parameters and code sum; `s`: this thread's part.
template <int TPR>
__device__ __forceinline__ void finish_row(uint64_t row, const RowParams &p, uint32_t s, ltq_qparams *qp, int32_t *sums)
{
    s = __reduce_add_sync(0xFFFFFFFFu, s);
    const int lane = threadIdx.x & 31;
    if (TPR > 32) {
        __shared__ uint32_t s_sum[TPR / 32];
        if (lane == 0) s_sum[threadIdx.x >> 5] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            s = 0;
#pragma unroll
            for (int w = 0; w < TPR / 32; w++) s += s_sum[w];
        }
        if (threadIdx.x >= 32) return;
    }
    if (lane == 0) {
        put_params(qp + row, p);
        if (sums) sums[row] = (int32_t)s;
    }
}

__host__ __device__ constexpr int cta_size(int tpr) { return tpr == 32 ? 128 : tpr; }

}  // namespace

// TPR threads share a row (32: a warp, with four warps in a CTA; otherwise the CTA) and keep it in registers, NV 16-byte vectors
// each, between the reduction and the quantisation: every input byte is read once.  Rows start 16-byte aligned (x) and 8-byte
// (float: 4-byte) aligned (q).  Bound by HBM, cols * (element + 1) + 12 bytes per row, and at 16-bit types nearly by issue
// (about ten instructions per element).  Measured, 16384 x 8192 bfloat16 (floor 62 us): 32 / 64 / 128 / 256 threads on a row 149 /
// 94 / 78 / 88 us; 8192 x 8192 float (52 us): 69 / 69 / 57 / 54; 4096 x 4096 bfloat16: 16 / 12 / 13 / 17.
template <int DT, int TPR, int NV>
__global__ void __launch_bounds__(cta_size(TPR))
quantize_tokens_kernel(const typename Elem<DT>::T *__restrict__ x, uint64_t rows, uint32_t cols, uint64_t ld_x, uint8_t *__restrict__ q,
                       uint32_t q_pitch, ltq_qparams *__restrict__ qp, int32_t *__restrict__ sums)
{
    griddep_launch_dependents();
    griddep_wait();
    using E = Elem<DT>;
    constexpr int PER16 = E::PER16, ROWS = cta_size(TPR) / TPR;
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const uint32_t nvec = cols / PER16;
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
        const RowParams p = shared_params<TPR>(range.low(), range.high());
        uint8_t *qr = q + row * q_pitch;
        uint32_t s = 0;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const uint32_t i = (uint32_t)j * TPR + lane;
            if (i < nvec) {
                const uint32_t a = p.finite ? quant4_row(E::four(v[j], 0), p.scale, p.zpf, p.inv) : 0u;
                s = __dp4a(a, 0x01010101u, s);
                if (PER16 == 8) {
                    const uint32_t b = p.finite ? quant4_row(E::four(v[j], 1), p.scale, p.zpf, p.inv) : 0u;
                    s = __dp4a(b, 0x01010101u, s);
                    reinterpret_cast<uint2 *>(qr)[i] = make_uint2(a, b);
                } else {
                    reinterpret_cast<uint32_t *>(qr)[i] = a;
                }
            }
        }
        for (uint32_t i = cols + lane; i < q_pitch; i += TPR) qr[i] = 0;
        finish_row<TPR>(row, p, s, qp, sums);
    }
}

// Rows that do not start on vector boundaries: the same with NE single elements per thread.
template <int DT, int TPR, int NE>
__global__ void __launch_bounds__(cta_size(TPR))
quantize_tokens_single_kernel(const typename Elem<DT>::T *__restrict__ x, uint64_t rows, uint32_t cols, uint64_t ld_x, uint8_t *__restrict__ q,
                              uint32_t q_pitch, ltq_qparams *__restrict__ qp, int32_t *__restrict__ sums)
{
    griddep_launch_dependents();
    griddep_wait();
    using E = Elem<DT>;
    constexpr int ROWS = cta_size(TPR) / TPR;
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    for (uint64_t row = (uint64_t)blockIdx.x * ROWS + sub; row < rows; row += (uint64_t)gridDim.x * ROWS) {
        const typename E::T *xr = x + row * ld_x;
        float v[NE], lo = 0.f, hi = 0.f;
#pragma unroll
        for (int j = 0; j < NE; j++) {
            const uint32_t i = (uint32_t)j * TPR + lane;
            v[j] = i < cols ? E::one(xr[i]) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < NE; j++) {
            lo = min_nan(lo, v[j]);
            hi = max_nan(hi, v[j]);
        }
        const RowParams p = shared_params<TPR>(lo, hi);
        uint8_t *qr = q + row * q_pitch;
        uint32_t s = 0;
#pragma unroll
        for (int j = 0; j < NE; j += 4) {
            const uint32_t w = p.finite ? quant4_row(make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]), p.scale, p.zpf, p.inv) : 0u;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t i = (uint32_t)(j + k) * TPR + lane, c = w >> (8 * k) & 0xFF;
                if (i < cols) {
                    s += c;
                    qr[i] = (uint8_t)c;
                }
            }
        }
        for (uint32_t i = cols + lane; i < q_pitch; i += TPR) qr[i] = 0;
        finish_row<TPR>(row, p, s, qp, sums);
    }
}

// Any width: element by element, the row read twice (the second time out of L2).
template <int DT>
__global__ void __launch_bounds__(CTA)
quantize_tokens_any_kernel(const typename Elem<DT>::T *__restrict__ x, uint64_t rows, uint64_t cols, uint64_t ld_x, uint8_t *__restrict__ q,
                           uint64_t q_pitch, ltq_qparams *__restrict__ qp, int32_t *__restrict__ sums)
{
    griddep_launch_dependents();
    griddep_wait();
    using E = Elem<DT>;
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const typename E::T *xr = x + row * ld_x;
        float lo = 0.f, hi = 0.f;
        for (uint64_t i = threadIdx.x; i < cols; i += CTA) {
            const float v = E::one(xr[i]);
            lo = min_nan(lo, v);
            hi = max_nan(hi, v);
        }
        const RowParams p = shared_params<CTA>(lo, hi);
        uint8_t *qr = q + row * q_pitch;
        uint32_t s = 0;
        for (uint64_t i = threadIdx.x; i < cols; i += CTA) {
            const uint32_t a = p.finite ? quant4_row(make_float4(E::one(xr[i]), 0.f, 0.f, 0.f), p.scale, p.zpf, p.inv) & 0xFF : 0u;
            s += a;
            qr[i] = (uint8_t)a;
        }
        for (uint64_t i = cols + threadIdx.x; i < q_pitch; i += CTA) qr[i] = 0;
        finish_row<CTA>(row, p, s, qp, sums);
    }
}

namespace {

struct RowCall {
    const void *x;
    uint64_t rows, cols, ld_x;
    uint8_t *q;
    uint64_t q_pitch;
    ltq_qparams *qp;
    int32_t *sums;
    int sms;
    cudaStream_t stream;
};
template <int DT, int TPR, typename Kernel>
cudaError_t launch_rows(Kernel kernel, const RowCall &c)
{
    const uint64_t per = cta_size(TPR) / TPR, want = (c.rows + per - 1) / per, cap = (uint64_t)c.sms * (2048 / cta_size(TPR));
    return launch_chained(kernel, dim3((unsigned)(want < cap ? want : cap)), dim3(cta_size(TPR)), 0, c.stream,
                          static_cast<const typename Elem<DT>::T *>(c.x), c.rows, (uint32_t)c.cols, c.ld_x, c.q, (uint32_t)c.q_pitch, c.qp, c.sums);
}

template <int DT>
cudaError_t launch_quantize_dt(const RowCall &c)
{
    constexpr uint64_t P = Elem<DT>::PER16;
    const bool aligned = c.cols % P == 0 && c.ld_x % P == 0 && c.q_pitch % P == 0 && (((uintptr_t)c.x & 15) == 0) && (((uintptr_t)c.q & (P - 1)) == 0);
    const uint64_t vecs = c.cols / P;
    if (aligned) {
        if (vecs <= 32 * 4) return launch_rows<DT, 32>(quantize_tokens_kernel<DT, 32, 4>, c);
        if (c.rows < (uint64_t)c.sms) {   // fewer rows than SMs: as many threads on a row as there are
            if (vecs <= 256 * 1) return launch_rows<DT, 256>(quantize_tokens_kernel<DT, 256, 1>, c);
            if (vecs <= 256 * 2) return launch_rows<DT, 256>(quantize_tokens_kernel<DT, 256, 2>, c);
            if (vecs <= 256 * 4) return launch_rows<DT, 256>(quantize_tokens_kernel<DT, 256, 4>, c);
        }
        if (vecs <= 128 * 2) return launch_rows<DT, 128>(quantize_tokens_kernel<DT, 128, 2>, c);
        if (vecs <= 128 * 4) return launch_rows<DT, 128>(quantize_tokens_kernel<DT, 128, 4>, c);
        if (vecs <= 128 * 8) return launch_rows<DT, 128>(quantize_tokens_kernel<DT, 128, 8>, c);
        if (vecs <= 256 * 8) return launch_rows<DT, 256>(quantize_tokens_kernel<DT, 256, 8>, c);
        if (vecs <= 256 * 16) return launch_rows<DT, 256>(quantize_tokens_kernel<DT, 256, 16>, c);
    } else {
        if (c.cols <= 32 * 8) return launch_rows<DT, 32>(quantize_tokens_single_kernel<DT, 32, 8>, c);
        if (c.cols <= 128 * 8) return launch_rows<DT, 128>(quantize_tokens_single_kernel<DT, 128, 8>, c);
        if (c.cols <= 256 * 16) return launch_rows<DT, 256>(quantize_tokens_single_kernel<DT, 256, 16>, c);
    }
    const uint64_t cap = (uint64_t)c.sms * 8;
    return launch_chained(quantize_tokens_any_kernel<DT>, dim3((unsigned)(c.rows < cap ? c.rows : cap)), dim3(CTA), 0, c.stream,
                          static_cast<const typename Elem<DT>::T *>(c.x), c.rows, c.cols, c.ld_x, c.q, c.q_pitch, c.qp, c.sums);
}

}  // namespace

cudaError_t launch_quantize_tokens(const void *x, int dtype, uint64_t rows, uint64_t cols, uint64_t ld_x, uint8_t *q, uint64_t q_pitch,
                                   ltq_qparams *qp, int32_t *sums, int sms, cudaStream_t stream)
{
    count_launch();
    const RowCall c{x, rows, cols, ld_x, q, q_pitch, qp, sums, sms, stream};
    return dtype == LTQ_F32 ? launch_quantize_dt<LTQ_F32>(c) : (dtype == LTQ_F16 ? launch_quantize_dt<LTQ_F16>(c) : launch_quantize_dt<LTQ_BF16>(c));
}

// ---- dequantise ---------------------------------------------------------------------------------------------------------
// value = scale * (q - zero), rounded to float and then to the output type.  A warp takes DEQ_STEPS runs of 32 x VEC codes of one row,
// all loads before the first store; VEC codes make one 16-byte store, so that both sides are whole lines.
constexpr int DEQ_STEPS = 4;

template <int DT>
__global__ void __launch_bounds__(CTA)
dequantize_tokens_kernel(typename Elem<DT>::T *__restrict__ x, uint64_t ld_x, const uint8_t *__restrict__ q, const ltq_qparams *__restrict__ qp,
                         uint64_t rows, uint64_t cols, uint32_t pieces, bool vec)
{
    griddep_launch_dependents();
    griddep_wait();
    using E = Elem<DT>;
    constexpr int VEC = E::PER16, PIECE = 32 * VEC * DEQ_STEPS;
    const int lane = threadIdx.x & 31;
    const uint64_t nwarps = ((uint64_t)gridDim.x * CTA) >> 5;
    for (uint64_t w = ((uint64_t)blockIdx.x * CTA + threadIdx.x) >> 5; w < rows * pieces; w += nwarps) {
        const uint64_t row = w / pieces, c0 = (w - row * pieces) * PIECE;
        const uint8_t *qr = q + row * cols;
        typename E::T *xr = x + row * ld_x;
        if (vec) {
            uint32_t word[DEQ_STEPS][VEC / 4];
#pragma unroll
            for (int i = 0; i < DEQ_STEPS; i++) {
                const uint64_t c = c0 + (uint64_t)(i * 32 + lane) * VEC;
                if (c < cols) {
                    if (VEC == 8) *reinterpret_cast<uint2 *>(word[i]) = __ldcs(reinterpret_cast<const uint2 *>(qr + c));
                    else word[i][0] = __ldcs(reinterpret_cast<const uint32_t *>(qr + c));
                }
            }
            const float scale = qp[row].scale;
            const int zp = (int)qp[row].zero_point;
#pragma unroll
            for (int i = 0; i < DEQ_STEPS; i++) {
                const uint64_t c = c0 + (uint64_t)(i * 32 + lane) * VEC;
                if (c >= cols) break;
                float v[VEC];
#pragma unroll
                for (int k = 0; k < VEC; k++) v[k] = __fmul_rn(scale, (float)((int)(word[i][k / 4] >> (8 * (k % 4)) & 0xFF) - zp));
                uint4 o;
                if (DT == LTQ_F32) o = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
                else o = make_uint4(token_bits2<DT>(v[0], v[1]), token_bits2<DT>(v[2], v[3]), token_bits2<DT>(v[4 % VEC], v[5 % VEC]), token_bits2<DT>(v[6 % VEC], v[7 % VEC]));
                __stcs(reinterpret_cast<uint4 *>(xr + c), o);
            }
        } else {
            constexpr int N = PIECE / 32;
            uint8_t b[N];
#pragma unroll
            for (int i = 0; i < N; i++) b[i] = c0 + i * 32 + lane < cols ? qr[c0 + i * 32 + lane] : (uint8_t)0;
            const float scale = qp[row].scale;
            const int zp = (int)qp[row].zero_point;
#pragma unroll
            for (int i = 0; i < N; i++)
                if (c0 + i * 32 + lane < cols) xr[c0 + i * 32 + lane] = E::out(__fmul_rn(scale, (float)((int)b[i] - zp)));
        }
    }
}

namespace {

template <int DT>
cudaError_t launch_dequantize_dt(void *x, uint64_t ld_x, const uint8_t *q, const ltq_qparams *qp, uint64_t rows, uint64_t cols, int sms,
                                 cudaStream_t stream)
{
    constexpr uint64_t VEC = Elem<DT>::PER16, PIECE = 32 * VEC * DEQ_STEPS;
    const uint64_t pieces = (cols + PIECE - 1) / PIECE, want = (rows * pieces + 7) / 8, cap = (uint64_t)sms * 64;
    const bool vec = cols % VEC == 0 && ld_x % VEC == 0 && ((uintptr_t)x & 15) == 0 && ((uintptr_t)q & (VEC - 1)) == 0;
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
