// Linear layer in 8-bit integers: a scale per token (row of x) and per output channel (row of the weight).
//
//   quantise a row   a = max_k |x_k|,  s = a / 127,  q_k = rne(127 x_k / a)
//   product          y[t, n] = float(sum_k q[t, k] wq[n, k]) * s[t] * ws[n] + bias[n]
//
// Rows of 8-bit operands are padded with zeros to a multiple of 16 bytes (pitch = cols rounded up). The
// sum is an exact 32-bit integer (in <= 131056 keeps it below 2^31 for every pair of 8-bit values), so a value
// does not depend on how the reduction is split, nor on the number of rows of the call.
#include "common.cuh"

namespace sf {

constexpr int kQThreads = 256;

// The integer nearest to 127 x / a (ties to even) for |x| <= a, decided as if the quotient were exact: a
// multiplication by the rounded 127 / a is within 2^-16 of it; where that leaves doubt (closer than 2^-12 to a half, or a row
// so small that 127 / a overflows) the quotient itself is formed.
//  bf16: 127 x has 15 significant bits, so it is exact in fp32; a quotient of such numbers that is not half-way between
//        integers is at least 1 / (2^9 * 2^gap) away (gap: how many powers of two |x| is below a, the quotient
//        being about 2^(7 - gap)), while the rounded fp32 quotient is within 2^(7 - gap - 24) of it.
//  fp32: product and quotient in fp64 (31 and 53 bits, the same argument).
struct RowScale {
    float a, inv;
    bool doubt;  // every element takes the quotient
};
__device__ __forceinline__ RowScale row_scale(float a) {
    RowScale r;
    r.a = a;
    r.inv = __fdiv_rn(127.0f, a);
    r.doubt = a < 0x1p-118f;
    return r;
}
__device__ __forceinline__ int quotient(__nv_bfloat16, float x, float a) {
    // 127 x would leave fp32 at the top of its range: both sides are moved by an exact power of two there
    const bool huge = a >= 0x1p119f;
    return __float2int_rn(__fdiv_rn((huge ? 127.0f * 0x1p-10f : 127.0f) * x, huge ? a * 0x1p-10f : a));
}
__device__ __forceinline__ int quotient(float, float x, float a) { return __double2int_rn(127.0 * (double)x / (double)a); }
template <typename T>
__device__ __forceinline__ int quantise(T tag, float x, const RowScale& r) {
    const float v = x * r.inv, n = rintf(v);
    if (r.doubt || fabsf(v - n) > 0.5f - 0x1p-12f) return quotient(tag, x, r.a);
    return __float2int_rn(n);
}

template <typename T>
__device__ __forceinline__ float as_f32(T v) { return (float)v; }

// One block per row. A row whose largest magnitude is infinite or NaN gets a NaN scale and zeros.
template <typename T>
__global__ void __launch_bounds__(kQThreads)
int8_quantize_kernel(const T* __restrict__ x, int64_t ld, int8_t* __restrict__ q, float* __restrict__ scale, int cols,
                     int pitch) {
    __shared__ uint32_t part[kQThreads / 32];
    const T* row = x + (int64_t)blockIdx.x * ld;
    uint32_t top = 0;  // bit pattern of the largest magnitude: a NaN is above infinity
    for (int k = threadIdx.x; k < cols; k += kQThreads) top = max(top, __float_as_uint(as_f32(row[k])) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQThreads / 32; ++w) top = max(top, part[w]);
    const bool finite = top < 0x7f800000u;
    const float a = __uint_as_float(top);
    const RowScale rs = row_scale(a);
    if (threadIdx.x == 0) scale[blockIdx.x] = finite ? __fdiv_rn(a, 127.0f) : __uint_as_float(0x7fffffffu);
    int8_t* out = q + (int64_t)blockIdx.x * pitch;
    for (int k = threadIdx.x; k < pitch; k += kQThreads)
        out[k] = (int8_t)(k < cols && finite && top != 0 ? quantise(T(), as_f32(row[k]), rs) : 0);
}

// One place for the arithmetic behind the sum, so that every kernel rounds alike.
__device__ __forceinline__ float int8_scaled(int acc, float xs, float ws) { return __int2float_rn(acc) * xs * ws; }

constexpr int kSimpleTile = 32;
template <typename T>
__global__ void __launch_bounds__(256)
int8_gemm_simple_kernel(const int8_t* __restrict__ xq, const float* __restrict__ xs, const int8_t* __restrict__ wq,
                        const float* __restrict__ ws, const T* __restrict__ bias, T* __restrict__ y, int rows, int pitch,
                        int out) {
    __shared__ int a[kSimpleTile][5], b[kSimpleTile][5];
    const int t0 = blockIdx.y * kSimpleTile, n0 = blockIdx.x * kSimpleTile;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    int acc[4] = {0, 0, 0, 0};
    for (int k = 0; k < pitch; k += 16) {
        if (threadIdx.x < 128) {
            const int r = threadIdx.x >> 2, w = threadIdx.x & 3;
            a[r][w] = t0 + r < rows ? *reinterpret_cast<const int*>(xq + (int64_t)(t0 + r) * pitch + k + 4 * w) : 0;
        } else {
            const int r = (threadIdx.x - 128) >> 2, w = threadIdx.x & 3;
            b[r][w] = n0 + r < out ? *reinterpret_cast<const int*>(wq + (int64_t)(n0 + r) * pitch + k + 4 * w) : 0;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) acc[i] = __dp4a(a[ty * 4 + i][w], b[tx][w], acc[i]);
        __syncthreads();
    }
    const int n = n0 + tx;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = t0 + ty * 4 + i;
        if (t < rows && n < out) {
            float v = int8_scaled(acc[i], xs[t], ws[n]);
            if (bias) v += as_f32(bias[n]);
            y[(int64_t)t * out + n] = (T)v;
        }
    }
}

static int check_int8(const char* who, int64_t rows, int64_t in, int64_t out) {
    if (rows < 0 || in <= 0 || out <= 0) return fail(SF_ERR_BAD_ARG, "%s: rows must not be negative, in and out positive", who);
    if (rows > 0x7fffff00 || out > 0x7fffff00) return fail(SF_ERR_UNSUPPORTED, "%s: dimension beyond 2^31", who);
    if (in > SF_INT8_MAX_IN)
        return fail(SF_ERR_UNSUPPORTED, "%s: in=%lld: beyond %lld the 32-bit sum of 8-bit products could overflow", who,
                    (long long)in, (long long)SF_INT8_MAX_IN);
    return SF_OK;
}

static int quantize_impl(const void* x, int dtype, int64_t ld, int8_t* q, float* scale, int64_t rows, int64_t cols,
                         cudaStream_t st) {
    const int pitch = (int)((cols + 15) / 16 * 16);
    if (dtype == SF_F32)
        int8_quantize_kernel<float><<<(int)rows, kQThreads, 0, st>>>((const float*)x, ld, q, scale, (int)cols, pitch);
    else
        int8_quantize_kernel<__nv_bfloat16><<<(int)rows, kQThreads, 0, st>>>((const __nv_bfloat16*)x, ld, q, scale, (int)cols, pitch);
    SF_CHECK_CUDA(cudaGetLastError());
    return SF_OK;
}

static int gemm_impl(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, const void* bias, void* y, int dtype,
                     int64_t rows, int64_t in, int64_t out, int32_t* status, cudaStream_t st) {
    const int pitch = (int)((in + 15) / 16 * 16);
    dim3 grid((unsigned)((out + kSimpleTile - 1) / kSimpleTile), (unsigned)((rows + kSimpleTile - 1) / kSimpleTile));
    (void)status;
    if (grid.y > 65535) return fail(SF_ERR_UNSUPPORTED, "int8 product: too many rows");
    if (dtype == SF_F32)
        int8_gemm_simple_kernel<float><<<grid, 256, 0, st>>>(xq, xs, wq, ws, (const float*)bias, (float*)y, (int)rows, pitch, (int)out);
    else
        int8_gemm_simple_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(xq, xs, wq, ws, (const __nv_bfloat16*)bias, (__nv_bfloat16*)y, (int)rows, pitch, (int)out);
    SF_CHECK_CUDA(cudaGetLastError());
    return SF_OK;
}

}  // namespace sf

using namespace sf;

extern "C" {

int64_t sf_int8_pitch(int64_t cols) { return (cols + 15) / 16 * 16; }

int sf_int8_quantize_rows(const void* x, int dtype, int64_t ld, int8_t* q, float* scale, int64_t rows, int64_t cols,
                          void* stream) {
    if (int rc = check_int8("sf_int8_quantize_rows", rows, cols, 1)) return rc;
    SF_CHECK_ARG(dtype == SF_F32 || dtype == SF_BF16, "sf_int8_quantize_rows: dtype must be SF_F32 or SF_BF16");
    if (rows == 0) return SF_OK;
    SF_CHECK_ARG(x && q && scale, "sf_int8_quantize_rows: x, q and scale must be non-null");
    SF_CHECK_ARG(ld >= cols || rows == 1, "sf_int8_quantize_rows: ld=%lld is smaller than a row", (long long)ld);
    if (!aligned16(q)) return fail(SF_ERR_ALIGNMENT, "sf_int8_quantize_rows: q must be 16-byte aligned");
    return quantize_impl(x, dtype, ld, q, scale, rows, cols, (cudaStream_t)stream);
}

static int check_product(const char* who, const void* wq, const float* ws, const void* y, int dtype, int64_t rows, int64_t in,
                         int64_t out) {
    if (int rc = check_int8(who, rows, in, out)) return rc;
    if (dtype != SF_F32 && dtype != SF_BF16) return fail(SF_ERR_BAD_ARG, "%s: dtype must be SF_F32 or SF_BF16", who);
    if (rows == 0) return SF_OK;
    if (!wq || !ws || !y) return fail(SF_ERR_BAD_ARG, "%s: weight, scales and y must be non-null", who);
    if (!aligned16(wq)) return fail(SF_ERR_ALIGNMENT, "%s: 8-bit operands must be 16-byte aligned", who);
    return SF_OK;
}

int sf_int8_gemm(const int8_t* xq, const float* x_scale, const int8_t* wq, const float* w_scale, const void* bias, void* y,
                 int dtype, int64_t rows, int64_t in, int64_t out, int32_t* status, void* stream) {
    if (int rc = check_product("sf_int8_gemm", wq, w_scale, y, dtype, rows, in, out)) return rc;
    if (rows == 0) return SF_OK;
    SF_CHECK_ARG(xq && x_scale, "sf_int8_gemm: xq and x_scale must be non-null");
    if (!aligned16(xq)) return fail(SF_ERR_ALIGNMENT, "sf_int8_gemm: 8-bit operands must be 16-byte aligned");
    return gemm_impl(xq, x_scale, wq, w_scale, bias, y, dtype, rows, in, out, status, (cudaStream_t)stream);
}

int64_t sf_int8_linear_workspace_bytes(int64_t rows, int64_t in) {
    return rows <= 0 || in <= 0 ? 0 : rows * ((in + 15) / 16 * 16) + rows * 4;
}

int sf_int8_linear(const void* x, int64_t ld, const int8_t* wq, const float* w_scale, const void* bias, void* y, int dtype,
                   int64_t rows, int64_t in, int64_t out, void* workspace, int32_t* status, void* stream) {
    if (int rc = check_product("sf_int8_linear", wq, w_scale, y, dtype, rows, in, out)) return rc;
    if (rows == 0) return SF_OK;
    SF_CHECK_ARG(x && workspace, "sf_int8_linear: x and workspace must be non-null");
    SF_CHECK_ARG(ld >= in || rows == 1, "sf_int8_linear: ld=%lld is smaller than a row", (long long)ld);
    if (!aligned16(workspace)) return fail(SF_ERR_ALIGNMENT, "sf_int8_linear: workspace must be 16-byte aligned");
    int8_t* xq = static_cast<int8_t*>(workspace);
    float* xs = reinterpret_cast<float*>(xq + rows * sf_int8_pitch(in));
    if (int rc = quantize_impl(x, dtype, ld, xq, xs, rows, in, (cudaStream_t)stream)) return rc;
    return gemm_impl(xq, xs, wq, w_scale, bias, y, dtype, rows, in, out, status, (cudaStream_t)stream);
}

}  // extern "C"
