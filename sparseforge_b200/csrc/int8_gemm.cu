// Linear layer in 8-bit integers: a scale per token (row of x) and per output channel (row of the weight).
//
//   quantise a row   a = max_k |x_k|,  s = a / 127,  q_k = rne(127 x_k / a)
//   product          y[t, n] = float(sum_k q[t, k] wq[n, k]) * s[t] * ws[n] + bias[n]
//
// Rows of 8-bit operands are padded with zeros to a multiple of 16 bytes (pitch = cols rounded up). The
// sum is an exact 32-bit integer (in <= 131056 keeps it below 2^31 for every pair of 8-bit values), so a value
// does not depend on how the reduction is split, nor on the number of rows of the call.
#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "ptx_sm100.cuh"

namespace sf {

int make_byte_tensor_map(CUtensorMap* map, const void* ptr, int64_t pitch, int64_t outer, int box_outer);

constexpr int kQThreads = 256;
constexpr int kQVecResident = 2048;  // threads per SM of the register-resident quantiser

// The integer nearest to 127 x / a (ties to even) for |x| <= a, decided as if the quotient were exact, from a
// multiplication by an approximate 127 / a (relative error below 2^-22: the reciprocal's 2^-23, two roundings).
//  bf16: with gap the number of powers of two that |x| is below a, the quotient is below 2^(7 - gap); 127 x and a being integers of
//        15 and 8 bits times a power of two, a quotient that is not half-way between integers is at least 2^-(9 + gap) away
//        from it. A tie needs 254 x / a odd: x = a / 2 (63.5, to the even 64), since 127 divides no 8-bit significand but
//        254. So the factor is raised by 2^-21, more than its error, which sends ties away from zero; with the raise the
//        product is within 2^-(13.4 + gap) of the quotient (2^-21 + 2^-22 of it), which decides everything else. Rows whose a
//        has the significand 254 take quotients.
//  fp32: where the product is closer than 2^-14 to a half the quotient is formed, in fp64 (31 and 53 bits, as above).
// Where the reciprocal would leave the normal range every element of the row takes the quotient.
constexpr float kClear = 0.5f - 0x1p-14f;  // a rounding that moved the value by no more leaves no doubt
struct RowScale {
    float a, inv;
    bool doubt;  // every element takes the quotient
};
template <typename T>
__device__ __forceinline__ RowScale row_scale(float a) {
    constexpr bool bf16 = sizeof(T) == 2;
    RowScale r;
    r.a = a;
    r.inv = (bf16 ? 127.0f * (1.0f + 0x1p-21f) : 127.0f) * fast_rcp(a);
    r.doubt = a < 0x1p-118f || a > 0x1p118f || (bf16 && (__float_as_uint(a) & 0x007f0000u) == 0x007e0000u);
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
    if (r.doubt || (sizeof(T) == 4 && fabsf(v - n) > kClear)) return quotient(tag, x, r.a);
    return __float2int_rn(n);
}

template <typename T>
__device__ __forceinline__ float as_f32(T v) { return (float)v; }

__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float nan_f32() { return __uint_as_float(0x7fffffffu); }

// Eight elements as they lie in memory (16 bytes of bf16, 32 of fp32).
template <typename T>
struct Raw8;
template <>
struct Raw8<__nv_bfloat16> {
    uint4 v;
    __device__ __forceinline__ void clear() { v = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = ptx::ld_global_v4(p); }
    __device__ __forceinline__ void load_edge(const __nv_bfloat16* row, int first, int cols) {  // zero outside the row
        const unsigned short* u = reinterpret_cast<const unsigned short*>(row);
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = first + i >= 0 && first + i < cols ? ptx::ld_global_u16(u + first + i) : 0u;
        v = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
    __device__ __forceinline__ void unpack(float (&x)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};
template <>
struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void clear() { a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    __device__ __forceinline__ void load(const float* p) {
        const uint4 u = ptx::ld_global_v4(p), w = ptx::ld_global_v4(p + 4);
        a = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
        b = make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
    }
    __device__ __forceinline__ void load_edge(const float* row, int first, int cols) {  // zero outside the row
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = first + i >= 0 && first + i < cols ? ptx::ld_global_f32(row + first + i) : 0.0f;
        a = make_float4(w[0], w[1], w[2], w[3]);
        b = make_float4(w[4], w[5], w[6], w[7]);
    }
    __device__ __forceinline__ void unpack(float (&x)[8]) const {
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
};
// The largest magnitude so far as a bit pattern, ordered like the values with a NaN above infinity. bf16: two patterns of
// 16 bits side by side; top_bits() gives the fp32 pattern.
__device__ __forceinline__ uint32_t top8(const Raw8<__nv_bfloat16>& r, uint32_t top) {
    const uint32_t m = 0x7fff7fffu;
    return __vmaxu2(__vmaxu2(__vmaxu2(r.v.x & m, r.v.y & m), __vmaxu2(r.v.z & m, r.v.w & m)), top);
}
__device__ __forceinline__ uint32_t top8(const Raw8<float>& r, uint32_t top) {
    float x[8];
    r.unpack(x);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude_bits(x[i]));
    return top;
}
__device__ __forceinline__ uint32_t top_bits(__nv_bfloat16, uint32_t top) { return max(top << 16, top & 0xffff0000u); }
__device__ __forceinline__ uint32_t top_bits(float, uint32_t top) { return top; }

__device__ __forceinline__ uint2 pack8(const uint32_t (&u)[8]) {  // the low byte of each
    const uint32_t a0 = __byte_perm(u[0], u[1], 0x0040), a1 = __byte_perm(u[2], u[3], 0x0040);
    const uint32_t b0 = __byte_perm(u[4], u[5], 0x0040), b1 = __byte_perm(u[6], u[7], 0x0040);
    return make_uint2(__byte_perm(a0, a1, 0x5410), __byte_perm(b0, b1, 0x5410));
}
template <typename T>
__device__ __noinline__ uint2 quotient8(Raw8<T> r, float a) {
    float x[8];
    uint32_t u[8];
    r.unpack(x);
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = (uint32_t)quotient(T(), x[i], a);
    return pack8(u);
}

// Eight integers, one per byte. Adding 3 * 2^22 rounds to an integer and leaves it in the low byte: one multiply-add
// per element. fp32: what the rounding moved says whether any of the eight is in doubt (three more).
template <typename T>
__device__ __forceinline__ uint2 quantise8(const Raw8<T>& r, const RowScale& rs) {
    constexpr float magic = 12582912.0f;
    if (rs.doubt) return quotient8(r, rs.a);
    float x[8];
    r.unpack(x);
    uint32_t u[8];
    float moved = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = __fmaf_rn(x[i], rs.inv, magic);
        if (sizeof(T) == 4) moved = fmaxf(moved, fabsf(__fmaf_rn(x[i], rs.inv, -(t - magic))));
        u[i] = __float_as_uint(t);
    }
    if (sizeof(T) == 4 && moved > kClear) return quotient8(r, rs.a);
    return pack8(u);
}

// A row whose largest magnitude is infinite or NaN gets a NaN scale and zeros.
// Rows on 16-byte boundaries, a multiple of 8 long: TPR threads hold a row in registers (NV groups of eight each)
// between finding its largest magnitude and rounding it: one read, one write. Blocks stay and take row after row; the
// loads of the next are issued before the present one is reduced, so that the memory system is never left idle.
template <typename T, int THREADS, int TPR, int NV>
__global__ void __launch_bounds__(THREADS)
int8_quantize_vec_kernel(const T* x, int64_t ld, int8_t* __restrict__ q, float* __restrict__ scale, int rows,
                         int cols, int pitch) {
    __shared__ uint32_t part[2][THREADS / 32];
    ptx::dependency_wait();
    ptx::launch_dependents();  // only now: what ran before this kernel is complete for the one behind it as well
    constexpr int PER_BLOCK = THREADS / TPR;
    const int lane = threadIdx.x % TPR, nv = cols >> 3;
    int row = blockIdx.x * PER_BLOCK + threadIdx.x / TPR;
    const int step = gridDim.x * PER_BLOCK;
    Raw8<T> next[NV];
    auto fetch = [&](int from) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (from < rows && lane + i * TPR < nv) next[i].load(x + from * ld + 8 * (lane + i * TPR));
    };
    fetch(row);
    for (int turn = 0; row < rows; row += step, turn ^= 1) {  // all threads of a row, with TPR > 32 of the block, alike
        Raw8<T> r[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) r[i] = next[i];
        if (row < rows - step) fetch(row + step);
        uint32_t top = 0;  // bit pattern of the largest magnitude: a NaN is above infinity
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + i * TPR < nv) top = top8(r[i], top);
        top = __reduce_max_sync(0xffffffffu, top_bits(T(), top));
        if (TPR > 32) {
            if ((threadIdx.x & 31) == 0) part[turn][threadIdx.x >> 5] = top;
            __syncthreads();  // the other half of `part` is still being read by slower warps
#pragma unroll
            for (int w = 0; w < TPR / 32; ++w) top = max(top, part[turn][w]);
        }
        const bool usable = top < 0x7f800000u && top != 0;
        const RowScale rs = row_scale<T>(__uint_as_float(top));
        if (lane == 0) scale[row] = top < 0x7f800000u ? __fdiv_rn(rs.a, 127.0f) : nan_f32();
        uint2* dst = reinterpret_cast<uint2*>(q + (int64_t)row * pitch);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + i * TPR < nv) dst[lane + i * TPR] = usable ? quantise8(r[i], rs) : make_uint2(0u, 0u);
        if (lane == 0 && (nv & 1)) dst[nv] = make_uint2(0u, 0u);
    }
}

// Any other row (any length, any element alignment): TPR threads per row. Loads are the 16-byte granules the row lies in;
// the two granules at its ends that it only partly fills are read element by element. A granule's eight results
// belong to two neighbouring 8-byte pieces of the output: the second part comes from the next lane, so a warp takes 32
// granules and writes 31 pieces. NV > 0: all of a row's granules stay in registers, NV per thread (rows of up to NV * 31 *
// TPR / 32 pieces); NV = 0: longer rows are read twice, the second time from a cache.
template <typename T>
__device__ __forceinline__ void load_granule(Raw8<T>& r, const T* row, int first, int cols) {  // elements first ... first + 7
    if (first >= 0 && first + 8 <= cols) r.load(row + first);
    else r.load_edge(row, first, cols);
}
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(kQThreads)
int8_quantize_any_kernel(const T* x, int64_t ld, int8_t* __restrict__ q, float* __restrict__ scale, int rows,
                         int cols, int pitch) {
    __shared__ uint32_t part[kQThreads / 32];
    ptx::dependency_wait();
    ptx::launch_dependents();
    constexpr int STEP = TPR / 32 * 31;
    const int wanted = blockIdx.x * (kQThreads / TPR) + threadIdx.x / TPR;
    const bool live = wanted < rows;
    const int r = live ? wanted : rows - 1;  // threads without a row follow the last one, for the barrier, and write nothing
    const T* row = x + (int64_t)r * ld;
    const int lead = (int)(reinterpret_cast<uintptr_t>(row) & 15) / (int)sizeof(T);  // elements of the first granule before the row
    const int granules = (cols + lead + 7) / 8, pieces = pitch / 8, me = threadIdx.x % TPR, lane = threadIdx.x & 31;
    const int first = me / 32 * 31;  // first piece of this warp
    Raw8<T> kept[NV ? NV : 1];
    uint32_t top = 0;
    if (NV) {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int v = first + u * STEP + lane;
            kept[u].clear();
            if (v < granules) load_granule(kept[u], row, 8 * v - lead, cols);
        }
#pragma unroll
        for (int u = 0; u < NV; ++u) top = top8(kept[u], top);
    } else {
#pragma unroll 4
        for (int v = me; v < granules; v += TPR) {
            Raw8<T> g;
            load_granule(g, row, 8 * v - lead, cols);
            top = top8(g, top);
        }
    }
    top = __reduce_max_sync(0xffffffffu, top_bits(T(), top));
    if (TPR > 32) {
        const int w0 = threadIdx.x / TPR * (TPR / 32);
        if (lane == 0) part[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < TPR / 32; ++w) top = max(top, part[w0 + w]);
    }
    const bool usable = top < 0x7f800000u && top != 0;
    const RowScale rs = row_scale<T>(__uint_as_float(top));
    if (live && me == 0) scale[r] = top < 0x7f800000u ? __fdiv_rn(rs.a, 127.0f) : nan_f32();
    unsigned long long* dst = reinterpret_cast<unsigned long long*>(q + (int64_t)r * pitch);
    auto put = [&](const Raw8<T>& g, int v) {
        unsigned long long bytes = 0;
        if (usable && v < granules) {
            const uint2 b = quantise8(g, rs);
            bytes = (unsigned long long)b.y << 32 | b.x;
        }
        const unsigned long long next = __shfl_down_sync(0xffffffffu, bytes, 1);
        if (live && lane < 31 && v < pieces) dst[v] = lead ? bytes >> (8 * lead) | next << (64 - 8 * lead) : bytes;
    };
    if (NV) {
#pragma unroll
        for (int u = 0; u < NV; ++u) put(kept[u], first + u * STEP + lane);
    } else {
#pragma unroll 2
        for (int base = first; base < pieces; base += STEP) {
            Raw8<T> g;
            g.clear();
            if (base + lane < granules) load_granule(g, row, 8 * (base + lane) - lead, cols);
            put(g, base + lane);
        }
    }
}

// One place for the arithmetic behind the sum, so that every kernel rounds alike (bias 0 where there is none). The sum times
// the token's scale is formed first: rounded once, and exact where it is subnormal (an integer times a multiple of 2^-149). From
// a scale of 2^96 on it could leave fp32 (the sum is below 2^31) though the result, after the channel's scale, does not: it
// is formed 2^32 lower there, with the same significand, and the rest in fp64.
constexpr float kHugeScale = 0x1p96f;
__device__ __noinline__ float int8_out_huge(int acc, float xs, float ws, float bias) {
    const float low = __fmul_rn(__int2float_rn(acc), xs * 0x1p-32f);
    return __double2float_rn(__fma_rn((double)low, (double)ws * 0x1p32, (double)bias));
}
__device__ __forceinline__ float int8_out_usual(int acc, float xs, float ws, float bias) {
    return __fmaf_rn(__fmul_rn(__int2float_rn(acc), xs), ws, bias);
}
__device__ __forceinline__ float int8_out(int acc, float xs, float ws, float bias) {
    return fabsf(xs) >= kHugeScale ? int8_out_huge(acc, xs, ws, bias) : int8_out_usual(acc, xs, ws, bias);
}

// ---------------------------------------------------------------------------------------------------------
// Many rows: persistent CTA pairs, 256 x 256 tiles, tcgen05.mma.cta_group::2.kind::i8.
//
// A = xq (rows x K), B = wq (out x K), both K-contiguous: the bytes of a stage are those of the bf16 pair
// kernel (128 bytes of K = 128 integers instead of 64 bf16; 16 KiB of A and 16 KiB of B per CTA, six stages), an
// instruction covers 32 of K at the bf16 instruction's cycle count. Two accumulators of 256 columns fill the tensor memory:
// the epilogue (integer -> float, two scales, bias, store) of a tile runs under the next tile's products.
// [8192, 4096] x [4096, 4096]: 84 us = 3260 TOP/s, the tensor pipe busy in 83 % of its cycles and more (operand delivery takes
// the rest, as in the bf16 kernel); [8192, 4096] x [11008, 4096]: 230 us = 3210 TOP/s under the power cap.
// ---------------------------------------------------------------------------------------------------------
constexpr int I8_BK = 128;                      // bytes = integers of K per stage: one 128-byte swizzled row
constexpr int I8_THREADS = 192;
constexpr int I8_STAGES = 6;
constexpr int I8_OPERAND_BYTES = 128 * I8_BK;   // 16 KiB: this CTA's 128 rows of A, and its half of B's 256 rows
constexpr int I8_STAGE_BYTES = 2 * I8_OPERAND_BYTES;
constexpr int I8_EPI_BYTES = 2 * 256 * 4;       // per epilogue warp: scales and bias of the tile's columns
constexpr int I8_PAIR_SMEM = I8_STAGES * I8_STAGE_BYTES + 4 * (I8_EPI_BYTES + 32 * 144) + 1024 + 256;  // and four turn buffers
constexpr int I8_RASTER_M = 16;                 // tile rows per raster group: panels are shared in L2

struct I8PairTail {
    uint64_t full[I8_STAGES];
    uint64_t empty[I8_STAGES];
    uint64_t tmem_full[2];
    uint64_t tmem_empty[2];
    uint32_t tmem_base;
    int abort_flag;
};

__device__ __forceinline__ void i8_tile_coords(int tile, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int per_group = I8_RASTER_M * tiles_n;
    const int g = tile / per_group, first = g * I8_RASTER_M;
    const int gm = min(I8_RASTER_M, tiles_m - first), r = tile - g * per_group;
    tm = first + r % gm;
    tn = r / gm;
}

// Results leave through a turn buffer in shared memory, 128 bytes of 32 rows at a time (64 bf16 or 32 fp32 columns): a
// thread holds one row, a store instruction then covers whole rows: four rows x 128 bytes in 16-byte pieces, or, where
// rows are not on 16-byte boundaries, 32 consecutive elements of one row. Stored straight from the threads that hold a row
// each, an odd number of channels cost [8192, 4096] x [4095, 4096] 348 us instead of 88 in bf16. In fp32, where a row of 128 bytes
// holds half as many columns, unaligned rows still cost more: [2048, 512] x [9001, 512] 47 us, x [9000, 512] 25 us.
constexpr int I8_TURN_ROW = 128 + 16;  // padding against bank conflicts
constexpr int I8_TURN_BYTES = 32 * I8_TURN_ROW;

__device__ __forceinline__ void turn_in(uint8_t* row, const float (&v)[32], int part, __nv_bfloat16) {  // part: left or right half
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[8 * j + 2 * i], v[8 * j + 2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<uint4*>(row + part * 64 + j * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
__device__ __forceinline__ void turn_in(uint8_t* row, const float (&v)[32], int, float) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        *reinterpret_cast<float4*>(row + j * 16) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}
// 32 rows of the turn buffer to y: dst is row 0's first column of the chunk, `rows` rows and `cols` columns of it exist.
template <typename T>
__device__ __forceinline__ void turn_out(const uint8_t* buf, T* dst, int64_t ld, int rows, int cols, bool vec, int lane) {
    constexpr int PIECE = 16 / sizeof(T), COLS = 128 / sizeof(T);
    if (vec) {
        const int piece = lane & 7;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
            if (r < rows && piece * PIECE < cols)  // ld is a multiple of PIECE, so a piece exists wholly or not at all
                *reinterpret_cast<uint4*>(dst + r * ld + piece * PIECE) = *reinterpret_cast<const uint4*>(buf + r * I8_TURN_ROW + piece * 16);
        }
    } else {
#pragma unroll 8
        for (int r = 0; r < 32; ++r) {
            if (r >= rows) break;
            const T* src = reinterpret_cast<const T*>(buf + r * I8_TURN_ROW);
#pragma unroll
            for (int c = 0; c < COLS; c += 32)
                if (c + lane < cols) dst[r * ld + c + lane] = src[c + lane];
        }
    }
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8_THREADS, 1)
int8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const float* xs, const float* __restrict__ ws, const T* __restrict__ bias, T* y, int rows, int out,
                 int pitch, int32_t* status) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = ptx::smem_u32(smem_raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw_addr);
    float* epi = reinterpret_cast<float*>(base_ptr + I8_STAGES * I8_STAGE_BYTES);
    uint8_t* turns = base_ptr + I8_STAGES * I8_STAGE_BYTES + 4 * I8_EPI_BYTES;
    I8PairTail* tail = reinterpret_cast<I8PairTail*>(turns + 4 * I8_TURN_BYTES);
    volatile int* abort_flag = &tail->abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta = ptx::cluster_ctarank();
    const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
    const int tiles_m = (rows + 255) / 256, tiles_n = (out + 255) / 256;
    const int total_tiles = tiles_m * tiles_n;
    const int num_kb = (pitch + I8_BK - 1) / I8_BK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < I8_STAGES; ++s) {
            ptx::mbar_init(ptx::smem_u32(&tail->full[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&tail->empty[s]), 1);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(ptx::smem_u32(&tail->tmem_full[a]), 1);
            ptx::mbar_init(ptx::smem_u32(&tail->tmem_empty[a]), 8);
        }
        tail->abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(ptx::smem_u32(&tail->tmem_base), 512);
        ptx::tmem_relinquish_pair();
    }
    if (warp == 0 && lane == 0) {
        ptx::prefetch_tensormap(&tmA);
        ptx::prefetch_tensormap(&tmB);
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync_all();
    ptx::tc_fence_after();
    const uint32_t tmem_base = tail->tmem_base;
    ptx::dependency_wait();  // the quantised rows are complete from here on

    if (warp == 0) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = pair; tile < total_tiles && ok; tile += num_pairs) {
            int tm, tn;
            i8_tile_coords(tile, tiles_m, tiles_n, tm, tn);
            const int m0 = tm * 256 + (int)cta * 128, n0 = tn * 256 + (int)cta * 128;
            for (int kb = 0; kb < num_kb; ++kb) {
                ok = ptx::mbar_wait(ptx::smem_u32(&tail->empty[stage]), phase ^ 1u, abort_flag, status, 41);
                if (!ok) break;
                if (lane == 0) {
                    const uint32_t local_bar = ptx::smem_u32(&tail->full[stage]);
                    const uint32_t bar = ptx::map_to_cta(local_bar, 0);
                    const uint32_t sa = base + stage * I8_STAGE_BYTES, sb = sa + I8_OPERAND_BYTES;
                    if (cta == 0) ptx::mbar_arrive_expect_tx(local_bar, 2 * I8_STAGE_BYTES);
                    ptx::tma_load_2d_pair(sa, &tmA, bar, kb * I8_BK, m0);
                    ptx::tma_load_2d_pair(sb, &tmB, bar, kb * I8_BK, n0);
                }
                __syncwarp();
                if (++stage == I8_STAGES) { stage = 0; phase ^= 1u; }
            }
        }
        if (!ok) for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else if (warp == 1) {
        if (cta == 0) {
            constexpr uint32_t idesc = ptx::make_idesc_i8(256, 256);
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            int t = 0;
            for (int tile = pair; tile < total_tiles && ok; tile += num_pairs, ++t) {
                const int acc = t & 1;
                ok = ptx::mbar_wait(ptx::smem_u32(&tail->tmem_empty[acc]), ((uint32_t)(t >> 1) & 1u) ^ 1u, abort_flag, status, 43);
                if (!ok) break;
                ptx::tc_fence_after();
                const uint32_t tmem_d = tmem_base + (uint32_t)(acc * 256);
                for (int kb = 0; kb < num_kb; ++kb) {
                    ok = ptx::mbar_wait(ptx::smem_u32(&tail->full[stage]), phase, abort_flag, status, 42);
                    if (!ok) break;
                    ptx::tc_fence_after();
                    if (lane == 0) {
                        const uint32_t sa = base + stage * I8_STAGE_BYTES, sb = sa + I8_OPERAND_BYTES;
#pragma unroll
                        for (int k = 0; k < 4; ++k)  // 32 integers = 32 bytes inside the 128-byte swizzled row
                            ptx::mma_i8_ss_pair(tmem_d, ptx::make_smem_desc(sa + k * 32, 16, 1024, 2),
                                                ptx::make_smem_desc(sb + k * 32, 16, 1024, 2), idesc, (kb | k) != 0 ? 1u : 0u);
                        ptx::mma_commit_pair(ptx::smem_u32(&tail->empty[stage]), (uint16_t)3);
                    }
                    __syncwarp();
                    if (++stage == I8_STAGES) { stage = 0; phase ^= 1u; }
                }
                if (!ok) break;
                if (lane == 0) ptx::mma_commit_pair(ptx::smem_u32(&tail->tmem_full[acc]), (uint16_t)3);
                __syncwarp();
            }
        }
    } else {
        const int q = warp & 3;
        const uint32_t leader_empty0 = ptx::map_to_cta(ptx::smem_u32(&tail->tmem_empty[0]), 0);
        const uint32_t leader_empty1 = ptx::map_to_cta(ptx::smem_u32(&tail->tmem_empty[1]), 0);
        float* cs = epi + (warp - 2) * 512;  // scales of the tile's 256 columns, then their bias
        uint8_t* turn = turns + (warp - 2) * I8_TURN_BYTES;
        const bool vec = ((int64_t)out * sizeof(T)) % 16 == 0 && (reinterpret_cast<uintptr_t>(y) & 15u) == 0;
        bool ok = true;
        int t = 0;
        for (int tile = pair; tile < total_tiles && ok; tile += num_pairs, ++t) {
            int tm, tn;
            i8_tile_coords(tile, tiles_m, tiles_n, tm, tn);
            const int row = tm * 256 + (int)cta * 128 + q * 32 + lane, n0 = tn * 256;
            const float rs = row < rows ? xs[row] : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int n = n0 + i * 32 + lane;
                cs[i * 32 + lane] = n < out ? ws[n] : 0.0f;
                cs[256 + i * 32 + lane] = bias != nullptr && n < out ? as_f32(bias[n]) : 0.0f;
            }
            __syncwarp();
            const int acc = t & 1;
            ok = ptx::mbar_wait(ptx::smem_u32(&tail->tmem_full[acc]), (uint32_t)(t >> 1) & 1u, abort_flag, status, 44);
            if (!ok) break;
            ptx::tc_fence_after();
            const uint32_t taddr = tmem_base + (uint32_t)(acc * 256) + ((uint32_t)(q * 32) << 16);
            constexpr int PARTS = 4 / (int)sizeof(T);  // accumulator reads of 32 columns per 128 bytes of a row
            auto put = [&](auto out_of) {
#pragma unroll 1
                for (int c = 0; c < 8; c += PARTS) {
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        const int col = (c + part) * 32;
                        uint32_t r[32];
                        ptx::tmem_ld_32x32b_x32(taddr + (uint32_t)col, r);
                        ptx::tmem_ld_wait();
                        float v[32];
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 s4 = *reinterpret_cast<const float4*>(cs + col + j);
                            const float4 b4 = *reinterpret_cast<const float4*>(cs + 256 + col + j);
                            v[j] = out_of((int)r[j], rs, s4.x, b4.x);
                            v[j + 1] = out_of((int)r[j + 1], rs, s4.y, b4.y);
                            v[j + 2] = out_of((int)r[j + 2], rs, s4.z, b4.z);
                            v[j + 3] = out_of((int)r[j + 3], rs, s4.w, b4.w);
                        }
                        turn_in(turn + lane * I8_TURN_ROW, v, part, T());
                    }
                    if (c + PARTS == 8) {  // the last of the accumulator has been read: the MMA warp may have it back
                        ptx::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) ptx::mbar_arrive_cluster(acc ? leader_empty1 : leader_empty0);
                    } else {
                        __syncwarp();
                    }
                    const int col = c * 32, row0 = row - lane;
                    if (row0 < rows && n0 + col < out)
                        turn_out(turn, y + (int64_t)row0 * out + n0 + col, (int64_t)out, rows - row0, out - n0 - col, vec, lane);
                    __syncwarp();  // the turn buffer and, after the last chunk, the column scales may be overwritten
                }
            };
            // a loop of its own for huge rows: a test inside one loop took [8192, 64] x [12288, 64] from 89 to 99 us
            if (__any_sync(0xffffffffu, fabsf(rs) >= kHugeScale)) put([](int a, float x, float w, float b) { return int8_out(a, x, w, b); });
            else put([](int a, float x, float w, float b) { return int8_out_usual(a, x, w, b); });
        }
    }

    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync_all();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem_base, 512);
    }
}

// ---------------------------------------------------------------------------------------------------------
// One row or two: no tensor cores, one launch. A block owns consecutive output channels; its 32 warps take their weight rows
// in pieces of 2 KiB, four 16-byte loads per lane straight into registers, the next piece under way while one is
// multiplied (dp4a): 128 KiB in flight per SM, as much as an SM's share of a [4096, 4096] weight, and the last turn is
// never more than one piece long. The first pieces are requested before the block quantises the tokens into shared
// memory: each block repeats that small work, which saves a launch and a wait. Pieces' sums meet in shared memory (integer
// additions: their order does not matter). [1, 4096] x [4096, 4096]: 5.9 us, x [11008, 4096]: 10.2 us, [1, 11008] x [4096,
// 11008]: 11.0 us back to back; from the end of the kernel ahead the weights are in within 5.8 us of the 10.2. The 64 registers of
// 1024 threads do not hold both pieces beside the quantiser: 20 to 92 bytes per thread are spilled around it.
// ---------------------------------------------------------------------------------------------------------
constexpr int GV_WARPS = 32, GV_THREADS = 32 * GV_WARPS;
constexpr int GV_LOADS = 4, GV_PIECE = GV_LOADS * 512;
constexpr int GV_X_BYTES = 128 * 1024;  // room for the quantised tokens
constexpr int GV_MAX_ROWS = 2;
constexpr int GV_CHANNELS = 2048;       // most output channels of a block
// Called back to back: 0 / 64 / 128 / 512 KiB fetched ahead per block take [1, 4096] x [4096, 4096] 6.5 / 5.9 / 6.3 / 6.3 us
// and x [11008, 4096] 11.3 / 10.2 / 10.0 / 11.5 us.
constexpr int GV_AHEAD_BYTES = 64 * 1024;

__device__ __forceinline__ int4 ld_weights(const int8_t* p) {
    int4 v;
    asm volatile("ld.global.L1::no_allocate.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

template <typename T, int ROWS>
__global__ void __launch_bounds__(GV_THREADS, 1)
int8_stream_kernel(const T* x, int64_t ld, const int8_t* wq, const float* ws, const T* bias, T* y, int in, int out,
                   int pitch, int vec) {
    extern __shared__ __align__(16) uint8_t xq[];  // [ROWS][pitch]
    __shared__ uint32_t part[ROWS][GV_WARPS];
    __shared__ int sums[ROWS][GV_CHANNELS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    ptx::launch_dependents();
    const int first = (int)((int64_t)out * blockIdx.x / gridDim.x);
    const int channels = (int)((int64_t)out * (blockIdx.x + 1) / gridDim.x) - first;
    if (lane == 0) {
        // while the kernel ahead finishes, the head of this block's weights comes as far as L2
        const int64_t bytes = min((int64_t)channels * pitch, (int64_t)GV_AHEAD_BYTES), at = (int64_t)warp * (GV_AHEAD_BYTES / GV_WARPS);
        if (at < bytes)
            ptx::prefetch_l2(wq + (int64_t)first * pitch + at, (uint32_t)min(bytes - at, (int64_t)(GV_AHEAD_BYTES / GV_WARPS)));
    }
    ptx::dependency_wait();
    const int pieces = (pitch + GV_PIECE - 1) / GV_PIECE;
    const int row_step = GV_WARPS / pieces, piece_step = GV_WARPS % pieces;
    int4 w[2][GV_LOADS];
    // the piece to fetch next, and the piece to multiply next: numbered row by row, every 32nd is this warp's
    int fr = warp / pieces, fp = warp % pieces, mr = fr, mp = fp;
    auto advance = [&](int& r, int& p) {
        r += row_step;
        p += piece_step;
        if (p >= pieces) { p -= pieces; ++r; }
    };
    auto fetch = [&](int4 (&dst)[GV_LOADS]) {
        const int at = fp * GV_PIECE + lane * 16;
        const int8_t* src = wq + (int64_t)(first + fr) * pitch + at;
#pragma unroll
        for (int j = 0; j < GV_LOADS; ++j)
            dst[j] = fr < channels && at + j * 512 < pitch ? ld_weights(src + j * 512) : make_int4(0, 0, 0, 0);
        advance(fr, fp);
    };
    fetch(w[0]);
    fetch(w[1]);
    for (int i = threadIdx.x; i < ROWS * GV_CHANNELS; i += GV_THREADS) (&sums[0][0])[i] = 0;

    // the tokens, quantised
    uint32_t top[ROWS];
#pragma unroll
    for (int t = 0; t < ROWS; ++t) top[t] = 0;
    const int nv = vec ? in >> 3 : 0;
    for (int v = threadIdx.x; v < nv; v += GV_THREADS)
#pragma unroll
        for (int t = 0; t < ROWS; ++t) {
            Raw8<T> r;
            r.load(x + t * ld + 8 * v);
            top[t] = top8(r, top[t]);
        }
#pragma unroll
    for (int t = 0; t < ROWS; ++t) top[t] = top_bits(T(), top[t]);
    for (int k = 8 * nv + threadIdx.x; k < in; k += GV_THREADS)
#pragma unroll
        for (int t = 0; t < ROWS; ++t) top[t] = max(top[t], magnitude_bits(as_f32(x[t * ld + k])));
#pragma unroll
    for (int t = 0; t < ROWS; ++t) {
        top[t] = __reduce_max_sync(0xffffffffu, top[t]);
        if (lane == 0) part[t][warp] = top[t];
    }
    __syncthreads();
    float xs[ROWS];
#pragma unroll
    for (int t = 0; t < ROWS; ++t) {
        top[t] = __reduce_max_sync(0xffffffffu, part[t][lane]);
        const RowScale rs = row_scale<T>(__uint_as_float(top[t]));
        const bool usable = top[t] < 0x7f800000u && top[t] != 0;
        xs[t] = top[t] < 0x7f800000u ? __fdiv_rn(rs.a, 127.0f) : nan_f32();
        for (int v = threadIdx.x; v < nv; v += GV_THREADS) {
            Raw8<T> r;
            r.load(x + t * ld + 8 * v);
            *reinterpret_cast<uint2*>(xq + t * pitch + 8 * v) = usable ? quantise8(r, rs) : make_uint2(0u, 0u);
        }
        for (int k = 8 * nv + threadIdx.x; k < pitch; k += GV_THREADS)
            xq[t * pitch + k] = (uint8_t)(k < in && usable ? quantise(T(), as_f32(x[t * ld + k]), rs) : 0);
    }
    __syncthreads();

    auto multiply = [&](const int4 (&v)[GV_LOADS]) {
        const int at = mp * GV_PIECE + lane * 16;
        int acc[ROWS];
#pragma unroll
        for (int t = 0; t < ROWS; ++t) acc[t] = 0;
#pragma unroll
        for (int j = 0; j < GV_LOADS; ++j)
            if (at + j * 512 < pitch) {
#pragma unroll
                for (int t = 0; t < ROWS; ++t) {
                    const int4 q = *reinterpret_cast<const int4*>(xq + t * pitch + at + j * 512);
                    acc[t] = __dp4a(v[j].x, q.x, acc[t]);
                    acc[t] = __dp4a(v[j].y, q.y, acc[t]);
                    acc[t] = __dp4a(v[j].z, q.z, acc[t]);
                    acc[t] = __dp4a(v[j].w, q.w, acc[t]);
                }
            }
#pragma unroll
        for (int t = 0; t < ROWS; ++t) {
            const int sum = __reduce_add_sync(0xffffffffu, acc[t]);
            if (lane == 0) atomicAdd(&sums[t][mr], sum);
        }
        advance(mr, mp);
    };
    while (mr < channels) {
        multiply(w[0]);
        fetch(w[0]);
        if (mr >= channels) break;
        multiply(w[1]);
        fetch(w[1]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < channels; i += GV_THREADS) {
        const float cs = ws[first + i], cb = bias != nullptr ? as_f32(bias[first + i]) : 0.0f;
#pragma unroll
        for (int t = 0; t < ROWS; ++t) y[(int64_t)t * out + first + i] = (T)int8_out(sums[t][i], xs[t], cs, cb);
    }
}

// ---------------------------------------------------------------------------------------------------------
// Few rows: D[128 PAIR output channels, BN tokens] = wq . xq^T, the reduction cut over the CTAs of a cluster.
//
// The weight is what has to be read, so it is the 128-row operand and the tokens are the narrow one. A tile's K range
// is cut into `split` parts so that about all SMs stream weights; the parts' CTAs form a cluster, each leaves its partial
// sums (exact integers) in its shared memory, and after a cluster barrier every CTA adds up its share of the token
// columns (column c belongs to part c mod split) over all parts and writes them: one launch, no workspace, any order of
// arrival gives the same sum. (Stores into the owner's shared memory instead save the second barrier but cost
// more than it: [64, 4096] x [4096, 4096] 9.5 -> 15.9 us.)
// PAIR = 2 (256 tokens): two CTAs share a 256 x 256 tile (cta_group::2) and each loads half of the tokens, for long
// reductions over some hundred rows, where the traffic into the SMs is what bounds the tile.
// The weight loads of the first stages are issued before the kernel waits for the quantised rows.
// [16, 4096] x [11008, 4096]: 13.3 us back to back, of which 8.1 the stream of weights (5.5 TB/s), 0.6 setting up, 1.6 joining
// and writing, the rest handing over between launches; [16, 4096] x [4096, 4096]: 7.9 us, [64, 4096] x [4096, 4096]: 9.6 us.
// ---------------------------------------------------------------------------------------------------------
template <int BN, int PAIR>
struct I8Few {
    static constexpr int STAGES = BN > 64 ? 6 : (BN <= 32 ? 5 : 4);  // up to 64 tokens 93 to 103 KB: two CTAs per SM
    static constexpr int X_ROWS = BN / PAIR;
    static constexpr int STAGE_BYTES = I8_OPERAND_BYTES + X_ROWS * I8_BK;
    static constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
    static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 + 256 + 1024;
    static constexpr int MAX_SPLIT = PAIR == 2 ? 2 : 8;  // clusters of at most eight CTAs, of four where one fills an SM
    static_assert(128 * BN * 4 <= STAGES * STAGE_BYTES, "partial sums reuse the ring");
};

template <int STAGES>
struct I8FewTail {
    uint64_t full[STAGES];
    uint64_t empty[STAGES];
    uint64_t tmem_full;
    uint32_t tmem_base;
    int abort_flag;
    int any_huge;   // one of the scales is beyond kHugeScale
    float xs[256];  // scales of the tile's tokens
};

// Four consecutive output channels of one token.
__device__ __forceinline__ void store4(__nv_bfloat16* dst, const float (&v)[4], int valid, bool vec) {
    if (vec && valid >= 4) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < valid) dst[i] = __float2bfloat16_rn(v[i]);
    }
}
__device__ __forceinline__ void store4(float* dst, const float (&v)[4], int valid, bool vec) {
    if (vec && valid >= 4) {
        *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < valid) dst[i] = v[i];
    }
}

template <typename T, int BN, int PAIR>
__global__ void __launch_bounds__(I8_THREADS, BN > 64 ? 1 : 2)
int8_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                const float* xs, const float* __restrict__ ws, const T* __restrict__ bias, T* y, int rows, int out,
                int pitch, int split, int tiles_t, int32_t* status) {
    using C = I8Few<BN, PAIR>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = ptx::smem_u32(smem_raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw_addr);
    auto* tail = reinterpret_cast<I8FewTail<C::STAGES>*>(base_ptr + C::STAGES * C::STAGE_BYTES);
    volatile int* abort_flag = &tail->abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool clustered = PAIR * split > 1;
    const int crank = clustered ? (int)ptx::cluster_ctarank() : 0;
    const int half = PAIR == 2 ? crank & 1 : 0, part_no = crank / PAIR;
    const uint32_t leader = (uint32_t)(part_no * PAIR);
    const int tile = blockIdx.x / (PAIR * split);
    const int n0 = (tile / tiles_t * PAIR + half) * 128, t0 = tile % tiles_t * BN;
    const int num_kb = (pitch + I8_BK - 1) / I8_BK;
    const int kb0 = (int)((int64_t)num_kb * part_no / split), kb1 = (int)((int64_t)num_kb * (part_no + 1) / split);
    const int ahead = min(C::STAGES, kb1 - kb0);

    auto load = [&](int stage, int kb, bool weights, bool tokens) {
        const uint32_t local = ptx::smem_u32(&tail->full[stage]);
        const uint32_t sw = base + stage * C::STAGE_BYTES, sx = sw + I8_OPERAND_BYTES;
        if (PAIR == 2) {
            const uint32_t bar = ptx::map_to_cta(local, leader);
            if (weights) {
                if (half == 0) ptx::mbar_arrive_expect_tx(local, 2 * C::STAGE_BYTES);
                ptx::tma_load_2d_pair(sw, &tmW, bar, kb * I8_BK, n0);
            }
            if (tokens) ptx::tma_load_2d_pair(sx, &tmX, bar, kb * I8_BK, t0 + half * C::X_ROWS);
        } else {
            if (weights) {
                ptx::mbar_arrive_expect_tx(local, C::STAGE_BYTES);
                ptx::tma_load_2d(sw, &tmW, local, kb * I8_BK, n0);
            }
            if (tokens) ptx::tma_load_2d(sx, &tmX, local, kb * I8_BK, t0);
        }
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            ptx::mbar_init(ptx::smem_u32(&tail->full[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&tail->empty[s]), 1);
        }
        ptx::mbar_init(ptx::smem_u32(&tail->tmem_full), 1);
        tail->abort_flag = tail->any_huge = 0;
        ptx::fence_barrier_init();
        if (PAIR == 1)  // nobody else's barriers are involved: the weights are on their way before the block is set up
            for (int s = 0; s < ahead; ++s) load(s, kb0 + s, true, false);
    }
    if (warp == 1) {
        if (PAIR == 2) {
            ptx::tmem_alloc_pair(ptx::smem_u32(&tail->tmem_base), C::TMEM_COLS);
            ptx::tmem_relinquish_pair();
        } else {
            ptx::tmem_alloc(ptx::smem_u32(&tail->tmem_base), C::TMEM_COLS);
            ptx::tmem_relinquish();
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (PAIR == 2) ptx::cluster_sync_all();  // the other CTA's copies and commits arrive on this CTA's barriers
    ptx::tc_fence_after();
    ptx::launch_dependents();
    const uint32_t tmem_base = tail->tmem_base;

    if (warp == 0) {
        if (PAIR == 2 && lane == 0)
            for (int s = 0; s < ahead; ++s) load(s, kb0 + s, true, false);
        ptx::dependency_wait();
        if (lane == 0)
            for (int s = 0; s < ahead; ++s) load(s, kb0 + s, false, true);
        __syncwarp();
        int stage = 0;
        uint32_t phase = 0;  // the first round of the ring is under way: wait for its release
        bool ok = true;
        for (int kb = kb0 + ahead; kb < kb1; ++kb) {
            ok = ptx::mbar_wait(ptx::smem_u32(&tail->empty[stage]), phase, abort_flag, status, 51);
            if (!ok) break;
            if (lane == 0) load(stage, kb, true, true);
            __syncwarp();
            if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok) for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else if (warp == 1 && half == 0) {
        constexpr uint32_t idesc = ptx::make_idesc_i8(128 * PAIR, BN);
        const uint16_t both = (uint16_t)(3u << leader);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            ok = ptx::mbar_wait(ptx::smem_u32(&tail->full[stage]), phase, abort_flag, status, 52);
            if (!ok) break;
            ptx::tc_fence_after();
            if (lane == 0) {
                const uint32_t sw = base + stage * C::STAGE_BYTES, sx = sw + I8_OPERAND_BYTES;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint64_t wd = ptx::make_smem_desc(sw + k * 32, 16, 1024, 2), xd = ptx::make_smem_desc(sx + k * 32, 16, 1024, 2);
                    const uint32_t add = (kb != kb0 || k != 0) ? 1u : 0u;
                    if (PAIR == 2) ptx::mma_i8_ss_pair(tmem_base, wd, xd, idesc, add);
                    else ptx::mma_i8_ss(tmem_base, wd, xd, idesc, add);
                }
                if (PAIR == 2) ptx::mma_commit_pair(ptx::smem_u32(&tail->empty[stage]), both);
                else ptx::mma_commit(ptx::smem_u32(&tail->empty[stage]));
            }
            __syncwarp();
            if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
        if (ok && lane == 0) {
            if (PAIR == 2) ptx::mma_commit_pair(ptx::smem_u32(&tail->tmem_full), both);
            else ptx::mma_commit(ptx::smem_u32(&tail->tmem_full));
        }
        __syncwarp();
    }
    // everything the MMAs read has been read once the accumulator is complete: the ring is free for partial sums,
    // laid out [token][128 channels]
    int* part = reinterpret_cast<int*>(base_ptr);
    // output: a warp takes whole token columns, a lane four channels of each; their scales are fetched ahead
    const int n = n0 + 4 * lane, valid = out - n;
    float cs[4], cb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        cs[i] = i < valid ? ws[n + i] : 0.0f;
        cb[i] = bias != nullptr && i < valid ? as_f32(bias[n + i]) : 0.0f;
    }
    ptx::dependency_wait();
    if (warp >= 2) {
        for (int c = threadIdx.x - 64; c < BN; c += 128) {
            const float scale = t0 + c < rows ? xs[t0 + c] : 0.0f;
            tail->xs[c] = scale;
            if (fabsf(scale) >= kHugeScale) tail->any_huge = 1;
        }
        const bool done = ptx::mbar_wait(ptx::smem_u32(&tail->tmem_full), 0, abort_flag, status, 54);
        if (done) {
            ptx::tc_fence_after();
            const int q = warp & 3;
            const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16);
            const int last = min(BN, rows - t0);
#pragma unroll 1
            for (int c = 0; c < last; c += 16) {
                uint32_t r[16];
                ptx::tmem_ld_32x32b_x16(taddr + (uint32_t)c, r);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) part[(c + j) * 128 + q * 32 + lane] = (int)r[j];
            }
        }
    }
    ptx::tc_fence_before();
    if (split > 1) {
        __syncwarp();
        ptx::cluster_sync_all();
    } else {
        __syncthreads();
    }
    if (*abort_flag == 0) {
        const bool vec = out % 4 == 0 && (reinterpret_cast<uintptr_t>(y) & (4 * sizeof(T) - 1)) == 0;
        const uint32_t mine = ptx::smem_u32(part) + (uint32_t)lane * 16u;
        const int last = min(BN, rows - t0);
        constexpr int GROUP = 4, WARPS = I8_THREADS / 32;  // columns whose loads are in flight together; all warps take part
        for (int c0 = part_no + split * warp; c0 < last; c0 += WARPS * GROUP * split) {
            int4 sum[GROUP];
#pragma unroll
            for (int g = 0; g < GROUP; ++g) sum[g] = make_int4(0, 0, 0, 0);
            for (int s = 0; s < split; ++s) {
                const uint32_t peer = clustered ? ptx::map_to_cta(mine, (uint32_t)(s * PAIR + half)) : mine;
                int4 v[GROUP];
#pragma unroll
                for (int g = 0; g < GROUP; ++g) {
                    const int c = c0 + WARPS * split * g;
                    v[g] = make_int4(0, 0, 0, 0);
                    if (c < last) v[g] = ptx::ld_shared_cluster_v4(peer + (uint32_t)c * 512u);
                }
#pragma unroll
                for (int g = 0; g < GROUP; ++g) {
                    sum[g].x += v[g].x; sum[g].y += v[g].y; sum[g].z += v[g].z; sum[g].w += v[g].w;
                }
            }
            auto put = [&](auto out_of) {
#pragma unroll
                for (int g = 0; g < GROUP; ++g) {
                    const int c = c0 + WARPS * split * g;
                    if (c < last && valid > 0) {
                        const float rs = tail->xs[c];
                        const float v[4] = {out_of(sum[g].x, rs, cs[0], cb[0]), out_of(sum[g].y, rs, cs[1], cb[1]),
                                            out_of(sum[g].z, rs, cs[2], cb[2]), out_of(sum[g].w, rs, cs[3], cb[3])};
                        store4(y + (int64_t)(t0 + c) * out + n, v, valid, vec);
                    }
                }
            };
            // one test for the tile, not one per column: the columns' loads, products and stores stay interleaved
            if (tail->any_huge) put([](int a, float xs, float ws, float b) { return int8_out(a, xs, ws, b); });
            else put([](int a, float xs, float ws, float b) { return int8_out_usual(a, xs, ws, b); });
        }
    }
    __syncwarp();
    if (clustered) ptx::cluster_sync_all();  // this CTA's partial sums are read no more
    else __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after();
        if (PAIR == 2) ptx::tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
        else ptx::tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
}

// An address that elements of the type may start at (4 bytes for SF_F32 and 32-bit integers, 2 for SF_BF16).
static bool on_elements(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == SF_F32 ? 4 : 2) == 0; }

// One row or two, whose quantised form fits into shared memory, take the kernel without a workspace.
static bool takes_stream(int64_t rows, int64_t in) { return rows <= GV_MAX_ROWS && rows * ((in + 15) / 16 * 16) <= GV_X_BYTES; }

static int check_int8(const char* who, int64_t rows, int64_t in, int64_t out) {
    if (rows < 0 || in <= 0 || out <= 0) return fail(SF_ERR_BAD_ARG, "%s: rows must not be negative, in and out positive", who);
    if (rows > (1 << 30) || out > (1 << 30)) return fail(SF_ERR_UNSUPPORTED, "%s: rows or out beyond 2^30", who);
    if (in > SF_INT8_MAX_IN)
        return fail(SF_ERR_UNSUPPORTED, "%s: in=%lld: beyond %lld the 32-bit sum of 8-bit products could overflow", who,
                    (long long)in, (long long)SF_INT8_MAX_IN);
    return SF_OK;
}

// Launch that may be set up while the kernel before it in the stream still runs; every kernel launched this way waits for
// that one's results (griddepcontrol.wait, in every block) before it touches any of them. The product behind the
// quantiser loads weights before it waits: the quantiser lets it start only after its own wait, so whatever wrote the
// weights is complete by then. Called on its own the product is an ordinary launch (dependent = false).
template <typename... KArgs, typename... Args>
static cudaError_t launch_dependent(void (*kern)(KArgs...), int grid, int threads, int smem, int cluster, bool dependent,
                                    cudaStream_t st, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (dependent) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.numAttrs = (unsigned)n;
    cfg.attrs = attr;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

// Rows that start on 16-byte boundaries and are a multiple of 8 long move in 16-byte accesses.
static bool rows_vectorise(const void* x, int dtype, int64_t ld, int64_t rows, int64_t cols) {
    const int64_t esize = dtype == SF_F32 ? 4 : 2;
    return aligned16(x) && cols % 8 == 0 && (rows == 1 || ld * esize % 16 == 0);
}

template <typename T>
static int quantize_typed(const T* x, bool vec, int64_t ld, int8_t* q, float* scale, int64_t rows, int64_t cols,
                          cudaStream_t st) {
    const int pitch = (int)((cols + 15) / 16 * 16);
    // A warp per row up to 1024 elements, a block per row up to 32768, the row and the next one held in registers: [8192, 4096]
    // bf16: 17.7 us (5.7 TB/s) with 128 threads per row, 18.9 with 256, 21.5 with 512; [8192, 11008]: 44.3 us (6.1 TB/s). fp32
    // rows take twice the registers: [8192, 4096] 30.5 us (5.5 TB/s), [8192, 11008] 106 us (4.2 TB/s). In fp32 beyond 16384 two rows do
    // not fit the 64 registers of 1024 threads (368 bytes of spills per thread): [2048, 20000] 80 us, [2048, 32768] 101 us
    // (2.5 and 3.3 TB/s).
#define SF_I8_QUANT(THREADS, TPR, NV)                                                                                 \
    do {                                                                                                              \
        auto kern = int8_quantize_vec_kernel<T, THREADS, TPR, NV>;                                                    \
        const int64_t need = (rows + THREADS / TPR - 1) / (THREADS / TPR);                                            \
        const int grid = (int)std::min<int64_t>(need, (int64_t)sm_count() * (kQVecResident / THREADS));               \
        SF_CHECK_CUDA(launch_dependent(kern, grid, THREADS, 0, 1, true, st, x, ld, q, scale, (int)rows, (int)cols, pitch)); \
    } while (0)
    if (vec && cols <= 1024) {
        SF_I8_QUANT(256, 32, 4);
    } else if (vec && cols <= 4096) {
        SF_I8_QUANT(128, 128, 4);
    } else if (vec && cols <= 12288) {
        SF_I8_QUANT(256, 256, 6);
    } else if (vec && cols <= 16384) {
        SF_I8_QUANT(512, 512, 4);
    } else if (vec && cols <= 32768) {
        SF_I8_QUANT(1024, 1024, 4);
#undef SF_I8_QUANT
    // Unaligned rows; a warp per row where there are many short ones. Blocks leave after their rows, with nothing under way
    // while they reduce and round: [8192, 4095] bf16 30 us (3.4 TB/s), fp32 35 us (4.8 TB/s), [512, 11007] bf16 7.3 us.
#define SF_I8_QUANT_ANY(TPR, NV)                                                                                      \
    SF_CHECK_CUDA(launch_dependent(int8_quantize_any_kernel<T, TPR, NV>, (int)((rows + kQThreads / TPR - 1) / (kQThreads / TPR)), \
                                   kQThreads, 0, 1, true, st, x, ld, q, scale, (int)rows, (int)cols, pitch))
    } else if (pitch <= 8 * 31 * 4 && rows >= 16 * (int64_t)sm_count()) {
        SF_I8_QUANT_ANY(32, 4);
    } else if (pitch <= 8 * 31 * 4 * 5) {
        SF_I8_QUANT_ANY(128, 5);
    } else if (pitch <= 8 * 31 * 8 * 6) {
        SF_I8_QUANT_ANY(256, 6);
    } else {
        SF_I8_QUANT_ANY(256, 0);
    }
#undef SF_I8_QUANT_ANY
    return SF_OK;
}
static int quantize_impl(const void* x, int dtype, int64_t ld, int8_t* q, float* scale, int64_t rows, int64_t cols,
                         cudaStream_t st) {
    const bool vec = rows_vectorise(x, dtype, ld, rows, cols);
    return dtype == SF_F32 ? quantize_typed((const float*)x, vec, ld, q, scale, rows, cols, st)
                           : quantize_typed((const __nv_bfloat16*)x, vec, ld, q, scale, rows, cols, st);
}

// Raises a kernel's dynamic shared memory limit once per device and thread.
#define SF_I8_SMEM(kern, bytes)                                                                                     \
    do {                                                                                                            \
        static thread_local int configured_dev = -1;                                                                \
        int dev = 0;                                                                                                \
        SF_CHECK_CUDA(cudaGetDevice(&dev));                                                                         \
        if (configured_dev != dev) {                                                                                \
            SF_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));          \
            configured_dev = dev;                                                                                   \
        }                                                                                                           \
    } while (0)

template <typename T>
static int launch_pair(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, const void* bias, void* y,
                       int64_t rows, int pitch, int64_t out, int32_t* status, bool dependent, cudaStream_t st) {
    CUtensorMap tmA, tmB;
    if (int rc = make_byte_tensor_map(&tmA, xq, pitch, rows, 128)) return rc;
    if (int rc = make_byte_tensor_map(&tmB, wq, pitch, out, 128)) return rc;
    const int64_t tiles = ((rows + 255) / 256) * ((out + 255) / 256);
    if (tiles > 0x3fffffff) return fail(SF_ERR_UNSUPPORTED, "8-bit product: more than 2^30 tiles");
    const int pairs = (int)std::min<int64_t>(tiles, sm_count() / 2);
    auto kern = int8_pair_kernel<T>;
    SF_I8_SMEM(kern, I8_PAIR_SMEM);
    // the kernel's own cluster attribute (two CTAs) holds
    SF_CHECK_CUDA(launch_dependent(kern, 2 * pairs, I8_THREADS, I8_PAIR_SMEM, 0, dependent, st, tmA, tmB, xs, ws, (const T*)bias, (T*)y,
                                   (int)rows, (int)out, pitch, status));
    return SF_OK;
}

template <typename T, int BN, int PAIR>
static int launch_few(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, const void* bias, void* y,
                      int64_t rows, int pitch, int64_t out, int32_t* status, bool dependent, cudaStream_t st) {
    using C = I8Few<BN, PAIR>;
    CUtensorMap tmW, tmX;
    if (int rc = make_byte_tensor_map(&tmW, wq, pitch, out, 128)) return rc;
    if (int rc = make_byte_tensor_map(&tmX, xq, pitch, rows, C::X_ROWS)) return rc;
    const int64_t tiles_t = (rows + BN - 1) / BN, tiles = (out + 128 * PAIR - 1) / (128 * PAIR) * tiles_t;
    if (tiles * 8 > 0x7fffffff) return fail(SF_ERR_UNSUPPORTED, "8-bit product: too many tiles");
    // Doubled until most SMs stream weights, as long as every CTA keeps a block of K; and on to two CTAs per SM (tiles of up
    // to 64 tokens), whose loads cover each other's latencies, while each keeps 16 blocks: shorter parts cost more in the join
    // than they save ([64, 4096] x [4096, 4096]: 9.3 us with four parts of 8 blocks, 10.5 with eight of 4).
    const int num_kb = (pitch + I8_BK - 1) / I8_BK;
    const int64_t sms = sm_count();
    int split = 1;
    while (split < C::MAX_SPLIT && 2 * split <= num_kb) {
        const int64_t ctas = tiles * PAIR * split;
        const bool idle = ctas * 4 < sms * (BN > 64 ? 2 : 3);
        const bool room = BN <= 64 && ctas <= sms && num_kb >= 32 * split;
        if (!idle && !room) break;
        split *= 2;
    }
    auto kern = int8_few_kernel<T, BN, PAIR>;
    SF_I8_SMEM(kern, C::SMEM);
    SF_CHECK_CUDA(launch_dependent(kern, (int)(tiles * PAIR * split), I8_THREADS, C::SMEM, PAIR * split, dependent, st, tmW, tmX,
                                   xs, ws, (const T*)bias, (T*)y, (int)rows, (int)out, pitch, split, (int)tiles_t, status));
    return SF_OK;
}

template <typename T, int ROWS>
static int launch_stream(const void* x, int64_t ld, const int8_t* wq, const float* ws, const void* bias, void* y, int64_t in,
                         int64_t out, bool vec, cudaStream_t st) {
    const int pitch = (int)((in + 15) / 16 * 16);
    const int smem = ROWS * pitch;
    auto kern = int8_stream_kernel<T, ROWS>;
    SF_I8_SMEM(kern, GV_X_BYTES);
    // one block per SM; fewer where that leaves a warp less than a piece, more where a block's channels would not fit
    const int64_t pieces = out * ((pitch + GV_PIECE - 1) / GV_PIECE);
    const int grid = (int)std::max(std::min<int64_t>(sm_count(), (pieces + GV_WARPS - 1) / GV_WARPS), (out + GV_CHANNELS - 2) / (GV_CHANNELS - 1));
    SF_CHECK_CUDA(launch_dependent(kern, grid, GV_THREADS, smem, 1, true, st, (const T*)x, ld, wq, ws, (const T*)bias, (T*)y, (int)in,
                                   (int)out, pitch, vec ? 1 : 0));
    return SF_OK;
}
template <typename T>
static int stream_typed(const void* x, int64_t ld, const int8_t* wq, const float* ws, const void* bias, void* y, int64_t rows,
                        int64_t in, int64_t out, bool vec, cudaStream_t st) {
    return rows == 1 ? launch_stream<T, 1>(x, ld, wq, ws, bias, y, in, out, vec, st)
                     : launch_stream<T, 2>(x, ld, wq, ws, bias, y, in, out, vec, st);
}

template <typename T>
static int gemm_typed(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, const void* bias, void* y,
                      int64_t rows, int64_t in, int64_t out, int32_t* status, bool dependent, cudaStream_t st) {
    const int pitch = (int)((in + 15) / 16 * 16);
    if (rows <= 16) return launch_few<T, 16, 1>(xq, xs, wq, ws, bias, y, rows, pitch, out, status, dependent, st);
    if (rows <= 32) return launch_few<T, 32, 1>(xq, xs, wq, ws, bias, y, rows, pitch, out, status, dependent, st);
    // More rows. While 128 x 64 tiles fit the chip at two per SM they are mostly the fastest, but their operands are loaded more
    // often: past 256 rows a long reduction takes 256 x 256 tiles cut in two where those fill half of the SMs and fit all. Beyond
    // that, persistent tiles. Graph times in us of 128 x 64 / cut / persistent tiles, over weights not in L2:
    //   [512, 4096] x [4096, 4096]   17.7 / 18.2 / 19.6     [512, 12288] x [4096, 12288]  39.1 / 30.6 / 41.3
    //   the reduction (8192):  [512, 6144] x [4096, 6144] 22.7 / 22.0 / 25.5, [320, 8192] x [4096, 8192] 26.6 / 23.3 / 29.6
    //   the count (19 to 37):  16 tiles, [320, 8192] x [2048, 8192] 18.1 / 21.9 / 28.8; 48 tiles, [320, 8192] x [6144, 8192]
    //                          28.1 / 33.1 / 30.7
    //   the rows (256):        [128, 8192] x [8192, 8192] 22.1 / 21.6 / 29.9, but [192, 8192] x [8192, 8192] 28.5 / 23.0 / 29.8 and
    //                          [256, 12288] x [6144, 12288] 38.7 / 29.2 / 39.8: at 129 to 256 rows of that length the rule is not
    //                          the best choice.
    const int64_t small = ((out + 127) / 128) * ((rows + 63) / 64), large = ((out + 255) / 256) * ((rows + 255) / 256);
    if (rows > 256 && pitch >= 8192 && large * 4 <= sm_count() && large * 8 >= sm_count())
        return launch_few<T, 256, 2>(xq, xs, wq, ws, bias, y, rows, pitch, out, status, dependent, st);
    if (small <= 2 * (int64_t)sm_count()) return launch_few<T, 64, 1>(xq, xs, wq, ws, bias, y, rows, pitch, out, status, dependent, st);
    return launch_pair<T>(xq, xs, wq, ws, bias, y, rows, pitch, out, status, dependent, st);
}

static int gemm_impl(const int8_t* xq, const float* xs, const int8_t* wq, const float* ws, const void* bias, void* y, int dtype,
                     int64_t rows, int64_t in, int64_t out, int32_t* status, bool dependent, cudaStream_t st) {
    return dtype == SF_F32 ? gemm_typed<float>(xq, xs, wq, ws, bias, y, rows, in, out, status, dependent, st)
                           : gemm_typed<__nv_bfloat16>(xq, xs, wq, ws, bias, y, rows, in, out, status, dependent, st);
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
    if (!on_elements(x, dtype) || !on_elements(scale, SF_F32))
        return fail(SF_ERR_ALIGNMENT, "sf_int8_quantize_rows: x and scale must be aligned to their elements");
    return quantize_impl(x, dtype, ld, q, scale, rows, cols, (cudaStream_t)stream);
}

static int check_product(const char* who, const void* wq, const float* ws, const void* bias, const void* y, int dtype,
                         int64_t rows, int64_t in, int64_t out, const int32_t* status) {
    if (int rc = check_int8(who, rows, in, out)) return rc;
    if (dtype != SF_F32 && dtype != SF_BF16) return fail(SF_ERR_BAD_ARG, "%s: dtype must be SF_F32 or SF_BF16", who);
    if (rows == 0) return SF_OK;
    if (!wq || !ws || !y) return fail(SF_ERR_BAD_ARG, "%s: weight, scales and y must be non-null", who);
    if (!aligned16(wq)) return fail(SF_ERR_ALIGNMENT, "%s: 8-bit operands must be 16-byte aligned", who);
    if (!on_elements(ws, SF_F32) || !on_elements(bias, dtype) || !on_elements(y, dtype) || !on_elements(status, SF_F32))
        return fail(SF_ERR_ALIGNMENT, "%s: scales, bias, y and status must be aligned to their elements", who);
    return SF_OK;
}

int sf_int8_gemm(const int8_t* xq, const float* x_scale, const int8_t* wq, const float* w_scale, const void* bias, void* y,
                 int dtype, int64_t rows, int64_t in, int64_t out, int32_t* status, void* stream) {
    if (int rc = check_product("sf_int8_gemm", wq, w_scale, bias, y, dtype, rows, in, out, status)) return rc;
    if (rows == 0) return SF_OK;
    SF_CHECK_ARG(xq && x_scale, "sf_int8_gemm: xq and x_scale must be non-null");
    if (!aligned16(xq)) return fail(SF_ERR_ALIGNMENT, "sf_int8_gemm: 8-bit operands must be 16-byte aligned");
    if (!on_elements(x_scale, SF_F32)) return fail(SF_ERR_ALIGNMENT, "sf_int8_gemm: x_scale must be aligned to its elements");
    return gemm_impl(xq, x_scale, wq, w_scale, bias, y, dtype, rows, in, out, status, false, (cudaStream_t)stream);
}

int64_t sf_int8_linear_workspace_bytes(int64_t rows, int64_t in) {
    if (rows <= 0 || in <= 0 || takes_stream(rows, in)) return 0;
    return rows * sf_int8_pitch(in) + rows * 4;
}

int sf_int8_linear(const void* x, int64_t ld, const int8_t* wq, const float* w_scale, const void* bias, void* y, int dtype,
                   int64_t rows, int64_t in, int64_t out, void* workspace, int32_t* status, void* stream) {
    if (int rc = check_product("sf_int8_linear", wq, w_scale, bias, y, dtype, rows, in, out, status)) return rc;
    if (rows == 0) return SF_OK;
    const bool stream_rows = takes_stream(rows, in);
    SF_CHECK_ARG(x && (workspace || stream_rows), "sf_int8_linear: x and workspace must be non-null");
    SF_CHECK_ARG(ld >= in || rows == 1, "sf_int8_linear: ld=%lld is smaller than a row", (long long)ld);
    if (!aligned16(workspace)) return fail(SF_ERR_ALIGNMENT, "sf_int8_linear: workspace must be 16-byte aligned");
    if (!on_elements(x, dtype)) return fail(SF_ERR_ALIGNMENT, "sf_int8_linear: x must be aligned to its elements");
    if (stream_rows) {
        const bool vec = rows_vectorise(x, dtype, ld, rows, in);
        return dtype == SF_F32 ? stream_typed<float>(x, ld, wq, w_scale, bias, y, rows, in, out, vec, (cudaStream_t)stream)
                               : stream_typed<__nv_bfloat16>(x, ld, wq, w_scale, bias, y, rows, in, out, vec, (cudaStream_t)stream);
    }
    int8_t* xq = static_cast<int8_t*>(workspace);
    float* xs = reinterpret_cast<float*>(xq + rows * sf_int8_pitch(in));
    if (int rc = quantize_impl(x, dtype, ld, xq, xs, rows, in, (cudaStream_t)stream)) return rc;
    return gemm_impl(xq, xs, wq, w_scale, bias, y, dtype, rows, in, out, status, true, (cudaStream_t)stream);
}

}  // extern "C"
