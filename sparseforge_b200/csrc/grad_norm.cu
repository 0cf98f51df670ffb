// Global norm of many gradient tensors, and clipping by it.
//
//   norm = sqrt(sum over every element of every tensor of g^2)      (or max |g|)
//   c    = min(1, max_norm / (norm + 1e-6)),   out = g * c           (c to 24 bits, the product to fp32 and then to out's type)
//
// The tensors of one call are described by a table that travels in the kernel's parameters: no copy of
// pointers to the device, so a call is one launch for the norm and one for the scaling, and can be captured.
// A tensor is cut into chunks of equal length; the chunks of all tensors are numbered through and dealt out
// round robin to a grid of one resident wave, so 4096-element vectors and 45-million-element matrices share a launch.
//
// Range and order of the sum of squares: eight squares are added in fp32 (a bf16 square is exact there), the sums of
// eight in fp64. Where the fp32 sum of eight leaves [2^-100, 2^120] its elements are squared in fp64 instead, so
// neither large nor tiny gradients (whose squares leave fp32) change the norm. Partial sums have one slot per block and
// are added in one fixed order: the result does not depend on timing.
//
// Both passes are bound by HBM. One decoder layer in bf16 (202 M elements): norm 64 us (6.3 TB/s), norm and clipping into
// other buffers 193 us (three passes over 405 MB, 6.3 TB/s); 150 tensors of 1.9 M elements in all: 6 and 10 us. From a
// captured graph, without the host's share.
#include <cstdlib>

#include <algorithm>
#include <memory>
#include <new>

#include "common.cuh"
#include "ptx_sm100.cuh"

namespace sf {

constexpr int kGnThreads = 512;
constexpr int kGnSlots = 1024;       // partial results one launch may write (its largest grid)
constexpr int kGnVec = 8;            // elements per access group: 16 bytes of bf16, 32 of fp32
// Loads in flight. Norm: 4 blocks of 512 threads per SM with two 16-byte loads each (bf16, four decoder layers, 1.62 GB:
// 265 us = 6.1 TB/s; 2 blocks with four loads 282 us, 3 blocks with four 421 us, 2 blocks with eight 495 us). Scaling: 2
// blocks with four (fp32 in and out, one layer: 256 us; 4 blocks with two 313 us; bf16 the same either way).
constexpr int kGnNormBlocks = 4, kGnNormBatch = 2;
constexpr int kGnClipBlocks = 2, kGnClipBatch = 4;
constexpr int kGnChunkUnit = kGnThreads * kGnVec;

enum { GN_L2 = SF_NORM_L2, GN_INF = SF_NORM_INF };

struct GnTensor {
    const void* in;
    void* out;
    int64_t n;
};
// kind bits of a table entry; from bit 4 on: elements before the first one that is on a 16-byte boundary on both sides
enum { GN_IN_BF16 = 1, GN_OUT_BF16 = 2, GN_VEC = 4, GN_IN_PLACE = 8, GN_HEAD_SHIFT = 4 };
template <int CAP>
struct GnTable {
    GnTensor t[CAP];
    uint32_t first[CAP + 1];  // number of the tensor's first chunk; first[count] = chunks of the launch
    uint8_t kind[CAP];
    uint32_t keep_from;       // chunks from here on are read again soon (the scaling starts with them)
    int all_in_place;         // with a coefficient of 1 there is nothing to do
    int count;
    int chunk;  // elements per chunk, a multiple of kGnChunkUnit
};

template <int CAP>
__device__ __forceinline__ int find_tensor(const GnTable<CAP>& tab, uint32_t c) {
    int lo = 0, hi = tab.count - 1;  // the last tensor whose first chunk is <= c
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

struct NormAcc {
    double sum;
    uint32_t top;  // bit pattern of the largest |g|: ordered like the values, a NaN above infinity
};

// MAXNORM: the largest magnitude instead of the sum of squares
template <bool MAXNORM>
__device__ __forceinline__ void acc8(NormAcc& a, const float (&x)[8]) {
    if (MAXNORM) {
#pragma unroll
        for (int i = 0; i < 8; ++i) a.top = max(a.top, __float_as_uint(x[i]) & 0x7fffffffu);
        return;
    }
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        s0 = fmaf(x[i], x[i], s0);
        s1 = fmaf(x[i + 1], x[i + 1], s1);
    }
    const float s = s0 + s1;
    if (s >= 0x1p-100f && s <= 0x1p120f) {
        a.sum += (double)s;
    } else {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) any |= __float_as_uint(x[i]) << 1;
        if (any != 0) {  // not eight zeros
#pragma unroll
            for (int i = 0; i < 8; ++i) a.sum = fma((double)x[i], (double)x[i], a.sum);
        }
    }
}
template <bool MAXNORM>
__device__ __forceinline__ void acc1(NormAcc& a, float x) {
    if (MAXNORM) a.top = max(a.top, __float_as_uint(x) & 0x7fffffffu);
    else a.sum = fma((double)x, (double)x, a.sum);
}

__device__ __forceinline__ void unpack_bf16(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack_f32(const uint4& a, const uint4& b, float (&x)[8]) {
    x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y); x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
    x[4] = __uint_as_float(b.x); x[5] = __uint_as_float(b.y); x[6] = __uint_as_float(b.z); x[7] = __uint_as_float(b.w);
}

// All threads of a block: sum (or largest) over the block, in an order fixed by the thread numbers. The result
// is valid in thread 0.
__device__ __forceinline__ NormAcc block_merge(NormAcc a, NormAcc* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a.sum += __shfl_down_sync(0xffffffffu, a.sum, o);
        a.top = max(a.top, __shfl_down_sync(0xffffffffu, a.top, o));
    }
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kGnThreads / 32; ++w) {
            a.sum += part[w].sum;
            a.top = max(a.top, part[w].top);
        }
    }
    return a;
}

// Read-only loads of the norm: the chunks that the scaling will read first (the last ones) are left in L2 as usual,
// those before them are marked as the first to go.
__device__ __forceinline__ uint4 ld_norm(const uint4* p, bool keep) {
    return keep ? __ldg(p) : __ldcs(p);
}

template <int CAP, bool MAXNORM>
__global__ void __launch_bounds__(kGnThreads, kGnNormBlocks)
grad_norm_partial_kernel(const __grid_constant__ GnTable<CAP> tab, double* __restrict__ slots) {
    __shared__ NormAcc part[kGnThreads / 32];
    NormAcc acc{0.0, 0u};
    const uint32_t chunks = tab.first[tab.count];
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int ti = find_tensor(tab, c);
        const int64_t at = (int64_t)(c - tab.first[ti]) * tab.chunk;
        const int len = (int)min((int64_t)tab.chunk, tab.t[ti].n - at);
        const int kind = tab.kind[ti];
        // a chunk is a multiple of eight long, so every chunk of a tensor starts as far from a boundary as the first
        const int head = min(len, kind >> GN_HEAD_SHIFT), nv = (kind & GN_VEC) ? (len - head) / kGnVec : 0;
        const bool keep = c >= tab.keep_from;
        if (kind & GN_IN_BF16) {
            const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(tab.t[ti].in) + at;
            const uint4* q = reinterpret_cast<const uint4*>(p + head);
#pragma unroll 1
            for (int v = threadIdx.x; v < nv; v += kGnNormBatch * kGnThreads) {
                uint4 r[kGnNormBatch];  // loads of a batch are in flight together
#pragma unroll
                for (int u = 0; u < kGnNormBatch; ++u)
                    if (v + u * kGnThreads < nv) r[u] = ld_norm(q + v + u * kGnThreads, keep);
#pragma unroll
                for (int u = 0; u < kGnNormBatch; ++u)
                    if (v + u * kGnThreads < nv) {
                        float x[8];
                        unpack_bf16(r[u], x);
                        acc8<MAXNORM>(acc, x);
                    }
            }
#pragma unroll 1
            for (int i = threadIdx.x; i < len - nv * kGnVec; i += kGnThreads)
                acc1<MAXNORM>(acc, __bfloat162float(p[i < head ? i : i + nv * kGnVec]));
        } else {
            const float* p = static_cast<const float*>(tab.t[ti].in) + at;
            const uint4* q = reinterpret_cast<const uint4*>(p + head);
#pragma unroll 1
            for (int v = threadIdx.x; v < nv; v += kGnNormBatch / 2 * kGnThreads) {
                uint4 r[kGnNormBatch];
#pragma unroll
                for (int u = 0; u < kGnNormBatch / 2; ++u)
                    if (v + u * kGnThreads < nv) {
                        r[2 * u] = ld_norm(q + 2 * (v + u * kGnThreads), keep);
                        r[2 * u + 1] = ld_norm(q + 2 * (v + u * kGnThreads) + 1, keep);
                    }
#pragma unroll
                for (int u = 0; u < kGnNormBatch / 2; ++u)
                    if (v + u * kGnThreads < nv) {
                        float x[8];
                        unpack_f32(r[2 * u], r[2 * u + 1], x);
                        acc8<MAXNORM>(acc, x);
                    }
            }
#pragma unroll 1
            for (int i = threadIdx.x; i < len - nv * kGnVec; i += kGnThreads) acc1<MAXNORM>(acc, p[i < head ? i : i + nv * kGnVec]);
        }
    }
    // the kernel behind this one may be set up meanwhile; it waits for these slots
    ptx::launch_dependents();
    acc = block_merge(acc, part);
    if (threadIdx.x == 0) slots[blockIdx.x] = MAXNORM ? (double)__uint_as_float(acc.top) : acc.sum;
}

// The norm from all slots, by every thread block that needs it: each computes the same value. Valid in every thread.
__device__ __forceinline__ double norm_of_slots(const double* slots, int count, bool maxnorm, NormAcc* part,
                                                double* shared_norm) {
    NormAcc a{0.0, 0u};
    for (int i = threadIdx.x; i < count; i += kGnThreads) {
        if (maxnorm) a.top = max(a.top, __float_as_uint((float)slots[i]));
        else a.sum += slots[i];
    }
    a = block_merge(a, part);
    if (threadIdx.x == 0) *shared_norm = maxnorm ? (double)__uint_as_float(a.top) : sqrt(a.sum);
    __syncthreads();
    return *shared_norm;
}

__global__ void __launch_bounds__(kGnThreads)
grad_norm_final_kernel(const double* slots, int count, int kind, float* norm) {
    __shared__ NormAcc part[kGnThreads / 32];
    __shared__ double value;
    ptx::dependency_wait();
    const double v = norm_of_slots(slots, count, kind == GN_INF, part, &value);
    if (threadIdx.x == 0) *norm = (float)v;
}

// out = in * c. slots: the norm's partial results, which every block adds up for itself (norm_out gets the
// value); or, with slots = NULL, the norm is read from norm_in.
template <int CAP>
__global__ void __launch_bounds__(kGnThreads, kGnClipBlocks)
grad_clip_kernel(const __grid_constant__ GnTable<CAP> tab, const double* slots, int slot_count, int kind,
                 const float* norm_in, float* norm_out, double max_norm) {
    __shared__ NormAcc part[kGnThreads / 32];
    __shared__ double value;
    ptx::dependency_wait();
    double norm;
    if (slots != nullptr) {
        norm = norm_of_slots(slots, slot_count, kind == GN_INF, part, &value);
        if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    } else {
        norm = (double)*norm_in;
    }
    const double ratio = max_norm / (norm + 1e-6);
    // A coefficient below fp32's normal range would lose bits (gradients near the top of the range, a small max_norm): it is
    // held 2^126 higher there, and what it gives is moved back by an exact power of two.
    const bool low = ratio < 0x1p-126;
    const float c = ratio >= 1.0 ? 1.0f : (float)(low ? ratio * 0x1p126 : ratio);  // a NaN stays one
    const float back = low ? 0x1p-126f : 1.0f;
    if (c == 1.0f && tab.all_in_place) return;
    const uint32_t chunks = tab.first[tab.count];
    for (uint32_t k = blockIdx.x; k < chunks; k += gridDim.x) {
        const uint32_t ch = chunks - 1 - k;  // backwards: what the norm read last is still in L2
        const int ti = find_tensor(tab, ch);
        const int ent = tab.kind[ti];
        if ((ent & GN_IN_PLACE) && c == 1.0f) continue;
        const int64_t at = (int64_t)(ch - tab.first[ti]) * tab.chunk;
        const int len = (int)min((int64_t)tab.chunk, tab.t[ti].n - at);
        const int head = min(len, ent >> GN_HEAD_SHIFT), nv = (ent & GN_VEC) ? (len - head) / kGnVec : 0;
        const bool ib = ent & GN_IN_BF16, ob = ent & GN_OUT_BF16;
        const char* ip = static_cast<const char*>(tab.t[ti].in) + at * (ib ? 2 : 4);
        char* op = static_cast<char*>(tab.t[ti].out) + at * (ob ? 2 : 4);
        const char* iv = ip + head * (ib ? 2 : 4);
        char* ov = op + head * (ob ? 2 : 4);
        if (ib && ob) {
            const uint4* q = reinterpret_cast<const uint4*>(iv);
            for (int v = threadIdx.x; v < nv; v += kGnClipBatch * kGnThreads) {
                uint4 r[kGnClipBatch];
#pragma unroll
                for (int u = 0; u < kGnClipBatch; ++u)
                    if (v + u * kGnThreads < nv) r[u] = ld_stream16(q + v + u * kGnThreads);
#pragma unroll
                for (int u = 0; u < kGnClipBatch; ++u)
                    if (v + u * kGnThreads < nv) {
                        float x[8];
                        unpack_bf16(r[u], x);
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = x[i] * c * back;
                        Vec8<__nv_bfloat16>::store(reinterpret_cast<__nv_bfloat16*>(ov) + (v + u * kGnThreads) * kGnVec, x);
                    }
            }
        } else {
            constexpr int U = kGnClipBatch / 2;
            for (int v = threadIdx.x; v < nv; v += U * kGnThreads) {
                uint4 r[U][2];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (v + u * kGnThreads < nv) {
                        const uint4* q = reinterpret_cast<const uint4*>(iv) + (ib ? 1 : 2) * (v + u * kGnThreads);
                        r[u][0] = ld_stream16(q);
                        if (!ib) r[u][1] = ld_stream16(q + 1);
                    }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (v + u * kGnThreads < nv) {
                        const int at = (v + u * kGnThreads) * kGnVec;
                        float x[8];
                        if (ib) unpack_bf16(r[u][0], x);
                        else unpack_f32(r[u][0], r[u][1], x);
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = x[i] * c * back;
                        if (ob) Vec8<__nv_bfloat16>::store(reinterpret_cast<__nv_bfloat16*>(ov) + at, x);
                        else Vec8<float>::store(reinterpret_cast<float*>(ov) + at, x);
                    }
            }
        }
        for (int j = threadIdx.x; j < len - nv * kGnVec; j += kGnThreads) {
            const int i = j < head ? j : j + nv * kGnVec;
            const float x = (ib ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(ip)[i])
                                : reinterpret_cast<const float*>(ip)[i]) * c * back;
            if (ob) reinterpret_cast<__nv_bfloat16*>(op)[i] = __float2bfloat16_rn(x);
            else reinterpret_cast<float*>(op)[i] = x;
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------
constexpr int kGnCap = 448;       // tensors per launch: a table of 13 KiB, below the 32 KiB of kernel parameters
constexpr int kGnCapSmall = 32;   // a table of 1 KiB for short lists
// What the norm leaves in the 126 MB L2 for the scaling, which reads it first and marks it as the first to go: the last 80 MiB
// of the list, over its launches. A norm alone cannot know whether a scaling follows (sf_clip_grads), so it marks them too.
// One decoder layer, inputs not in L2 before: with 64 / 80 / 96 / 128 MiB bf16 takes 197.4 / 197.8 / 198.3 / 199.0 us, fp32
// clipped into bf16 (which displaces less) 324.0 / 320.9 / 320.9 / 321.7. Nothing kept: 7 % more on 192 MB of bf16.
constexpr int64_t kGnKeepBytes = 80 << 20;

static int64_t gn_launches(int64_t count) { return count <= 0 ? 1 : (count + kGnCap - 1) / kGnCap; }

static int gn_check(const char* who, const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int64_t count) {
    if (count < 0) return fail(SF_ERR_BAD_ARG, "%s: count must not be negative", who);
    if (count > (1 << 20)) return fail(SF_ERR_UNSUPPORTED, "%s: more than 2^20 tensors", who);
    if (count > 0 && (!grads || !sizes || !dtypes)) return fail(SF_ERR_BAD_ARG, "%s: grads, sizes and dtypes must be non-null", who);
    for (int64_t i = 0; i < count; ++i) {
        if (sizes[i] < 0 || sizes[i] > ((int64_t)1 << 42)) return fail(SF_ERR_BAD_ARG, "%s: size of tensor %lld out of range", who, (long long)i);
        if (dtypes[i] != SF_F32 && dtypes[i] != SF_BF16)
            return fail(SF_ERR_BAD_ARG, "%s: dtype of tensor %lld must be SF_F32 or SF_BF16", who, (long long)i);
        if (sizes[i] > 0 && !grads[i]) return fail(SF_ERR_BAD_ARG, "%s: tensor %lld is null", who, (long long)i);
        if (reinterpret_cast<uintptr_t>(grads[i]) % (dtypes[i] == SF_BF16 ? 2 : 4))
            return fail(SF_ERR_ALIGNMENT, "%s: tensor %lld is not aligned to its elements", who, (long long)i);
    }
    return SF_OK;
}

static int gn_check_results(const char* who, const float* norm, const double* scratch) {
    if (reinterpret_cast<uintptr_t>(norm) % sizeof(float) || reinterpret_cast<uintptr_t>(scratch) % sizeof(double))
        return fail(SF_ERR_ALIGNMENT, "%s: norm and scratch must be aligned to their elements", who);
    return SF_OK;
}

// Every output is either its own input (same address, same type) or overlaps no other tensor of the call: blocks work
// on the tensors in any order.
struct GnSpan {
    uintptr_t begin, end;
    int writes;
};
static int gn_check_overlap(const char* who, const void* const* grads, void* const* outs, const int64_t* sizes,
                            const int32_t* in_dt, const int32_t* out_dt, int64_t count, const float* norm, int norm_written) {
    GnSpan* sp = new (std::nothrow) GnSpan[2 * count + 1];
    if (!sp) return fail(SF_ERR_BAD_ARG, "%s: out of host memory", who);
    int64_t k = 0;
    sp[k++] = GnSpan{reinterpret_cast<uintptr_t>(norm), reinterpret_cast<uintptr_t>(norm) + 4, norm_written};
    for (int64_t i = 0; i < count; ++i) {
        if (sizes[i] == 0) continue;
        const uintptr_t o = reinterpret_cast<uintptr_t>(outs[i]), g = reinterpret_cast<uintptr_t>(grads[i]);
        sp[k++] = GnSpan{o, o + (uintptr_t)sizes[i] * (out_dt[i] == SF_BF16 ? 2 : 4), 1};
        if (!(o == g && in_dt[i] == out_dt[i])) sp[k++] = GnSpan{g, g + (uintptr_t)sizes[i] * (in_dt[i] == SF_BF16 ? 2 : 4), 0};
    }
    std::sort(sp, sp + k, [](const GnSpan& a, const GnSpan& b) { return a.begin < b.begin; });
    uintptr_t any_end = 0, out_end = 0;
    bool bad = false;
    for (int64_t i = 0; i < k && !bad; ++i) {
        bad = sp[i].begin < (sp[i].writes ? any_end : out_end);
        any_end = std::max(any_end, sp[i].end);
        if (sp[i].writes) out_end = std::max(out_end, sp[i].end);
    }
    delete[] sp;
    if (bad) return fail(SF_ERR_BAD_ARG, "%s: an output overlaps another tensor of the call or the norm (the same gradient twice?)", who);
    return SF_OK;
}

static int gn_grid(int64_t chunks, int blocks_per_sm) {
    const int64_t cap = std::min<int64_t>(kGnSlots, (int64_t)sm_count() * blocks_per_sm);
    return (int)std::max<int64_t>(1, std::min(chunks, cap));
}

// Fills the table with tensors [from, to), the last keep_bytes of which are marked to stay in L2. Returns the number of chunks.
template <int CAP>
static int64_t gn_fill(GnTable<CAP>& tab, const void* const* grads, void* const* outs, const int64_t* sizes,
                       const int32_t* in_dt, const int32_t* out_dt, int64_t from, int64_t to, int64_t keep_bytes = 0) {
    int64_t total = 0;
    for (int64_t i = from; i < to; ++i) total += sizes[i];
    // the longest chunk that still gives every block of a resident wave some; small sets get short chunks, huge
    // ones longer chunks so that their number stays a 32-bit one
    int64_t chunk = kGnChunkUnit;
    while (chunk < 4 * kGnChunkUnit && total / (2 * chunk) >= (int64_t)sm_count() * 8) chunk *= 2;
    while (total / chunk > 0x3fffffff) chunk *= 2;
    tab.chunk = (int)chunk;
    tab.count = 0;
    tab.all_in_place = 1;
    uint32_t c = 0;
    for (int64_t i = from; i < to; ++i) {
        if (sizes[i] == 0) continue;
        const int k = tab.count++;
        void* o = outs ? outs[i] : nullptr;
        tab.t[k] = GnTensor{grads[i], o, sizes[i]};
        const int odt = out_dt ? out_dt[i] : in_dt[i];
        const int is = in_dt[i] == SF_BF16 ? 2 : 4, os = odt == SF_BF16 ? 2 : 4;
        int head = 0;  // the first element that is on a 16-byte boundary on both sides, if there is one
        while (head < 8 && ((reinterpret_cast<uintptr_t>(grads[i]) + head * is) % 16 ||
                            (o && (reinterpret_cast<uintptr_t>(o) + head * os) % 16)))
            ++head;
        tab.kind[k] = (uint8_t)((is == 2 ? GN_IN_BF16 : 0) | (os == 2 ? GN_OUT_BF16 : 0) |
                                (o == grads[i] && is == os ? GN_IN_PLACE : 0) |
                                (head < 8 ? GN_VEC | head << GN_HEAD_SHIFT : 0));
        tab.all_in_place &= (tab.kind[k] & GN_IN_PLACE) != 0;
        tab.first[k] = c;
        c += (uint32_t)((sizes[i] + chunk - 1) / chunk);
    }
    tab.first[tab.count] = c;
    tab.keep_from = c;
    for (int k = tab.count - 1; k >= 0; --k) {
        const int64_t esize = tab.kind[k] & GN_IN_BF16 ? 2 : 4, bytes = tab.t[k].n * esize;
        tab.keep_from = tab.first[k];
        if (bytes > keep_bytes) {  // only the tensor's last chunks
            tab.keep_from = tab.first[k + 1] - (uint32_t)(keep_bytes / (chunk * esize));
            break;
        }
        keep_bytes -= bytes;
    }
    return c;
}

// Launch behind the kernel before it in the stream: set up while that one still runs, waits for its results.
template <typename... KArgs, typename... Args>
static cudaError_t gn_launch_dependent(void (*kern)(KArgs...), int grid, cudaStream_t st, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kGnThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

// What each launch may leave in L2: the share of the whole list's last kGnKeepBytes that is not taken by the launches behind
// it. Asked launch by launch, in order; one walk over the list in all.
struct GnKeep {
    const int64_t* sizes;
    const int32_t* dtypes;
    int64_t start, behind = 0;  // bytes from tensor `start` on (kGnKeepBytes or more, or all), then from the launch's end on
    GnKeep(const int64_t* sizes_, const int32_t* dtypes_, int64_t count) : sizes(sizes_), dtypes(dtypes_), start(count) {
        while (start > 0 && behind < kGnKeepBytes) behind += bytes(--start);
    }
    int64_t bytes(int64_t i) const { return sizes[i] * (dtypes[i] == SF_BF16 ? 2 : 4); }
    int64_t of_launch(int64_t from, int64_t to) {
        for (int64_t i = std::max(from, start); i < to; ++i) behind -= bytes(i);
        return to <= start ? 0 : std::max<int64_t>(0, kGnKeepBytes - behind);
    }
};

// Launches the partial sums of tensors [from, to); *slots grows by the number of slots written.
template <int CAP>
static int gn_partials_part(const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int64_t from, int64_t to,
                            int64_t keep_bytes, int kind, double* scratch, int* slots, cudaStream_t st) {
    GnTable<CAP> tab;
    const int64_t chunks = gn_fill(tab, grads, nullptr, sizes, dtypes, nullptr, from, to, keep_bytes);
    if (chunks == 0) return SF_OK;
    const int grid = gn_grid(chunks, kGnNormBlocks);
    if (kind == GN_INF) grad_norm_partial_kernel<CAP, true><<<grid, kGnThreads, 0, st>>>(tab, scratch + *slots);
    else grad_norm_partial_kernel<CAP, false><<<grid, kGnThreads, 0, st>>>(tab, scratch + *slots);
    SF_CHECK_CUDA(cudaGetLastError());
    *slots += grid;
    return SF_OK;
}

static int gn_partials(const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int64_t count, int kind,
                       double* scratch, int* slots, cudaStream_t st) {
    *slots = 0;
    GnKeep keeping(sizes, dtypes, count);
    for (int64_t from = 0; from < count; from += kGnCap) {
        const int64_t to = std::min(count, from + kGnCap), keep = keeping.of_launch(from, to);
        const int rc = to - from <= kGnCapSmall
                           ? gn_partials_part<kGnCapSmall>(grads, sizes, dtypes, from, to, keep, kind, scratch, slots, st)
                           : gn_partials_part<kGnCap>(grads, sizes, dtypes, from, to, keep, kind, scratch, slots, st);
        if (rc) return rc;
    }
    return SF_OK;
}

template <int CAP>
static int gn_scale_part(const void* const* grads, void* const* outs, const int64_t* sizes, const int32_t* in_dt,
                         const int32_t* out_dt, int64_t from, int64_t to, const double* slots, int slot_count, int kind,
                         const float* norm_in, float* norm_out, double max_norm, bool dependent, cudaStream_t st) {
    GnTable<CAP> tab;
    const int grid = gn_grid(gn_fill(tab, grads, outs, sizes, in_dt, out_dt, from, to), kGnClipBlocks);
    if (dependent)
        SF_CHECK_CUDA(gn_launch_dependent(grad_clip_kernel<CAP>, grid, st, tab, slots, slot_count, kind, norm_in,
                                          norm_out, max_norm));
    else
        grad_clip_kernel<CAP><<<grid, kGnThreads, 0, st>>>(tab, slots, slot_count, kind, norm_in, norm_out, max_norm);
    SF_CHECK_CUDA(cudaGetLastError());
    return SF_OK;
}

static int gn_scale(const void* const* grads, void* const* outs, const int64_t* sizes, const int32_t* in_dt,
                    const int32_t* out_dt, int64_t count, const double* slots, int slot_count, int kind,
                    const float* norm_in, float* norm_out, double max_norm, cudaStream_t st) {
    const int64_t parts = gn_launches(count);
    // the tensors the norm read last come first; only the first of the launches follows the norm directly
    for (int64_t part = parts - 1; part >= 0; --part) {
        const int64_t from = part * kGnCap, to = std::min(count, from + kGnCap);
        float* no = part == 0 ? norm_out : nullptr;
        const bool dep = slot_count > 0 && part == parts - 1;
        const int rc = to - from <= kGnCapSmall
                           ? gn_scale_part<kGnCapSmall>(grads, outs, sizes, in_dt, out_dt, from, to, slots, slot_count, kind,
                                                        norm_in, no, max_norm, dep, st)
                           : gn_scale_part<kGnCap>(grads, outs, sizes, in_dt, out_dt, from, to, slots, slot_count, kind,
                                                   norm_in, no, max_norm, dep, st);
        if (rc) return rc;
    }
    return SF_OK;
}

}  // namespace sf

using namespace sf;

extern "C" {

int64_t sf_grad_norm_scratch_doubles(int64_t count) { return gn_launches(count) * kGnSlots; }

int64_t sf_selftest_grad_norm_kept_bytes(const int64_t* sizes, const int32_t* dtypes, int64_t count, int64_t launch) {
    if (!sizes || !dtypes || count < 0 || launch < 0 || launch >= gn_launches(count)) return -1;
    for (int64_t i = 0; i < count; ++i)
        if (sizes[i] < 0 || sizes[i] > ((int64_t)1 << 42) || (dtypes[i] != SF_F32 && dtypes[i] != SF_BF16)) return -1;
    const int64_t from = launch * kGnCap, to = std::min(count, from + kGnCap);
    GnKeep keeping(sizes, dtypes, count);
    int64_t keep = 0;
    for (int64_t part = 0; part <= launch; ++part) keep = keeping.of_launch(part * kGnCap, std::min(count, (part + 1) * kGnCap));
    const std::unique_ptr<const void*[]> nowhere(new (std::nothrow) const void*[count ? count : 1]());
    const std::unique_ptr<GnTable<kGnCap>> tab(new (std::nothrow) GnTable<kGnCap>);
    if (!tab || !nowhere) return -1;
    gn_fill(*tab, nowhere.get(), nullptr, sizes, dtypes, nullptr, from, to, keep);
    int64_t kept = 0;
    for (int k = 0; k < tab->count; ++k) {
        const int64_t before = tab->keep_from > tab->first[k] ? (int64_t)(tab->keep_from - tab->first[k]) * tab->chunk : 0;
        kept += std::max<int64_t>(0, tab->t[k].n - before) * (tab->kind[k] & GN_IN_BF16 ? 2 : 4);
    }
    return kept;
}

int sf_grad_norm(const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int64_t count, int kind,
                 float* norm, double* scratch, void* stream) {
    if (int rc = gn_check("sf_grad_norm", grads, sizes, dtypes, count)) return rc;
    SF_CHECK_ARG(kind == GN_L2 || kind == GN_INF, "sf_grad_norm: kind must be SF_NORM_L2 or SF_NORM_INF");
    SF_CHECK_ARG(norm && scratch, "sf_grad_norm: norm and scratch must be non-null");
    if (int rc = gn_check_results("sf_grad_norm", norm, scratch)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    int slots = 0;
    if (int rc = gn_partials(grads, sizes, dtypes, count, kind, scratch, &slots, st)) return rc;
    if (slots > 0) SF_CHECK_CUDA(gn_launch_dependent(grad_norm_final_kernel, 1, st, scratch, slots, kind, norm));
    else grad_norm_final_kernel<<<1, kGnThreads, 0, st>>>(scratch, slots, kind, norm);
    SF_CHECK_CUDA(cudaGetLastError());
    return SF_OK;
}

static int clip_check(const char* who, const void* const* grads, void* const* outs, const int64_t* sizes, const int32_t* in_dt,
                     const int32_t* out_dt, int64_t count, double max_norm, const float* norm, int norm_written) {
    if (int rc = gn_check(who, grads, sizes, in_dt, count)) return rc;
    if (!norm) return fail(SF_ERR_BAD_ARG, "%s: norm must be non-null", who);
    if (int rc = gn_check_results(who, norm, nullptr)) return rc;
    if (count > 0 && (!outs || !out_dt)) return fail(SF_ERR_BAD_ARG, "%s: outs and their dtypes must be non-null", who);
    if (int rc = gn_check(who, const_cast<const void* const*>(outs), sizes, out_dt, count)) return rc;
    if (!(max_norm >= 0.0)) return fail(SF_ERR_BAD_ARG, "%s: max_norm must not be negative or NaN", who);
    return gn_check_overlap(who, grads, outs, sizes, in_dt, out_dt, count, norm, norm_written);
}

int sf_clip_grads(const void* const* grads, void* const* outs, const int64_t* sizes, const int32_t* in_dtypes,
                  const int32_t* out_dtypes, int64_t count, const float* norm, double max_norm, void* stream) {
    if (int rc = clip_check("sf_clip_grads", grads, outs, sizes, in_dtypes, out_dtypes, count, max_norm, norm, 0)) return rc;
    if (count == 0) return SF_OK;
    return gn_scale(grads, outs, sizes, in_dtypes, out_dtypes, count, nullptr, 0, GN_L2, norm, nullptr, max_norm,
                    (cudaStream_t)stream);
}

int sf_clip_grad_norm(const void* const* grads, void* const* outs, const int64_t* sizes, const int32_t* in_dtypes,
                      const int32_t* out_dtypes, int64_t count, int kind, double max_norm, float* norm, double* scratch,
                      void* stream) {
    if (int rc = clip_check("sf_clip_grad_norm", grads, outs, sizes, in_dtypes, out_dtypes, count, max_norm, norm, 1)) return rc;
    SF_CHECK_ARG(kind == GN_L2 || kind == GN_INF, "sf_clip_grad_norm: kind must be SF_NORM_L2 or SF_NORM_INF");
    SF_CHECK_ARG(scratch != nullptr, "sf_clip_grad_norm: scratch must be non-null");
    if (int rc = gn_check_results("sf_clip_grad_norm", norm, scratch)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    int slots = 0;
    if (int rc = gn_partials(grads, sizes, in_dtypes, count, kind, scratch, &slots, st)) return rc;
    return gn_scale(grads, outs, sizes, in_dtypes, out_dtypes, count, scratch, slots, kind, nullptr, norm, max_norm, st);
}

}  // extern "C"
