// The global norm of a list of gradients and the list scaled by it:
//
//   norm = sqrt(sum over all tensors of sum g^2);   out = g * f,   f = 1 if norm <= clip else clip / norm
//
// (tf.global_norm / tf.clip_by_global_norm; where the norm is not finite every output is NaN, as there).  The tensors may be
// fp32, bf16 and fp16, of any number, size and mix.  Bound by memory: every gradient is read once for the norm, then read and
// written once more, because no output can be written before the last input has been read.
//
// The squares are summed in fp64 - |g| up to fp32's largest value neither overflows nor loses small gradients beside it, and
// one billion terms keep fp32's precision - and in an order that the sizes alone determine: a workgroup's chunks, its
// threads, then the workgroups' partial sums one after another in one fixed tree.  No atomics; two runs agree bit for bit.
//
// The list travels as a kernel argument (at most GN_LIST tensors a launch, longer lists take more launches): no table in
// device memory that a captured graph would have to keep alive, no copy from the host.
#include "common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

constexpr int GN_LIST = 96;              // 96 x 32 bytes of kernel argument, below 4 KB
constexpr int GN_THREADS = 256;
constexpr int GN_CHUNK = 8192;           // elements of one tensor that a workgroup takes at a time
constexpr int GN_MAX_PARTIALS = 1024;    // workgroups of the norm pass, all launches together

struct TensorList {
    const void* src[GN_LIST];
    void* dst[GN_LIST];
    long long n[GN_LIST];
    int chunk_end[GN_LIST];              // running sum of the tensors' chunk counts
    unsigned char type[GN_LIST];         // 0 fp32, 1 bf16, 2 fp16
    int count;
};

__device__ __forceinline__ float gn_load(const float* p) { return *p; }
__device__ __forceinline__ float gn_load(const __hip_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float gn_load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void gn_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void gn_store(__hip_bfloat16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void gn_store(__half* p, float v) { *p = __float2half(v); }

// the tensor that holds chunk c of the launch
__device__ __forceinline__ int gn_find(const TensorList& list, int c) {
    int lo = 0, hi = list.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list.chunk_end[mid] > c) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ double gn_square_sum(const void* src, long long begin, long long end) {
    const T* p = static_cast<const T*>(src);
    double s = 0.0;
    for (long long i = begin + threadIdx.x; i < end; i += GN_THREADS) {
        const double v = (double)gn_load(p + i);
        s += v * v;
    }
    return s;
}

template <typename T>
__device__ __forceinline__ void gn_scale(const void* src, void* dst, long long begin, long long end, float f) {
    const T* p = static_cast<const T*>(src);
    T* q = static_cast<T*>(dst);
    for (long long i = begin + threadIdx.x; i < end; i += GN_THREADS) gn_store(q + i, gn_load(p + i) * f);
}

// the sum over the workgroup, in every thread and in a fixed order
__device__ __forceinline__ double gn_block_sum(double v) {
    __shared__ double part[GN_THREADS / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < GN_THREADS / 64; ++w) s += part[w];
    return s;
}

__global__ __launch_bounds__(GN_THREADS) void gn_norm_kernel(const TensorList list, double* __restrict__ partials) {
    const int chunks = list.chunk_end[list.count - 1];
    double s = 0.0;
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = gn_find(list, c);
        const long long begin = (long long)(c - (t ? list.chunk_end[t - 1] : 0)) * GN_CHUNK;
        const long long end = begin + GN_CHUNK < list.n[t] ? begin + GN_CHUNK : list.n[t];
        if (list.type[t] == 0) s += gn_square_sum<float>(list.src[t], begin, end);
        else if (list.type[t] == 1) s += gn_square_sum<__hip_bfloat16>(list.src[t], begin, end);
        else s += gn_square_sum<__half>(list.src[t], begin, end);
    }
    s = gn_block_sum(s);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

__device__ __forceinline__ double gn_total(const double* __restrict__ partials, int count) {
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += GN_THREADS) s += partials[i];
    return sqrt(gn_block_sum(s));
}

__global__ __launch_bounds__(GN_THREADS) void gn_finish_kernel(const double* __restrict__ partials, int count,
                                                               float* __restrict__ norm) {
    const double v = gn_total(partials, count);
    if (threadIdx.x == 0) *norm = (float)v;
}

__global__ __launch_bounds__(GN_THREADS) void gn_scale_kernel(const TensorList list, const double* __restrict__ partials,
                                                              int count, float clip, float* __restrict__ norm) {
    const double v = gn_total(partials, count);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
    const float f = !isfinite(v) ? __builtin_nanf("") : v <= (double)clip ? 1.0f : (float)((double)clip / v);
    const int chunks = list.chunk_end[list.count - 1];
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = gn_find(list, c);
        if (f == 1.0f && list.src[t] == list.dst[t]) continue;      // in place and nothing to clip
        const long long begin = (long long)(c - (t ? list.chunk_end[t - 1] : 0)) * GN_CHUNK;
        const long long end = begin + GN_CHUNK < list.n[t] ? begin + GN_CHUNK : list.n[t];
        if (list.type[t] == 0) gn_scale<float>(list.src[t], list.dst[t], begin, end, f);
        else if (list.type[t] == 1) gn_scale<__hip_bfloat16>(list.src[t], list.dst[t], begin, end, f);
        else gn_scale<__half>(list.src[t], list.dst[t], begin, end, f);
    }
}

// Fills `list` from tensor `first` on; returns the tensor after the last one taken.
int gn_fill(TensorList& list, const long long* src, const long long* dst, const long long* n, const signed char* type,
            int first, int count) {
    int chunks = 0, k = 0, t = first;
    for (; t < count && k < GN_LIST; ++t) {
        if (n[t] <= 0) continue;
        const long long c = (n[t] + GN_CHUNK - 1) / GN_CHUNK;
        list.src[k] = reinterpret_cast<const void*>(src[t]);
        list.dst[k] = dst ? reinterpret_cast<void*>(dst[t]) : nullptr;
        list.n[k] = n[t];
        list.type[k] = (unsigned char)type[t];
        chunks += (int)c;
        list.chunk_end[k++] = chunks;
    }
    list.count = k;
    return t;
}

}  // namespace

// doubles of scratch that a call needs
DTF_API int dtf_global_norm_partials() { return GN_MAX_PARTIALS; }

// src / dst: addresses of the tensors (dst null: the norm alone), n: elements, type: 0 fp32, 1 bf16, 2 fp16.
// norm: one float.  clip > 0 (infinity: never clips).
DTF_API int dtf_global_norm(const long long* src, const long long* dst, const long long* n, const signed char* type, int count,
                            float clip, double* partials, float* norm, hipStream_t stream) {
    if (count < 0 || (dst && !(clip > 0.f))) return -1;
    long long left = 0;
    int live = 0;
    for (int t = 0; t < count; ++t) {
        if (n[t] < 0 || type[t] < 0 || type[t] > 2) return -1;
        left += (n[t] + GN_CHUNK - 1) / GN_CHUNK;
        live += n[t] > 0;
    }
    const long long all = left;
    int launches = (live + GN_LIST - 1) / GN_LIST;
    if (launches > GN_MAX_PARTIALS / 2 || all > 0x3fffffff) return -2;    // 49152 tensors, 8.8e12 elements
    TensorList list;
    int used = 0;
    for (int t = 0, k = 0; k < launches; ++k) {
        t = gn_fill(list, src, nullptr, n, type, t, count);
        const int chunks = list.chunk_end[list.count - 1];
        // this launch's share of the partial sums, by its share of the work; one at least
        long long g = 1 + (long long)((double)(GN_MAX_PARTIALS - launches) * (double)chunks / (double)all);
        if (g > chunks) g = chunks;
        if (used + g > GN_MAX_PARTIALS) g = GN_MAX_PARTIALS - used;
        hipLaunchKernelGGL(gn_norm_kernel, dim3((int)g), dim3(GN_THREADS), 0, stream, list, partials + used);
        DTF_CHECK_LAUNCH();
        used += (int)g;
    }
    if (!dst || live == 0) {
        hipLaunchKernelGGL(gn_finish_kernel, dim3(1), dim3(GN_THREADS), 0, stream, partials, used, norm);
        DTF_CHECK_LAUNCH();
        return 0;
    }
    for (int t = 0, k = 0; k < launches; ++k) {
        t = gn_fill(list, src, dst, n, type, t, count);
        const int chunks = list.chunk_end[list.count - 1];
        const int g = chunks < 2048 ? chunks : 2048;
        hipLaunchKernelGGL(gn_scale_kernel, dim3(g), dim3(GN_THREADS), 0, stream, list, partials, used, clip,
                           k == 0 ? norm : nullptr);
        DTF_CHECK_LAUNCH();
    }
    return 0;
}
