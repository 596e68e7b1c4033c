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
// The list travels as a kernel argument (longer lists take more launches): no table in device memory that a captured graph
// would have to keep alive, no copy from the host.  A tensor is cut into chunks of 8192 values, which the workgroups find by a
// search over the chunks' running count; all of a chunk's loads (16 bytes a lane, at any alignment) are in flight at once.
//
// Measured: 1.087e9 fp32 gradients 0.73 ms for the norm (6.0 TB/s) and 1.68 ms for the scaling (5.2 TB/s), where a large copy
// reaches 4.6 TB/s; 400 gradients of mixed types and 1 to 262144 values 16 and 38 us in five launches (the host's checks of 800
// tensors take 0.2 ms), six gradients of an MLP 4.4 and 5.2 us.
#include "common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

constexpr int GN_THREADS = 256;
constexpr int GN_CHUNK = 8192;           // values of one tensor that a workgroup takes at a time: 32 a thread
constexpr int GN_MAX_PARTIALS = 1024;    // workgroups of the norm pass, all launches together

// COUNT tensors of a launch; with the kernels' other arguments below 4 KB
template <int COUNT, bool OUT>
struct TensorList {
    static constexpr int MOST = COUNT;
    const void* src[COUNT];
    void* dst[OUT ? COUNT : 1];
    int chunk_end[COUNT];                // running sum of the tensors' chunk counts
    unsigned short last[COUNT];          // values in the last chunk - 1, and type << 13: 0 fp32, 1 bf16, 2 fp16
    int count;
};
typedef TensorList<256, false> NormList;
typedef TensorList<176, true> ScaleList;
static_assert(sizeof(NormList) + 16 <= 4096 && sizeof(ScaleList) + 32 <= 4096 && GN_CHUNK == 1 << 13, "kernel arguments");

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// 16 bytes as floats and back
template <typename T>
struct Pack;
template <>
struct Pack<float> {
    static constexpr int VEC = 4;
    typedef u32x4 any __attribute__((aligned(4)));
    static __device__ __forceinline__ float get(const u32x4& q, int e) { return __uint_as_float(q[e]); }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[4]) {
        return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    }
    static __device__ __forceinline__ float load(const float* p) { return *p; }
    static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
};
template <>
struct Pack<__hip_bfloat16> {
    static constexpr int VEC = 8;
    typedef u32x4 any __attribute__((aligned(2)));
    static __device__ __forceinline__ float get(const u32x4& q, int e) {
        return __uint_as_float(e & 1 ? q[e >> 1] & 0xffff0000u : q[e >> 1] << 16);
    }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[8]) {
        typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
        b16x8 h;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = (__bf16)v[e];
        return __builtin_bit_cast(u32x4, h);
    }
    static __device__ __forceinline__ float load(const __hip_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ void store(__hip_bfloat16* p, float v) { *p = __float2bfloat16(v); }
};
template <>
struct Pack<__half> {
    static constexpr int VEC = 8;
    typedef u32x4 any __attribute__((aligned(2)));
    static __device__ __forceinline__ float get(const u32x4& q, int e) {
        return (float)__builtin_bit_cast(_Float16, (unsigned short)(e & 1 ? q[e >> 1] >> 16 : q[e >> 1] & 0xffffu));
    }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[8]) {
        typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
        h16x8 h;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = (_Float16)v[e];
        return __builtin_bit_cast(u32x4, h);
    }
    static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
    static __device__ __forceinline__ void store(__half* p, float v) { *p = __float2half(v); }
};

// the tensor that holds chunk c of the launch, and where in it the chunk lies
template <typename L>
__device__ __forceinline__ int gn_find(const L& list, int c, long long& begin, int& size) {
    int lo = 0, hi = list.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list.chunk_end[mid] > c) hi = mid;
        else lo = mid + 1;
    }
    begin = (long long)(c - (lo ? list.chunk_end[lo - 1] : 0)) * GN_CHUNK;
    size = c + 1 == list.chunk_end[lo] ? (list.last[lo] & (GN_CHUNK - 1)) + 1 : GN_CHUNK;
    return lo;
}

template <typename T>
__device__ __forceinline__ double gn_square_sum(const void* src, long long begin, int size) {
    constexpr int VEC = Pack<T>::VEC, TURNS = GN_CHUNK / GN_THREADS / VEC;
    const T* p = static_cast<const T*>(src) + begin;
    double s = 0.0;
    if (size == GN_CHUNK) {
        u32x4 q[TURNS];
#pragma unroll
        for (int k = 0; k < TURNS; ++k) q[k] = *reinterpret_cast<const typename Pack<T>::any*>(p + (k * GN_THREADS + threadIdx.x) * VEC);
        double t[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int k = 0; k < TURNS; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const double v = (double)Pack<T>::get(q[k], e);
                t[e & 3] = fma(v, v, t[e & 3]);
            }
        s = (t[0] + t[1]) + (t[2] + t[3]);
    } else {
#pragma unroll 8
        for (int i = threadIdx.x; i < size; i += GN_THREADS) {
            const double v = (double)Pack<T>::load(p + i);
            s = fma(v, v, s);
        }
    }
    return s;
}

template <typename T>
__device__ __forceinline__ void gn_scale(const void* src, void* dst, long long begin, int size, float f) {
    constexpr int VEC = Pack<T>::VEC, TURNS = GN_CHUNK / GN_THREADS / VEC;
    const T* p = static_cast<const T*>(src) + begin;
    T* q = static_cast<T*>(dst) + begin;
    if (size == GN_CHUNK) {
        u32x4 x[TURNS];
#pragma unroll
        for (int k = 0; k < TURNS; ++k) x[k] = *reinterpret_cast<const typename Pack<T>::any*>(p + (k * GN_THREADS + threadIdx.x) * VEC);
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
            float v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = Pack<T>::get(x[k], e) * f;
            *reinterpret_cast<typename Pack<T>::any*>(q + (k * GN_THREADS + threadIdx.x) * VEC) = Pack<T>::pack(v);
        }
    } else {
#pragma unroll 8
        for (int i = threadIdx.x; i < size; i += GN_THREADS) Pack<T>::store(q + i, Pack<T>::load(p + i) * f);
    }
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

__global__ __launch_bounds__(GN_THREADS) void gn_norm_kernel(const NormList list, double* __restrict__ partials) {
    const int chunks = list.chunk_end[list.count - 1];
    double s = 0.0;
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        long long begin;
        int size;
        const int t = gn_find(list, c, begin, size), type = list.last[t] >> 13;
        if (type == 0) s += gn_square_sum<float>(list.src[t], begin, size);
        else if (type == 1) s += gn_square_sum<__hip_bfloat16>(list.src[t], begin, size);
        else s += gn_square_sum<__half>(list.src[t], begin, size);
    }
    s = gn_block_sum(s);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

__device__ __forceinline__ double gn_total(const double* __restrict__ partials, int count) {
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < GN_MAX_PARTIALS / GN_THREADS; ++k) {
        const int i = k * GN_THREADS + threadIdx.x;
        s += i < count ? partials[i] : 0.0;
    }
    return sqrt(gn_block_sum(s));
}

__global__ __launch_bounds__(GN_THREADS) void gn_finish_kernel(const double* __restrict__ partials, int count,
                                                               float* __restrict__ norm) {
    const double v = gn_total(partials, count);
    if (threadIdx.x == 0) *norm = (float)v;
}

__global__ __launch_bounds__(GN_THREADS) void gn_scale_kernel(const ScaleList list, const double* __restrict__ partials,
                                                              int count, double clip, float* __restrict__ norm) {
    const double v = gn_total(partials, count);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
    const float f = !isfinite(v) ? __builtin_nanf("") : v <= clip ? 1.0f : (float)(clip / v);
    const int chunks = list.chunk_end[list.count - 1];
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        long long begin;
        int size;
        const int t = gn_find(list, c, begin, size), type = list.last[t] >> 13;
        if (f == 1.0f && list.src[t] == list.dst[t]) continue;      // in place and nothing to clip
        if (type == 0) gn_scale<float>(list.src[t], list.dst[t], begin, size, f);
        else if (type == 1) gn_scale<__hip_bfloat16>(list.src[t], list.dst[t], begin, size, f);
        else gn_scale<__half>(list.src[t], list.dst[t], begin, size, f);
    }
}

// Fills `list` from tensor `first` on; returns the tensor after the last one taken.
template <typename L>
int gn_fill(L& list, const long long* src, const long long* dst, const long long* n, const signed char* type, int first, int count) {
    int chunks = 0, k = 0, t = first;
    for (; t < count && k < L::MOST; ++t) {
        if (n[t] <= 0) continue;
        list.src[k] = reinterpret_cast<const void*>(src[t]);
        if (dst) list.dst[k] = reinterpret_cast<void*>(dst[t]);
        list.last[k] = (unsigned short)(((n[t] - 1) & (GN_CHUNK - 1)) | type[t] << 13);
        chunks += (int)((n[t] + GN_CHUNK - 1) / GN_CHUNK);
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
                            double clip, double* partials, float* norm, hipStream_t stream) {
    if (count < 0 || (dst && !(clip > 0.0))) return -1;
    long long all = 0;
    int live = 0;
    for (int t = 0; t < count; ++t) {
        if (n[t] < 0 || type[t] < 0 || type[t] > 2) return -1;
        all += (n[t] + GN_CHUNK - 1) / GN_CHUNK;
        live += n[t] > 0;
    }
    const int launches = (live + NormList::MOST - 1) / NormList::MOST;
    if (launches > GN_MAX_PARTIALS / 2 || all > 0x3fffffff) return -2;    // 131072 tensors, 8.8e12 elements
    NormList list;
    int used = 0;
    for (int t = 0, k = 0; k < launches; ++k) {
        t = gn_fill(list, src, nullptr, n, type, t, count);
        const int chunks = list.chunk_end[list.count - 1];
        // this launch's share of the partial sums, by its share of the work; one at least
        long long g = 1 + (long long)((double)(GN_MAX_PARTIALS - launches) * (double)chunks / (double)all);
        if (g > chunks) g = chunks;
        if (used + g > GN_MAX_PARTIALS - (launches - 1 - k)) g = GN_MAX_PARTIALS - (launches - 1 - k) - used;
        hipLaunchKernelGGL(gn_norm_kernel, dim3((int)g), dim3(GN_THREADS), 0, stream, list, partials + used);
        DTF_CHECK_LAUNCH();
        used += (int)g;
    }
    if (!dst || live == 0) {
        hipLaunchKernelGGL(gn_finish_kernel, dim3(1), dim3(GN_THREADS), 0, stream, partials, used, norm);
        DTF_CHECK_LAUNCH();
        return 0;
    }
    ScaleList scale;
    for (int t = 0, done = 0; done < live;) {
        t = gn_fill(scale, src, dst, n, type, t, count);
        const int chunks = scale.chunk_end[scale.count - 1];
        const int g = chunks < 2048 ? chunks : 2048;
        hipLaunchKernelGGL(gn_scale_kernel, dim3(g), dim3(GN_THREADS), 0, stream, scale, partials, used, clip,
                           done == 0 ? norm : nullptr);
        DTF_CHECK_LAUNCH();
        done += scale.count;
    }
    return 0;
}
