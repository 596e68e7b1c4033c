// Group normalisation of a channels-last activation x [B, S, C] (S: all positions of one sample), with an activation:
//
//   forward    mean, var of every (sample, group) over its S x C/G values (var biased);  inv = 1 / sqrt(var + eps)
//              xhat = (x - mean) inv;  u = gamma_c xhat + beta_c;  y = act(u)
//   backward   du = dy act'(u) (u is recomputed from x);  dbeta_c = sum du;  dgamma_c = sum du xhat  (over samples and positions)
//              d = gamma_c du;  dx = inv (d - mean(d) - xhat mean(d xhat))  (means over the (sample, group))
//
// x, y, dy, dx are fp32, bf16 or fp16; gamma, beta, their gradients, all statistics and sums are fp32 or wider.  The mean is
// kept as two floats: where a group has few channels, dgamma is what remains when sum du (x - mean) cancels, and a mean
// rounded to one float would leave its rounding error times sum du there.
#include "common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

constexpr long long GRP_MAX_GRID = 1 << 20;

__device__ __forceinline__ float grp_load(const float* p) { return *p; }
__device__ __forceinline__ float grp_load(const __hip_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float grp_load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void grp_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void grp_store(__hip_bfloat16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void grp_store(__half* p, float v) { *p = __float2half(v); }

__device__ __forceinline__ float grp_act(float u, int act) {
    switch (act) {
        case ACT_RELU: return u < 0.f ? 0.f : u;           // NaN stays NaN
        case ACT_SIGMOID: return dtf_sigmoid(u);
        case ACT_TANH: return tanhf(u);
        case ACT_SILU: return u * dtf_sigmoid(u);
        default: return u;
    }
}
__device__ __forceinline__ float grp_slope(float u, int act) {
    switch (act) {
        case ACT_RELU: return u > 0.f ? 1.f : 0.f;
        case ACT_SIGMOID: {
            const float s = dtf_sigmoid(u);
            return s * (1.f - s);
        }
        case ACT_TANH: {
            const float t = tanhf(u);
            return 1.f - t * t;
        }
        case ACT_SILU: {
            const float s = dtf_sigmoid(u);
            return s * (1.f + u * (1.f - s));
        }
        default: return 1.f;
    }
}

// sum over a workgroup of 256, in every thread and in a fixed order
__device__ __forceinline__ double grp_block_sum(double v) {
    __shared__ double part[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

// One workgroup per (sample, group).  stats [3][B G]: mean, what the mean's rounding left, inv.
template <typename T>
__global__ __launch_bounds__(256) void grp_fwd_kernel(const T* __restrict__ X, T* __restrict__ Y, long long S, int C, int G,
                                                      const float* __restrict__ gamma, const float* __restrict__ beta,
                                                      float eps, int act, float* __restrict__ stats, long long BG) {
    const int cg = C / G;
    const long long n = S * cg;
    for (long long bg = blockIdx.x; bg < BG; bg += gridDim.x) {
    const int g = (int)(bg % G);
    const long long base = (bg / G) * S * C + (long long)g * cg;
    double s = 0.0;
    for (long long i = threadIdx.x; i < n; i += 256) s += (double)grp_load(X + base + (i / cg) * C + i % cg);
    const double mean = grp_block_sum(s) / (double)n;
    s = 0.0;
    for (long long i = threadIdx.x; i < n; i += 256) {
        const double d = (double)grp_load(X + base + (i / cg) * C + i % cg) - mean;
        s += d * d;
    }
    const float inv = (float)(1.0 / sqrt(grp_block_sum(s) / (double)n + (double)eps));
    const float hi = (float)mean, lo = (float)(mean - (double)hi);
    if (threadIdx.x == 0) {
        stats[bg] = hi;
        stats[BG + bg] = lo;
        stats[2 * BG + bg] = inv;
    }
    for (long long i = threadIdx.x; i < n; i += 256) {
        const int c = g * cg + (int)(i % cg);
        const long long at = base + (i / cg) * C + i % cg;
        const float xhat = ((grp_load(X + at) - hi) - lo) * inv;
        grp_store(Y + at, grp_act(xhat * (gamma ? gamma[c] : 1.f) + (beta ? beta[c] : 0.f), act));
    }
    }
}

// One workgroup per (sample, group): the channels' sums one after another (slab [B][2][C]), then dx.
template <typename T>
__global__ __launch_bounds__(256) void grp_bwd_kernel(const T* __restrict__ X, const T* __restrict__ DY, T* __restrict__ DX,
                                                      long long S, int C, int G, const float* __restrict__ gamma,
                                                      const float* __restrict__ beta, int act,
                                                      const float* __restrict__ stats, long long BG, float* __restrict__ slab) {
    const int cg = C / G;
    for (long long bg = blockIdx.x; bg < BG; bg += gridDim.x) {
    const long long b = bg / G;
    const int g = (int)(bg % G);
    const long long base = b * S * C + (long long)g * cg;
    const float hi = stats[bg], lo = stats[BG + bg], inv = stats[2 * BG + bg];
    double m0 = 0.0, m1 = 0.0;
    for (int k = 0; k < cg; ++k) {
        const int c = g * cg + k;
        const float ga = gamma ? gamma[c] : 1.f, be = beta ? beta[c] : 0.f;
        double s0 = 0.0, s1 = 0.0;
        for (long long s = threadIdx.x; s < S; s += 256) {
            const float xhat = ((grp_load(X + base + s * C + k) - hi) - lo) * inv;
            const float du = grp_load(DY + base + s * C + k) * grp_slope(xhat * ga + be, act);
            s0 += (double)du;
            s1 += (double)du * (double)xhat;
        }
        s0 = grp_block_sum(s0);
        s1 = grp_block_sum(s1);
        if (threadIdx.x == 0) {
            slab[b * 2 * C + c] = (float)s0;
            slab[b * 2 * C + C + c] = (float)s1;
        }
        m0 += (double)ga * s0;
        m1 += (double)ga * s1;
    }
    if (!DX) continue;
    const double n = (double)S * (double)cg;
    const float a0 = (float)(m0 / n), a1 = (float)(m1 / n);
    for (long long i = threadIdx.x; i < S * cg; i += 256) {
        const int k = (int)(i % cg), c = g * cg + k;
        const long long at = base + (i / cg) * C + k;
        const float ga = gamma ? gamma[c] : 1.f, be = beta ? beta[c] : 0.f;
        const float xhat = ((grp_load(X + at) - hi) - lo) * inv;
        const float d = ga * grp_load(DY + at) * grp_slope(xhat * ga + be, act);
        grp_store(DX + at, inv * (d - a0 - xhat * a1));
    }
    }
}

// dbeta / dgamma: the R partial rows of slab [R][2][C] added in fp64 and in a fixed order, 8 channels a workgroup
__global__ __launch_bounds__(256) void grp_params_kernel(const float* __restrict__ slab, long long R, int C,
                                                         float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ double part[2][32][8];
    const int cl = threadIdx.x & 7, rl = threadIdx.x >> 3;
    const int c = blockIdx.x * 8 + cl;
    double s0 = 0.0, s1 = 0.0;
    if (c < C)
        for (long long r = rl; r < R; r += 32) {
            s0 += (double)slab[r * 2 * C + c];
            s1 += (double)slab[r * 2 * C + C + c];
        }
    part[0][rl][cl] = s0;
    part[1][rl][cl] = s1;
    __syncthreads();
    if (rl != 0 || c >= C) return;
    for (int k = 1; k < 32; ++k) {
        s0 += part[0][k][cl];
        s1 += part[1][k][cl];
    }
    if (dbeta) dbeta[c] = (float)s0;
    if (dgamma) dgamma[c] = (float)s1;
}

template <typename T>
int grp_fwd(const void* X, void* Y, long long B, long long S, int C, int G, const float* gamma, const float* beta, float eps,
            int act, float* stats, hipStream_t stream) {
    hipLaunchKernelGGL(grp_fwd_kernel<T>, dim3((unsigned)(B * G < GRP_MAX_GRID ? B * G : GRP_MAX_GRID)), dim3(256), 0, stream, static_cast<const T*>(X),
                       static_cast<T*>(Y), S, C, G, gamma, beta, eps, act, stats, B * G);
    DTF_CHECK_LAUNCH();
    return 0;
}

template <typename T>
int grp_bwd(const void* X, const void* DY, void* DX, long long B, long long S, int C, int G, const float* gamma,
            const float* beta, int act, const float* stats, float* dgamma, float* dbeta, float* slab, hipStream_t stream) {
    hipLaunchKernelGGL(grp_bwd_kernel<T>, dim3((unsigned)(B * G < GRP_MAX_GRID ? B * G : GRP_MAX_GRID)), dim3(256), 0, stream, static_cast<const T*>(X),
                       static_cast<const T*>(DY), static_cast<T*>(DX), S, C, G, gamma, beta, act, stats, B * G, slab);
    DTF_CHECK_LAUNCH();
    if (dgamma || dbeta) {
        hipLaunchKernelGGL(grp_params_kernel, dim3((C + 7) / 8), dim3(256), 0, stream, slab, B, C, dgamma, dbeta);
        DTF_CHECK_LAUNCH();
    }
    return 0;
}

bool grp_args_ok(long long B, long long S, int C, int G, int type, int act) {
    return B > 0 && S > 0 && C > 0 && G > 0 && C % G == 0 && type >= 0 && type <= 2 && act >= ACT_NONE &&
           act <= ACT_SILU;
}

}  // namespace

// floats of scratch that the backward call needs
DTF_API long long dtf_groupnorm_workspace_floats(long long B, long long S, int C, int G) { return B * 2 * C; }

// type: 0 fp32, 1 bf16, 2 fp16.  gamma / beta may be null.  stats: 3 B G floats, kept for the backward call.
DTF_API int dtf_groupnorm_fwd(const void* X, void* Y, long long B, long long S, int C, int G, int type, const float* gamma,
                              const float* beta, float eps, int act, float* stats, hipStream_t stream) {
    if (!grp_args_ok(B, S, C, G, type, act)) return -1;
    if (type == 0) return grp_fwd<float>(X, Y, B, S, C, G, gamma, beta, eps, act, stats, stream);
    if (type == 1) return grp_fwd<__hip_bfloat16>(X, Y, B, S, C, G, gamma, beta, eps, act, stats, stream);
    return grp_fwd<__half>(X, Y, B, S, C, G, gamma, beta, eps, act, stats, stream);
}

// DX, dgamma, dbeta may each be null.
DTF_API int dtf_groupnorm_bwd(const void* X, const void* DY, void* DX, long long B, long long S, int C, int G, int type,
                              const float* gamma, const float* beta, int act, const float* stats, float* dgamma, float* dbeta,
                              float* workspace, hipStream_t stream) {
    if (!grp_args_ok(B, S, C, G, type, act)) return -1;
    if (type == 0) return grp_bwd<float>(X, DY, DX, B, S, C, G, gamma, beta, act, stats, dgamma, dbeta, workspace, stream);
    if (type == 1)
        return grp_bwd<__hip_bfloat16>(X, DY, DX, B, S, C, G, gamma, beta, act, stats, dgamma, dbeta, workspace, stream);
    return grp_bwd<__half>(X, DY, DX, B, S, C, G, gamma, beta, act, stats, dgamma, dbeta, workspace, stream);
}
