// Group normalisation of a channels-last activation x [B, S, C] (S: all positions of one sample), with an activation:
//
//   forward    mean, var of every (sample, group) over its S x C/G values (var biased);  inv = 1 / sqrt(var + eps)
//              xhat = (x - mean) inv;  u = gamma_c xhat + beta_c;  y = act(u)
//   backward   du = dy act'(u) (u is recomputed from x);  dbeta_c = sum du;  dgamma_c = sum du xhat  (over samples and positions)
//              d = gamma_c du;  dx = inv (d - mean(d) - xhat mean(d xhat))  (means over the (sample, group))
//
// x, y, dy, dx are fp32, bf16 or fp16; gamma, beta, their gradients, all statistics and sums are fp32 or wider.  The mean is
// kept as two floats: where a group has few channels, dgamma is what remains when sum du (x - mean) cancels, and a mean
// rounded to one float would leave its rounding error times sum du there.  u is rounded after every operation (no fused
// multiply-add), as the formula written out in separate operations is, so that values within a rounding of relu's border seldom
// fall on another side than there (one in some 1e8 does, with a gradient of its own in dx: no two ways of rounding agree on all).
//
// Everything is bound by memory.  A sample is one stream of S C values, read in vectors of 16 bytes at any alignment; a
// workgroup takes T vectors a turn, T a multiple of C / gcd(C, vector): then a thread meets the same channels every turn and
// keeps their constants in registers.
//   one   samples up to 128 KB (64 KB in 16 bits): a workgroup holds a sample in registers - x is read once and y written once,
//         backward dy and x once and dx once: the least there is.  The variance is taken about the channels' means, from the registers.
//   many  larger samples: partial sums of every channel over chunks of a sample (about a pivot, the channel's first value; fp32
//         over 8 turns, then fp64), joined per group; then one elementwise pass.  x is read twice a direction.
// All sums have an order that the sizes determine; no atomics.
//
// Whole vectors are taken without a test of every value (bf16 partial sums: 56 -> 33 us) where a second copy of the code does not
// cost more than the tests: not with sixteen vectors a thread, nor in the backward pass over larger samples.
//
// Measured (forward / backward, of the bytes that each cannot do without): 16384 x 24 x 24 x 32 fp32 relu 446 us (5.4 TB/s) /
// 640 us (5.7 TB/s), a large copy reaching 4.6 TB/s; 64 x 64 x 64 x 256 silu, read twice, fp32 170 / 187 us, bf16 83 / 134 us; 3 x
// 129 x 131 x 225 bf16 silu (four launches a direction) 35 / 54 us.  16-bit values with silu are bound by instructions
// (16384 x 12 x 12 x 64: 169 / 357 us, 3.6 / 2.5 TB/s): the exponential is computed in both passes of the backward kernel, since
// du would have to be kept in 32 bits beside x and dy.
#include "common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <type_traits>

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    typedef u32x4 any __attribute__((aligned(4)));
    static constexpr int VEC = 4;
    static __device__ __forceinline__ float get(const u32x4& q, int e) { return __uint_as_float(q[e]); }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[4]) {
        return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    }
    static __device__ __forceinline__ float load(const float* p) { return *p; }
    static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
};
template <>
struct Elem<__hip_bfloat16> {
    typedef u32x4 any __attribute__((aligned(2)));
    static constexpr int VEC = 8;
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
struct Elem<__half> {
    typedef u32x4 any __attribute__((aligned(2)));
    static constexpr int VEC = 8;
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

// VEC values at p, of which `live` exist (the rest reads as zero / is not written); any alignment
template <typename T, int VEC>
__device__ __forceinline__ u32x4 grp_load(const T* p, int live) {
    if (VEC == Elem<T>::VEC && live >= VEC) return *reinterpret_cast<const typename Elem<T>::any*>(p);
    float v[Elem<T>::VEC];
#pragma unroll
    for (int e = 0; e < Elem<T>::VEC; ++e) v[e] = e < VEC && e < live ? Elem<T>::load(p + e) : 0.f;
    return Elem<T>::pack(v);
}
template <typename T, int VEC>
__device__ __forceinline__ void grp_store(T* p, const float (&v)[VEC], int live) {
    if constexpr (VEC == Elem<T>::VEC) {
        if (live >= VEC) {
            *reinterpret_cast<typename Elem<T>::any*>(p) = Elem<T>::pack(v);
            return;
        }
    }
    {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (e < live) Elem<T>::store(p + e, v[e]);
    }
}

// 1 / (1 + exp(-u)) with the hardware's reciprocal (1 ulp) instead of a division; tanh u = 1 - 2 / (exp(2 u) + 1): off by some
// 2^-23 absolutely, which is what the output's terms are rounded to.  Divisions and tanhf would make these kernels bound by
// instructions (16384 x 12 x 12 x 64 bf16, silu, backward: 456 us with them).
__device__ __forceinline__ float grp_sigmoid(float u) { return __builtin_amdgcn_rcpf(1.f + __expf(-u)); }
__device__ __forceinline__ float grp_tanh(float u) { return 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __expf(2.f * u)); }

template <int VEC>
__device__ __forceinline__ void grp_act(float (&u)[VEC], int act) {
    switch (act) {
        case ACT_RELU:
#pragma unroll
            for (int e = 0; e < VEC; ++e) u[e] = u[e] < 0.f ? 0.f : u[e];           // NaN stays NaN
            break;
        case ACT_SIGMOID:
#pragma unroll
            for (int e = 0; e < VEC; ++e) u[e] = grp_sigmoid(u[e]);
            break;
        case ACT_TANH:
#pragma unroll
            for (int e = 0; e < VEC; ++e) u[e] = grp_tanh(u[e]);
            break;
        case ACT_SILU:
#pragma unroll
            for (int e = 0; e < VEC; ++e) u[e] *= grp_sigmoid(u[e]);
            break;
        default: break;
    }
}
// dy <- dy act'(u)
template <int VEC>
__device__ __forceinline__ void grp_slope(const float (&u)[VEC], float (&dy)[VEC], int act) {
    switch (act) {
        case ACT_RELU:
#pragma unroll
            for (int e = 0; e < VEC; ++e) dy[e] = u[e] > 0.f ? dy[e] : 0.f;
            break;
        case ACT_SIGMOID:
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float s = grp_sigmoid(u[e]);
                dy[e] *= s * (1.f - s);
            }
            break;
        case ACT_TANH:
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float t = grp_tanh(u[e]);
                dy[e] *= 1.f - t * t;
            }
            break;
        case ACT_SILU:
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float s = grp_sigmoid(u[e]);
                dy[e] *= s * (1.f + u[e] * (1.f - s));
            }
            break;
        default: break;
    }
}

__device__ __forceinline__ float grp_inv(double var, float eps) { return __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn((float)var, eps))); }

// f(e, channel, group) for the VEC neighbours from channel c0 on (after the last channel the first one follows)
template <int VEC, typename Fn>
__device__ __forceinline__ void grp_walk(int c0, int C, int cg, Fn f) {
    int c = c0, g = c0 / cg, in = c0 - g * cg;                // one division a thread; the others count on
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        f(e, c, g);
        ++c;
        if (++in == cg) {
            in = 0;
            ++g;
        }
        if (c == C) c = g = in = 0;
    }
}

// The channels of a thread's vector and their constants.
template <int VEC>
struct Lane {
    float ga[VEC], be[VEC], hi[VEC], lo[VEC], inv[VEC];
    __device__ __forceinline__ void params(int c0, int C, int cg, const float* __restrict__ gamma, const float* __restrict__ beta) {
        grp_walk<VEC>(c0, C, cg, [&](int e, int c, int) {
            ga[e] = gamma ? gamma[c] : 1.f;
            be[e] = beta ? beta[c] : 0.f;
        });
    }
    // st: hi, lo, inv of the sample's groups, `step` apart (global memory or LDS)
    __device__ __forceinline__ void stats(int c0, int C, int cg, const float* st, long long step) {
        grp_walk<VEC>(c0, C, cg, [&](int e, int, int g) {
            hi[e] = st[g];
            lo[e] = st[step + g];
            inv[e] = st[2 * step + g];
        });
    }
    __device__ __forceinline__ float xhat(float x, int e) const { return __fmul_rn(__fsub_rn(__fsub_rn(x, hi[e]), lo[e]), inv[e]); }
    __device__ __forceinline__ float u(float xh, int e) const { return __fadd_rn(__fmul_rn(xh, ga[e]), be[e]); }
};

// Sums over the workgroup, channel by channel, of NA values at once: thread t < T brings values of the channels (t VEC + e) % C,
// period P vectors; chan[a][C] receives the sums.  F: float or double.  `red` has room for NA T VEC values.
template <typename F, int VEC, int NA>
__device__ __forceinline__ void grp_channels(F (&v)[NA][VEC], int T, int P, int C, F* red, F* chan) {
    const int tid = threadIdx.x;
    int entries = T * VEC;                                    // entry i belongs to channel i % C
    if (P <= 32 && (P & (P - 1)) == 0 && T == (int)blockDim.x) {
        for (int o = P; o < 64; o <<= 1)
#pragma unroll
            for (int a = 0; a < NA; ++a)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[a][e] += __shfl_xor(v[a][e], o, 64);
        entries = (T / 64) * P * VEC;
        if ((tid & 63) < P)
#pragma unroll
            for (int a = 0; a < NA; ++a)
#pragma unroll
                for (int e = 0; e < VEC; ++e) red[a * entries + ((tid >> 6) * P + (tid & 63)) * VEC + e] = v[a][e];
    } else if (tid < T) {
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
            for (int e = 0; e < VEC; ++e) red[a * entries + tid * VEC + e] = v[a][e];
    }
    __syncthreads();
    // Few channels have many entries each: up to 64 lanes share a channel, eight entries at least a lane, and the sum is fp64
    // (hundreds of fp32 additions of like numbers all round to one side: with 6 channels of 3060 positions the mean was off by 7e-6).
    int shift = 0;
    while (shift < 6 && NA * C << (shift + 1) <= (int)blockDim.x && C << (shift + 4) <= entries) ++shift;
    const int lanes = 1 << shift, lane = tid & (lanes - 1);
    for (int i = tid >> shift; __any(i < NA * C); i += blockDim.x >> shift) {
        const int a = NA == 2 && i >= C ? 1 : 0, c = i - a * C;
        double s = 0.0;
        if (i < NA * C)
#pragma unroll 2
            for (int k = c + lane * C; k < entries; k += C * lanes) s += (double)red[a * entries + k];
        for (int o = lanes / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if (lane == 0 && i < NA * C) chan[i] = (F)s;
    }
    __syncthreads();
}

// f(g, sum over the group's channels of value(c, g)) for every group: a thread a group of few channels, a wave a group of many
// UNROLL 1 where registers are short: the forward kernel with sixteen vectors a thread takes 128 of them (443 us; 136 halve the
// workgroups on a compute unit: 635 us).
template <int UNROLL, typename V, typename Fn>
__device__ __forceinline__ void grp_groups(int G, int cg, V value, Fn f) {
    if (cg <= 32) {
        for (int g = threadIdx.x; g < G; g += blockDim.x) {
            double s = 0.0;
#pragma unroll UNROLL
            for (int k = 0; k < cg; ++k) s += value(g * cg + k, g);
            f(g, s);
        }
    } else {
        const int lane = threadIdx.x & 63;
        for (int g = threadIdx.x >> 6; g < G; g += blockDim.x >> 6) {
            double s = 0.0;
            for (int k = lane; k < cg; k += 64) s += value(g * cg + k, g);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
            if (lane == 0) f(g, s);
        }
    }
    __syncthreads();
}

// The compiler may not carry anything computed from the vectors past this point: they stay as the few registers they are.
template <int NV>
__device__ __forceinline__ void grp_forget(u32x4 (&q)[NV]) {
#pragma unroll
    for (int k = 0; k < NV; ++k) asm volatile("" : "+v"(q[k]));
}

// ---------------------------------------------------------------------------------------------- samples that fit a workgroup
template <typename T, int NV>
__global__ __launch_bounds__(512) void grp_one_fwd_kernel(const T* __restrict__ X, T* __restrict__ Y, int N, int C, int G, int TH, int P,
                                                          const float* __restrict__ gamma, const float* __restrict__ beta, float eps,
                                                          int act, float* __restrict__ stats, long long BG) {
    constexpr int VEC = Elem<T>::VEC;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* red = reinterpret_cast<float*>(smem);               // [2][blockDim VEC]
    float* chan = red + 2 * blockDim.x * VEC;                  // [2][C]
    float* piv = chan + 2 * C;                                 // [C]
    float* st = piv + C;                                       // [3][G]
    const long long b = blockIdx.x;
    const int tid = threadIdx.x, cg = C / G, c0 = (int)(((long long)tid * VEC) % C);
    const double n = (double)(N / G);
    const T* x = X + b * N;
    u32x4 q[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int at = (k * TH + tid) * VEC;
        q[k] = tid < TH && at < N ? grp_load<T, VEC>(x + at, N - at) : u32x4{0u, 0u, 0u, 0u};
    }
    float s[1][VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[0][e] = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[0][e] += Elem<T>::get(q[k], e);
    grp_channels<float, VEC, 1>(s, TH, P, C, red, chan);
    const double rows = (double)(N / C);
    for (int c = tid; c < C; c += blockDim.x) piv[c] = (float)((double)chan[c] / rows);
    __syncthreads();
    grp_forget(q);
    Lane<VEC> ln;
    grp_walk<VEC>(c0, C, cg, [&](int e, int c, int) { ln.hi[e] = piv[c]; });
    // about the channel's own mean, so that no partial sum is large: what its rounding left, and the squares
    float s2[2][VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) s2[0][e] = s2[1][e] = 0.f;
    auto about_mean = [&](int k, auto full) {                  // `full`: a whole vector
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (full || (tid < TH && (k * TH + tid) * VEC + e < N)) {
                const float d = Elem<T>::get(q[k], e) - ln.hi[e];
                s2[0][e] += d;
                s2[1][e] += d * d;
            }
    };
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int at = (k * TH + tid) * VEC;
        if (NV > 8) {
            if (k * TH * VEC >= N) break;
            about_mean(k, std::false_type());
        } else {
            if (tid >= TH || at >= N) break;
            if (at + VEC <= N) about_mean(k, std::true_type());
            else about_mean(k, std::false_type());
        }
    }
    grp_channels<float, VEC, 2>(s2, TH, P, C, red, chan);
    grp_groups<1>(G, cg, [&](int c, int) { return rows * (double)piv[c] + (double)chan[c]; }, [&](int g, double v) {
        st[g] = (float)(v / n);
        st[G + g] = (float)(v / n - (double)st[g]);
    });
    grp_groups<1>(G, cg, [&](int c, int g) {
        const double off = (double)piv[c] - (double)st[g] - (double)st[G + g];   // sum (x - mean)^2 from the sums about piv
        return (double)chan[C + c] + 2.0 * off * (double)chan[c] + rows * off * off;
    }, [&](int g, double v) {
        const double var = v / n;
        const float inv = grp_inv(var > 0.0 || var != var ? var : 0.0, eps);
        st[2 * G + g] = inv;
        stats[b * G + g] = st[g];
        stats[BG + b * G + g] = st[G + g];
        stats[2 * BG + b * G + g] = inv;
    });
    grp_forget(q);
    ln.params(c0, C, cg, gamma, beta);
    if (tid >= TH) return;
    ln.stats(c0, C, cg, st, G);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int at = (k * TH + tid) * VEC;
        if (at >= N) break;
        float u[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) u[e] = ln.u(ln.xhat(Elem<T>::get(q[k], e), e), e);
        grp_act<VEC>(u, act);
        grp_store<T, VEC>(Y + b * N + at, u, N - at);
    }
}

// A workgroup takes samples blockIdx.x, + gridDim.x, ...; slab [gridDim.x][2][C]: its sums of du and du xhat.
template <typename T, int NV>
__global__ __launch_bounds__(512) void grp_one_bwd_kernel(const T* __restrict__ X, const T* __restrict__ DY, T* __restrict__ DX, int N,
                                                          int C, int G, int TH, int P, long long B, const float* __restrict__ gamma,
                                                          const float* __restrict__ beta, int act, const float* __restrict__ stats,
                                                          long long BG, float* __restrict__ slab) {
    constexpr int VEC = Elem<T>::VEC;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* red = reinterpret_cast<float*>(smem);               // [2][blockDim VEC]
    float* chan = red + 2 * blockDim.x * VEC;                  // [2][C] du, du xhat of a sample
    float* sum = chan + 2 * C;                                 // [2][C] over the workgroup's samples
    float* m0 = sum + 2 * C;                                   // [G] means of d, d xhat
    float* m1 = m0 + G;
    const int tid = threadIdx.x, cg = C / G, c0 = (int)(((long long)tid * VEC) % C);
    const double n = (double)(N / G);
    for (int i = tid; i < 2 * C; i += blockDim.x) sum[i] = 0.f;
    Lane<VEC> ln;
    ln.params(c0, C, cg, gamma, beta);
    for (long long b = blockIdx.x; b < B; b += gridDim.x) {
        u32x4 qx[NV], qd[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = (k * TH + tid) * VEC;
            const bool live = tid < TH && at < N;
            qx[k] = live ? grp_load<T, VEC>(X + b * N + at, N - at) : u32x4{0u, 0u, 0u, 0u};
            qd[k] = live ? grp_load<T, VEC>(DY + b * N + at, N - at) : u32x4{0u, 0u, 0u, 0u};
        }
        ln.stats(c0, C, cg, stats + b * G, BG);
        float s[2][VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[0][e] = s[1][e] = 0.f;
        auto sum_du = [&](int k, auto full) {
            float xh[VEC], u[VEC], d[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                xh[e] = ln.xhat(Elem<T>::get(qx[k], e), e);
                u[e] = ln.u(xh[e], e);
                d[e] = Elem<T>::get(qd[k], e);
            }
            grp_slope<VEC>(u, d, act);
            if constexpr (VEC == 4) qd[k] = Elem<T>::pack(d);          // fp32: du takes dy's registers
            const int live = full ? VEC : tid < TH ? N - (k * TH + tid) * VEC : 0;
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (e < live) {
                    s[0][e] += d[e];
                    s[1][e] += d[e] * xh[e];
                }
        };
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = (k * TH + tid) * VEC;
            if (NV > 8) {
                if (k * TH * VEC >= N) break;
                sum_du(k, std::false_type());
            } else {
                if (tid >= TH || at >= N) break;
                if (at + VEC <= N) sum_du(k, std::true_type());
                else sum_du(k, std::false_type());
            }
        }
        grp_channels<float, VEC, 2>(s, TH, P, C, red, chan);
        for (int i = tid; i < 2 * C; i += blockDim.x) sum[i] += chan[i];
        if (!DX) {
            __syncthreads();
            continue;
        }
        grp_groups<4>(G, cg, [&](int c, int) { return (double)(gamma ? gamma[c] : 1.f) * (double)chan[c]; },
                   [&](int g, double v) { m0[g] = (float)(v / n); });
        grp_groups<4>(G, cg, [&](int c, int) { return (double)(gamma ? gamma[c] : 1.f) * (double)chan[C + c]; },
                   [&](int g, double v) { m1[g] = (float)(v / n); });
        grp_forget(qx);
        grp_forget(qd);
        float a0[VEC], a1[VEC];
        grp_walk<VEC>(c0, C, cg, [&](int e, int, int g) {
            a0[e] = m0[g];
            a1[e] = m1[g];
        });
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = (k * TH + tid) * VEC;
            if (tid >= TH || at >= N) break;
            float xh[VEC], u[VEC], d[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                xh[e] = ln.xhat(Elem<T>::get(qx[k], e), e);
                u[e] = ln.u(xh[e], e);
                d[e] = Elem<T>::get(qd[k], e);
            }
            if (VEC != 4) grp_slope<VEC>(u, d, act);
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[e] = ln.inv[e] * (d[e] * ln.ga[e] - a0[e] - xh[e] * a1[e]);
            grp_store<T, VEC>(DX + b * N + at, d, N - at);
        }
        __syncthreads();                                       // m0, m1 and chan have been read
    }
    if (!slab) return;
    for (int i = tid; i < 2 * C; i += blockDim.x) slab[(long long)blockIdx.x * 2 * C + i] = sum[i];
}

// ------------------------------------------------------------------------------------------------------------ larger samples
// A workgroup (sample and chunk, window of channels) takes turns [chunk per, ...) of the sample.  Where the period fits a
// workgroup, turn i covers the vectors i TH ... i TH + TH - 1 of the stream; else the window's channels of position i.
template <int VEC>
struct Stream {
    long long sample, chunk, turn0, turn1, step, first, N;
    int c0, live_threads;
    __device__ __forceinline__ Stream(long long S, int C, int TH, long long chunks, long long per) {
        N = S * C;
        sample = blockIdx.x / chunks;
        chunk = blockIdx.x - sample * chunks;
        const bool windows = gridDim.y > 1;
        const int window = blockIdx.y * TH * VEC;              // channels before this window
        step = windows ? C : (long long)TH * VEC;
        const long long turns = windows ? S : (N + step - 1) / step;
        turn0 = chunk * per;
        turn1 = turn0 + per < turns ? turn0 + per : turns;
        live_threads = windows && (C - window) / VEC < TH ? (C - window) / VEC : TH;
        first = window + (long long)threadIdx.x * VEC;
        c0 = (int)(first % C);
    }
    __device__ __forceinline__ long long at(long long turn) const { return turn * step + first; }
    __device__ __forceinline__ int live(long long at) const {
        return (int)threadIdx.x >= live_threads ? 0 : N - at >= VEC ? VEC : N > at ? (int)(N - at) : 0;
    }
};

// slab [sample][chunk][2][C] doubles.  Forward: sums of x - pivot and of its square, pivot = the channel's first value of the
// sample.  Backward: sums of du and du xhat.
template <typename T, int VEC, bool BWD>
__global__ __launch_bounds__(512) void grp_partial_kernel(const T* __restrict__ X, const T* __restrict__ DY, long long S, int C, int G,
                                                          int TH, int P, long long chunks, long long per,
                                                          const float* __restrict__ gamma, const float* __restrict__ beta, int act,
                                                          const float* __restrict__ stats, long long BG, double* __restrict__ slab) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const Stream<VEC> st(S, C, TH, chunks, per);
    const long long b = st.sample;
    const T* x = X + b * st.N;
    const T* dy = BWD ? DY + b * st.N : nullptr;
    const bool on = (int)threadIdx.x < st.live_threads;
    Lane<VEC> ln;
    float pivot[VEC];
    if (on) {
        if (BWD) {
            ln.params(st.c0, C, C / G, gamma, beta);
            ln.stats(st.c0, C, C / G, stats + b * G, BG);
        } else {
            grp_walk<VEC>(st.c0, C, C / G, [&](int e, int c, int) { pivot[e] = Elem<T>::load(x + c); });
        }
    }
    double d[2][VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) d[0][e] = d[1][e] = 0.0;
    constexpr int TURNS = BWD ? 4 : 8;
    // TURNS turns from turn i on; `full`: all of them exist and are whole vectors
    auto take = [&](long long i, auto full) {
        u32x4 qx[TURNS], qd[TURNS];
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
            const long long at = st.at(i + k);
            const int live = full ? VEC : i + k < st.turn1 ? st.live(at) : 0;
            qx[k] = live ? grp_load<T, VEC>(x + at, live) : u32x4{0u, 0u, 0u, 0u};
            if (BWD) qd[k] = live ? grp_load<T, VEC>(dy + at, live) : u32x4{0u, 0u, 0u, 0u};
        }
        float s0[VEC], s1[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) s0[e] = s1[e] = 0.f;
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
            const int live = full ? VEC : i + k < st.turn1 ? st.live(st.at(i + k)) : 0;
            if (BWD) {
                float xh[VEC], u[VEC], du[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    xh[e] = ln.xhat(Elem<T>::get(qx[k], e), e);
                    u[e] = ln.u(xh[e], e);
                    du[e] = Elem<T>::get(qd[k], e);
                }
                grp_slope<VEC>(u, du, act);
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (e < live) {
                        s0[e] += du[e];
                        s1[e] += du[e] * xh[e];
                    }
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (e < live) {
                        const float off = Elem<T>::get(qx[k], e) - pivot[e];
                        s0[e] += off;
                        s1[e] += off * off;
                    }
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            d[0][e] += (double)s0[e];
            d[1][e] += (double)s1[e];
        }
    };
    if (on)
        for (long long i = st.turn0; i < st.turn1; i += TURNS) {
            if (i + TURNS <= st.turn1 && st.at(i + TURNS - 1) + VEC <= st.N) take(i, std::true_type());
            else take(i, std::false_type());
        }
    double* out = slab + (long long)blockIdx.x * 2 * C;
    if (gridDim.y > 1) {                                       // the thread's channels are no other's
        if (on)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                out[st.c0 + e] = d[0][e];
                out[C + st.c0 + e] = d[1][e];
            }
        return;
    }
    double* red = reinterpret_cast<double*>(smem);             // [2][blockDim VEC], [2][C]
    double* chan = red + 2 * blockDim.x * VEC;
    grp_channels<double, VEC, 2>(d, TH, P, C, red, chan);
    for (int i = threadIdx.x; i < 2 * C; i += blockDim.x) out[i] = chan[i];
}

// Sums of R rows [2][C] at `rows`, channel c0 + (tid & 7), thirty-two lanes a channel; true in the lane that holds the result.
template <typename F>
__device__ __forceinline__ bool grp_rows(const F* __restrict__ rows, long long R, int C, int c, double& s0, double& s1) {
    __shared__ double part[2][32][8];
    const int cl = threadIdx.x & 7, rl = threadIdx.x >> 3;
    s0 = s1 = 0.0;
    if (c < C)
#pragma unroll 4
        for (long long r = rl; r < R; r += 32) {
            s0 += (double)rows[r * 2 * C + c];
            s1 += (double)rows[r * 2 * C + C + c];
        }
    __syncthreads();                                           // an earlier call's sums have been read
    part[0][rl][cl] = s0;
    part[1][rl][cl] = s1;
    __syncthreads();
    if (rl != 0 || c >= C) return false;
#pragma unroll
    for (int k = 1; k < 32; ++k) {
        s0 += part[0][k][cl];
        s1 += part[1][k][cl];
    }
    return true;
}

// The chunks of a sample joined: csum [sample][2][C] doubles; 8 channels of a sample an item.
__global__ __launch_bounds__(256) void grp_join_kernel(const double* __restrict__ slab, long long B, long long chunks, int C,
                                                       double* __restrict__ csum) {
    const int blocks = (C + 7) / 8;
    for (long long i = blockIdx.x; i < B * blocks; i += gridDim.x) {
        const long long b = i / blocks;
        const int c = (int)(i - b * blocks) * 8 + (threadIdx.x & 7);
        double s0, s1;
        if (!grp_rows(slab + b * chunks * 2 * C, chunks, C, c, s0, s1)) continue;
        csum[b * 2 * C + c] = s0;
        csum[b * 2 * C + C + c] = s1;
    }
}

// stats of the groups of a sample from the channels' sums about their pivots; a wave a group
template <typename T>
__global__ __launch_bounds__(256) void grp_stats_kernel(const double* __restrict__ csum, const T* __restrict__ X, long long S, int C, int G,
                                                        float eps, float* __restrict__ stats, long long BG) {
    const int cg = C / G, lane = threadIdx.x & 63;
    const double rows = (double)S;
    for (long long bg = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); bg < BG; bg += (long long)gridDim.x * 4) {
        const long long b = bg / G;
        const int g = (int)(bg - b * G);
        const double* s = csum + b * 2 * C;
        const T* first = X + b * S * C;
        double sum = 0.0;
        for (int c = g * cg + lane; c < (g + 1) * cg; c += 64) sum += rows * (double)Elem<T>::load(first + c) + s[c];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        const double mean = sum / (rows * cg);
        double m2 = 0.0;
        for (int c = g * cg + lane; c < (g + 1) * cg; c += 64) {
            const double off = (double)Elem<T>::load(first + c) - mean;  // sum (x - mean)^2 from the sums about the pivot
            m2 += s[C + c] + 2.0 * off * s[c] + rows * off * off;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m2 += __shfl_xor(m2, o, 64);
        if (lane) continue;
        const double var = m2 / (rows * cg);
        const float hi = (float)mean;
        stats[bg] = hi;
        stats[BG + bg] = (float)(mean - (double)hi);
        stats[2 * BG + bg] = grp_inv(var > 0.0 || var != var ? var : 0.0, eps);
    }
}

// The elementwise pass.  Backward: the groups' means of d and d xhat from the channels' sums first.
template <typename T, int VEC, bool BWD>
__global__ __launch_bounds__(512) void grp_apply_kernel(const T* __restrict__ X, const T* __restrict__ DY, T* __restrict__ OUT,
                                                        long long S, int C, int G, int TH, long long chunks, long long per,
                                                        const float* __restrict__ gamma, const float* __restrict__ beta, int act,
                                                        const float* __restrict__ stats, long long BG,
                                                        const double* __restrict__ csum) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const Stream<VEC> st(S, C, TH, chunks, per);
    const long long b = st.sample;
    const T* x = X + b * st.N;
    const T* dy = BWD ? DY + b * st.N : nullptr;
    const int cg = C / G;
    float* m0 = reinterpret_cast<float*>(smem);                // [G], [G]
    float* m1 = m0 + G;
    if (BWD) {
        const double* s = csum + b * 2 * C;
        const double n = (double)S * (double)cg;
        grp_groups<4>(G, cg, [&](int c, int) { return (double)(gamma ? gamma[c] : 1.f) * s[c]; },
                      [&](int g, double v) { m0[g] = (float)(v / n); });
        grp_groups<4>(G, cg, [&](int c, int) { return (double)(gamma ? gamma[c] : 1.f) * s[C + c]; },
                   [&](int g, double v) { m1[g] = (float)(v / n); });
    }
    if ((int)threadIdx.x >= st.live_threads) return;
    Lane<VEC> ln;
    ln.params(st.c0, C, C / G, gamma, beta);
    ln.stats(st.c0, C, cg, stats + b * G, BG);
    float a0[VEC], a1[VEC];
    if (BWD)
        grp_walk<VEC>(st.c0, C, cg, [&](int e, int, int g) {
            a0[e] = m0[g];
            a1[e] = m1[g];
        });
    constexpr int TURNS = 4;
    auto take = [&](long long i, auto full) {                  // as in the partial sums
        u32x4 qx[TURNS], qd[TURNS];
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
            const long long at = st.at(i + k);
            const int live = full ? VEC : i + k < st.turn1 ? st.live(at) : 0;
            qx[k] = live ? grp_load<T, VEC>(x + at, live) : u32x4{0u, 0u, 0u, 0u};
            if (BWD) qd[k] = live ? grp_load<T, VEC>(dy + at, live) : u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
            const long long at = st.at(i + k);
            const int live = full ? VEC : i + k < st.turn1 ? st.live(at) : 0;
            if (!live) break;
            float xh[VEC], u[VEC], d[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                xh[e] = ln.xhat(Elem<T>::get(qx[k], e), e);
                u[e] = ln.u(xh[e], e);
            }
            if (BWD) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) d[e] = Elem<T>::get(qd[k], e);
                grp_slope<VEC>(u, d, act);
#pragma unroll
                for (int e = 0; e < VEC; ++e) u[e] = ln.inv[e] * (d[e] * ln.ga[e] - a0[e] - xh[e] * a1[e]);
            } else {
                grp_act<VEC>(u, act);
            }
            grp_store<T, VEC>(OUT + b * st.N + at, u, live);
        }
    };
    for (long long i = st.turn0; i < st.turn1; i += TURNS) {
        if (!BWD && i + TURNS <= st.turn1 && st.at(i + TURNS - 1) + VEC <= st.N) take(i, std::true_type());
        else take(i, std::false_type());
    }
}

// dbeta / dgamma: R rows of [R][2][C] added in fp64
template <typename F>
__global__ __launch_bounds__(256) void grp_params_kernel(const F* __restrict__ rows, long long R, int C, float* __restrict__ dgamma,
                                                         float* __restrict__ dbeta) {
    const int c = blockIdx.x * 8 + (threadIdx.x & 7);
    double s0, s1;
    if (!grp_rows(rows, R, C, c, s0, s1)) return;
    if (dbeta) dbeta[c] = (float)s0;
    if (dgamma) dgamma[c] = (float)s1;
}

// ------------------------------------------------------------------------------------------------------------ host
int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

struct Plan {
    bool one;                  // a workgroup holds a sample
    int vec, period, block, threads, nv, windows;
    long long chunks, per;     // larger samples: chunks of a sample, turns a chunk
    long long rows;            // of partial sums over all samples
};

Plan make_plan(long long B, long long S, int C, int size) {
    Plan p = {};
    const long long N = S * C;
    p.vec = 16 / size;
    p.period = C / gcd(C, p.vec);
    const long long vectors = (N + p.vec - 1) / p.vec;
    p.windows = 1;
    p.one = p.period <= 512 && N * size <= (128 << 10);
    if (p.one) {
        // threads for up to four vectors each, then up to sixteen
        p.block = vectors <= 128 && p.period <= 64 ? 64 : vectors <= 2048 && p.period <= 256 ? 256 : 512;
        p.threads = p.block / p.period * p.period;
        p.nv = (int)((vectors + p.threads - 1) / p.threads);
        p.one = p.nv <= (size == 4 ? 16 : 8);                  // (16-bit values take twice their registers while they are summed)
        p.rows = B < 2048 ? B : 2048;
    }
    if (!p.one) {
        if (p.period > 512) {
            if (C % p.vec) p.vec = 1;
            p.block = p.threads = 256;
            p.windows = (C + 256 * p.vec - 1) / (256 * p.vec);
        } else {
            p.block = p.period <= 256 ? 256 : 512;
            p.threads = p.block / p.period * p.period;
        }
        const long long turns = p.windows > 1 ? S : (vectors + p.threads - 1) / p.threads;
        // some two thousand workgroups, eight turns each at least
        long long chunks = 2048 / (B * p.windows);
        if (chunks > turns / 8) chunks = turns / 8;
        if (chunks < 1) chunks = 1;
        p.per = (turns + chunks - 1) / chunks;
        p.chunks = (turns + p.per - 1) / p.per;
        p.rows = B * p.chunks;
    }
    return p;
}

unsigned loop_grid(long long items) { return (unsigned)(items < (1 << 20) ? items : 1 << 20); }

template <typename T>
int grp_one_lds(const Plan& p, int C, int G, bool bwd) {
    return (2 * p.block * Elem<T>::VEC + 2 * C + (bwd ? 2 * C + 2 * G : C + 3 * G)) * 4;
}

template <typename F>
int with_lds(F* kernel, int bytes) {
    return bytes <= (48 << 10) ? 0
                               : (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

struct Args {
    long long B, S;
    int C, G, act;
    const float *gamma, *beta;
    hipStream_t stream;
};

template <typename T, int NV>
int one_fwd(const Plan& p, const Args& a, const T* X, T* Y, float eps, float* stats) {
    const int lds = grp_one_lds<T>(p, a.C, a.G, false);
    auto* kernel = &grp_one_fwd_kernel<T, NV>;
    if (int rc = with_lds(kernel, lds)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)a.B), dim3(p.block), lds, a.stream, X, Y, (int)(a.S * a.C), a.C, a.G, p.threads, p.period,
                       a.gamma, a.beta, eps, a.act, stats, a.B * a.G);
    DTF_CHECK_LAUNCH();
    return 0;
}
template <typename T, int NV>
int one_bwd(const Plan& p, const Args& a, const T* X, const T* DY, T* DX, const float* stats, float* slab) {
    const int lds = grp_one_lds<T>(p, a.C, a.G, true);
    auto* kernel = &grp_one_bwd_kernel<T, NV>;
    if (int rc = with_lds(kernel, lds)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)p.rows), dim3(p.block), lds, a.stream, X, DY, DX, (int)(a.S * a.C), a.C, a.G, p.threads,
                       p.period, a.B, a.gamma, a.beta, a.act, stats, a.B * a.G, slab);
    DTF_CHECK_LAUNCH();
    return 0;
}

template <typename T, int VEC, bool BWD>
int partial(const Plan& p, const Args& a, const T* X, const T* DY, const float* stats, double* slab, double* csum) {
    const int lds = p.windows > 1 ? 0 : (2 * p.block * VEC + 2 * a.C) * 8;
    auto* kernel = &grp_partial_kernel<T, VEC, BWD>;
    if (int rc = with_lds(kernel, lds)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(p.chunks * a.B), p.windows), dim3(p.block), lds, a.stream, X, DY, a.S, a.C, a.G,
                       p.threads, p.period, p.chunks, p.per, a.gamma, a.beta, a.act, stats, a.B * a.G, slab);
    DTF_CHECK_LAUNCH();
    hipLaunchKernelGGL(grp_join_kernel, dim3(loop_grid(a.B * ((a.C + 7) / 8))), dim3(256), 0, a.stream, slab, a.B, p.chunks, a.C, csum);
    DTF_CHECK_LAUNCH();
    return 0;
}
template <typename T, int VEC, bool BWD>
int apply(const Plan& p, const Args& a, const T* X, const T* DY, T* OUT, const float* stats, const double* csum) {
    const int lds = BWD ? 2 * a.G * 4 : 0;
    auto* kernel = &grp_apply_kernel<T, VEC, BWD>;
    if (int rc = with_lds(kernel, lds)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(p.chunks * a.B), p.windows), dim3(p.block), lds, a.stream, X, DY, OUT, a.S, a.C, a.G,
                       p.threads, p.chunks, p.per, a.gamma, a.beta, a.act, stats, a.B * a.G, csum);
    DTF_CHECK_LAUNCH();
    return 0;
}

// slab [rows][2][C] doubles (floats where a workgroup holds a sample), then csum [B][2][C] doubles
double* csum_of(const Plan& p, const Args& a, double* ws) { return ws + p.rows * 2 * a.C; }

template <typename T>
int grp_fwd(const Args& a, const void* X, void* Y, float eps, float* stats, double* ws) {
    const Plan p = make_plan(a.B, a.S, a.C, sizeof(T));
    const T* x = static_cast<const T*>(X);
    T* y = static_cast<T*>(Y);
    if (p.one) {
        if (p.nv <= 2) return one_fwd<T, 2>(p, a, x, y, eps, stats);
        if (p.nv <= 4) return one_fwd<T, 4>(p, a, x, y, eps, stats);
        if (p.nv <= 8) return one_fwd<T, 8>(p, a, x, y, eps, stats);
        return one_fwd<T, Elem<T>::VEC == 4 ? 16 : 8>(p, a, x, y, eps, stats);
    }
    double* csum = csum_of(p, a, ws);
    const bool whole = p.vec == Elem<T>::VEC;
    int rc = whole ? partial<T, Elem<T>::VEC, false>(p, a, x, nullptr, nullptr, ws, csum)
                   : partial<T, 1, false>(p, a, x, nullptr, nullptr, ws, csum);
    if (rc) return rc;
    hipLaunchKernelGGL(grp_stats_kernel<T>, dim3(loop_grid((a.B * a.G + 3) / 4)), dim3(256), 0, a.stream, csum, x, a.S, a.C, a.G, eps,
                       stats, a.B * a.G);
    DTF_CHECK_LAUNCH();
    return whole ? apply<T, Elem<T>::VEC, false>(p, a, x, nullptr, y, stats, nullptr)
                 : apply<T, 1, false>(p, a, x, nullptr, y, stats, nullptr);
}

template <typename T>
int grp_bwd(const Args& a, const void* X, const void* DY, void* DX, const float* stats, float* dgamma, float* dbeta, double* ws) {
    const Plan p = make_plan(a.B, a.S, a.C, sizeof(T));
    const T *x = static_cast<const T*>(X), *dy = static_cast<const T*>(DY);
    T* dx = static_cast<T*>(DX);
    const bool params = dgamma || dbeta;
    const dim3 cgrid((a.C + 7) / 8);
    if (p.one) {
        float* slab = params ? reinterpret_cast<float*>(ws) : nullptr;
        const int rc = p.nv <= 2   ? one_bwd<T, 2>(p, a, x, dy, dx, stats, slab)
                       : p.nv <= 4 ? one_bwd<T, 4>(p, a, x, dy, dx, stats, slab)
                       : p.nv <= 8 ? one_bwd<T, 8>(p, a, x, dy, dx, stats, slab)
                                   : one_bwd<T, Elem<T>::VEC == 4 ? 16 : 8>(p, a, x, dy, dx, stats, slab);
        if (rc || !params) return rc;
        hipLaunchKernelGGL(grp_params_kernel<float>, cgrid, dim3(256), 0, a.stream, slab, p.rows, a.C, dgamma, dbeta);
        DTF_CHECK_LAUNCH();
        return 0;
    }
    double* csum = csum_of(p, a, ws);
    const bool whole = p.vec == Elem<T>::VEC;
    const int rc = whole ? partial<T, Elem<T>::VEC, true>(p, a, x, dy, stats, ws, csum) : partial<T, 1, true>(p, a, x, dy, stats, ws, csum);
    if (rc) return rc;
    if (params) {
        hipLaunchKernelGGL(grp_params_kernel<double>, cgrid, dim3(256), 0, a.stream, csum, a.B, a.C, dgamma, dbeta);
        DTF_CHECK_LAUNCH();
    }
    if (!dx) return 0;
    return whole ? apply<T, Elem<T>::VEC, true>(p, a, x, dy, dx, stats, csum) : apply<T, 1, true>(p, a, x, dy, dx, stats, csum);
}

bool grp_ok(long long B, long long S, int C, int G, int type, int act) {
    return B > 0 && S > 0 && C > 0 && G > 0 && C % G == 0 && type >= 0 && type <= 2 && act >= ACT_NONE && act <= ACT_SILU &&
           C <= (1 << 20) && G <= (1 << 14) && B <= (1 << 21);
}

}  // namespace

// At most 2097152 samples (a grid's threads are counted in 32 bits), 1048576 channels and 16384 groups (their means stand in LDS).
// doubles of scratch that a call needs, either direction
DTF_API long long dtf_groupnorm_workspace_doubles(long long B, long long S, int C, int type) {
    const Plan p = make_plan(B, S, C, type ? 2 : 4);
    return p.one ? p.rows * C : (p.rows + B) * 2 * C;
}

// type: 0 fp32, 1 bf16, 2 fp16.  gamma / beta may be null.  stats: 3 B G floats, kept for the backward call.
DTF_API int dtf_groupnorm_fwd(const void* X, void* Y, long long B, long long S, int C, int G, int type, const float* gamma,
                              const float* beta, float eps, int act, float* stats, double* workspace, hipStream_t stream) {
    if (!grp_ok(B, S, C, G, type, act)) return -1;
    const Args a = {B, S, C, G, act, gamma, beta, stream};
    if (type == 0) return grp_fwd<float>(a, X, Y, eps, stats, workspace);
    if (type == 1) return grp_fwd<__hip_bfloat16>(a, X, Y, eps, stats, workspace);
    return grp_fwd<__half>(a, X, Y, eps, stats, workspace);
}

// DX, dgamma, dbeta may each be null.
DTF_API int dtf_groupnorm_bwd(const void* X, const void* DY, void* DX, long long B, long long S, int C, int G, int type,
                              const float* gamma, const float* beta, int act, const float* stats, float* dgamma, float* dbeta,
                              double* workspace, hipStream_t stream) {
    if (!grp_ok(B, S, C, G, type, act)) return -1;
    const Args a = {B, S, C, G, act, gamma, beta, stream};
    if (type == 0) return grp_bwd<float>(a, X, DY, DX, stats, dgamma, dbeta, workspace);
    if (type == 1) return grp_bwd<__hip_bfloat16>(a, X, DY, DX, stats, dgamma, dbeta, workspace);
    return grp_bwd<__half>(a, X, DY, DX, stats, dgamma, dbeta, workspace);
}
