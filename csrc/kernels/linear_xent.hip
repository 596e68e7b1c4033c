// Softmax cross entropy of z = x w + b over a large vocabulary, without the logits [M, V] in memory:
//
//   lse_m = log sum_v exp z_mv;   loss_m = lse_m - z_m,label;   rows whose label is `ignore` count for nothing
//   dz = g_m (exp(z - lse) - onehot);   dx = dz w^T;   dw = x^T dz;   db = sum_m dz
//
// The vocabulary is taken in pieces: the forward pass keeps a running maximum and sum of every row, the backward pass computes
// a piece's logits again and turns them into the piece's dz at once.
//
// Masked classes (b = -infinity or the type's lowest value) get probability zero.  A label outside [0, V) that is not `ignore`
// makes the row's loss and gradients NaN.  x may hold anything in ignored rows.
#include "common.h"

#include <hip/hip_bf16.h>

namespace {

constexpr int XT = 64, XK = 16;          // output tile 64 x 64, 16 steps of the reduction in LDS

__device__ __forceinline__ float xe_load(const float* p) { return *p; }
__device__ __forceinline__ float xe_load(const __hip_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void xe_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void xe_store(__hip_bfloat16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ float xe_round(float v, int bf16) { return bf16 ? __bfloat162float(__float2bfloat16(v)) : v; }

// C tile (64 x 64) of A B with A(i, r) and B(r, j) given as functions; thread (ty, tx) holds rows ty + 16 a, columns tx + 16 c
template <typename FA, typename FB>
__device__ __forceinline__ void xe_tile(FA a_at, FB b_at, long long R, float (&acc)[4][4]) {
    __shared__ float as[XK][XT + 1], bs[XK][XT + 1];
    const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[a][c] = 0.f;
    for (long long r0 = 0; r0 < R; r0 += XK) {
        __syncthreads();
        for (int e = tid; e < XK * XT; e += 256) {
            const int r = e / XT, i = e % XT;
            as[r][i] = r0 + r < R ? a_at(i, r0 + r) : 0.f;
            bs[r][i] = r0 + r < R ? b_at(r0 + r, i) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < XK; ++r)
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[a][c] = fmaf(as[r][ty + 16 * a], bs[r][tx + 16 * c], acc[a][c]);
    }
}

// Logits of a 64 x 64 tile.  DZ false: the tile's maximum and sum of exponentials of every row, the label's logit.
// DZ true: dz into the piece's buffer [M, ld] (columns from v0).
template <typename T, bool DZ>
__global__ __launch_bounds__(256) void xe_logits_kernel(const T* __restrict__ X, const T* __restrict__ W, const T* __restrict__ Bv,
                                                        const long long* __restrict__ labels, long long M, long long K, long long V,
                                                        long long v0, long long vend, int bf16, long long ignore,
                                                        float* __restrict__ tmax, float* __restrict__ tsum, long long ntiles,
                                                        float* __restrict__ zlab, const float* __restrict__ lse,
                                                        const float* __restrict__ dloss, int dloss_stride,
                                                        const float* __restrict__ totals, int mean, float* __restrict__ dz,
                                                        long long ld) {
    __shared__ float zt[XT][XT + 1];
    const long long m0 = (long long)blockIdx.y * XT, n0 = v0 + (long long)blockIdx.x * XT;
    float acc[4][4];
    auto a_at = [&](int i, long long r) -> float {
        const long long m = m0 + i;
        return m < M && labels[m] != ignore ? xe_round(xe_load(X + m * K + r), bf16) : 0.f;
    };
    auto b_at = [&](long long r, int j) -> float { return n0 + j < vend ? xe_round(xe_load(W + r * V + n0 + j), bf16) : 0.f; };
    xe_tile(a_at, b_at, K, acc);
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const long long n = n0 + tx + 16 * c;
            zt[ty + 16 * a][tx + 16 * c] = n < vend ? acc[a][c] + (Bv ? xe_load(Bv + n) : 0.f) : -__builtin_inff();
        }
    __syncthreads();
    if (!DZ) {
        const long long m = m0 + threadIdx.x;
        if (threadIdx.x < XT && m < M) {
            float mx = -__builtin_inff(), s = 0.f;
            for (int j = 0; j < XT; ++j) {
                const float z = zt[threadIdx.x][j];
                mx = z > mx || z != z ? z : mx;
            }
            const float shift = mx == -__builtin_inff() ? 0.f : mx;
            for (int j = 0; j < XT; ++j) s += __expf(zt[threadIdx.x][j] - shift);
            const long long tile = (v0 / XT) + blockIdx.x;
            tmax[m * ntiles + tile] = mx;
            tsum[m * ntiles + tile] = s;
            const long long l = labels[m];
            if (l >= n0 && l < n0 + XT && l < vend) zlab[m] = zt[threadIdx.x][l - n0];
        }
    } else {
        for (int e = threadIdx.x; e < XT * XT; e += 256) {
            const int i = e / XT, j = e % XT;
            const long long m = m0 + i, n = n0 + j;
            if (m >= M || n >= vend) continue;
            const long long l = labels[m];
            float g = dloss[m * dloss_stride] * (mean ? 1.f / fmaxf(totals[1], 1.f) : 1.f);
            float d = 0.f;
            if (l != ignore) {
                if (l < 0 || l >= V) g = __builtin_nanf("");
                d = g * (n == l ? expm1f(zt[i][j] - lse[m]) : __expf(zt[i][j] - lse[m]));
            }
            dz[m * ld + (n - v0)] = xe_round(d, bf16);
        }
    }
}

// One wave per row: the tiles' maxima and sums joined; lse and loss.
__global__ __launch_bounds__(64) void xe_merge_kernel(const float* __restrict__ tmax, const float* __restrict__ tsum,
                                                      long long ntiles, const long long* __restrict__ labels, long long V,
                                                      long long ignore, const float* __restrict__ zlab, float* __restrict__ lse,
                                                      float* __restrict__ loss) {
    const long long m = blockIdx.x;
    float mx = -__builtin_inff();
    bool bad = false;
    for (long long t = threadIdx.x; t < ntiles; t += 64) {
        const float v = tmax[m * ntiles + t];
        bad |= v != v;
        mx = fmaxf(mx, v);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    float s = 0.f;
    for (long long t = threadIdx.x; t < ntiles; t += 64) {
        const float v = tmax[m * ntiles + t];
        if (v != -__builtin_inff()) s += tsum[m * ntiles + t] * __expf(v - mx);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (__any(bad)) s = __builtin_nanf("");
    if (threadIdx.x == 0) {
        const float l = mx + __logf(s);
        lse[m] = l;
        const long long at = labels[m];
        loss[m] = at == ignore ? 0.f : at < 0 || at >= V ? __builtin_nanf("") : l - zlab[m];
    }
}

// totals: sum of the losses, counted rows, mean over the counted rows (0 where there are none).  One workgroup, fixed order.
__global__ __launch_bounds__(256) void xe_total_kernel(const float* __restrict__ loss, const long long* __restrict__ labels,
                                                       long long M, long long ignore, float* __restrict__ totals) {
    __shared__ double part[2][256];
    double s = 0.0, n = 0.0;
    for (long long m = threadIdx.x; m < M; m += 256) {
        s += (double)loss[m];
        n += labels[m] != ignore ? 1.0 : 0.0;
    }
    part[0][threadIdx.x] = s;
    part[1][threadIdx.x] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 256; ++k) {
            s += part[0][k];
            n += part[1][k];
        }
        totals[0] = (float)s;
        totals[1] = (float)n;
        totals[2] = (float)(s / fmax(n, 1.0));
    }
}

// dx32 [M, K] (+)= dz [M, cols] w[:, v0 ...]^T
template <typename T>
__global__ __launch_bounds__(256) void xe_dx_kernel(const float* __restrict__ dz, long long ld, const T* __restrict__ W, long long M,
                                                    long long K, long long V, long long v0, long long cols, int bf16, int first,
                                                    int last, float* __restrict__ dx32, T* __restrict__ DX) {
    const long long m0 = (long long)blockIdx.y * XT, k0 = (long long)blockIdx.x * XT;
    float acc[4][4];
    auto a_at = [&](int i, long long r) -> float { return m0 + i < M ? dz[(m0 + i) * ld + r] : 0.f; };
    auto b_at = [&](long long r, int j) -> float { return k0 + j < K ? xe_round(xe_load(W + (k0 + j) * V + v0 + r), bf16) : 0.f; };
    xe_tile(a_at, b_at, cols, acc);
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const long long m = m0 + ty + 16 * a, k = k0 + tx + 16 * c;
            if (m >= M || k >= K) continue;
            const float v = acc[a][c] + (first ? 0.f : dx32[m * K + k]);
            if (last) xe_store(DX + m * K + k, v);
            else dx32[m * K + k] = v;
        }
}

// dw[:, v0 ...] = x^T dz; x counts as zero in ignored rows
template <typename T>
__global__ __launch_bounds__(256) void xe_dw_kernel(const T* __restrict__ X, const float* __restrict__ dz, long long ld,
                                                    const long long* __restrict__ labels, long long M, long long K, long long V,
                                                    long long v0, long long cols, int bf16, long long ignore, T* __restrict__ DW) {
    const long long k0 = (long long)blockIdx.y * XT, n0 = (long long)blockIdx.x * XT;
    float acc[4][4];
    auto a_at = [&](int i, long long r) -> float {
        return k0 + i < K && labels[r] != ignore ? xe_round(xe_load(X + r * K + k0 + i), bf16) : 0.f;
    };
    auto b_at = [&](long long r, int j) -> float { return n0 + j < cols ? dz[r * ld + n0 + j] : 0.f; };
    xe_tile(a_at, b_at, M, acc);
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const long long k = k0 + ty + 16 * a, n = n0 + tx + 16 * c;
            if (k < K && n < cols) xe_store(DW + k * V + v0 + n, acc[a][c]);
        }
}

template <typename T>
__global__ __launch_bounds__(256) void xe_db_kernel(const float* __restrict__ dz, long long ld, long long M, long long cols,
                                                    T* __restrict__ DB) {
    const long long n = (long long)blockIdx.x * 256 + threadIdx.x;
    if (n >= cols) return;
    float s = 0.f;
    for (long long m = 0; m < M; ++m) s += dz[m * ld + n];
    xe_store(DB + n, s);
}

long long xe_piece(long long M, long long V) {
    long long p = (64ll << 20) / (M * 4) / XT * XT;
    if (p < XT) p = XT;
    const long long all = (V + XT - 1) / XT * XT;
    return p < all ? p : all;
}

template <typename T>
int xe_forward(const void* X, const void* W, const void* Bv, const long long* labels, long long M, long long K, long long V, int bf16,
               long long ignore, float* loss, float* lse, float* zlab, float* totals, float* ws, hipStream_t stream) {
    const long long nt = (V + XT - 1) / XT;
    hipLaunchKernelGGL((xe_logits_kernel<T, false>), dim3((unsigned)nt, (unsigned)((M + XT - 1) / XT)), dim3(256), 0, stream,
                       static_cast<const T*>(X), static_cast<const T*>(W), static_cast<const T*>(Bv), labels, M, K, V, 0ll, V, bf16,
                       ignore, ws, ws + M * nt, nt, zlab, nullptr, nullptr, 0, nullptr, 0, nullptr, 0ll);
    DTF_CHECK_LAUNCH();
    hipLaunchKernelGGL(xe_merge_kernel, dim3((unsigned)M), dim3(64), 0, stream, ws, ws + M * nt, nt, labels, V, ignore, zlab, lse,
                       loss);
    DTF_CHECK_LAUNCH();
    hipLaunchKernelGGL(xe_total_kernel, dim3(1), dim3(256), 0, stream, loss, labels, M, ignore, totals);
    DTF_CHECK_LAUNCH();
    return 0;
}

template <typename T>
int xe_backward(const void* X, const void* W, const void* Bv, const long long* labels, long long M, long long K, long long V, int bf16,
                long long ignore, const float* lse, const float* totals, int mean, const float* dloss, int dloss_stride, void* DX,
                void* DW, void* DB, float* ws, hipStream_t stream) {
    const long long piece = xe_piece(M, V);
    float* dz = ws;
    float* dx32 = ws + M * piece;
    const T *x = static_cast<const T*>(X), *w = static_cast<const T*>(W), *b = static_cast<const T*>(Bv);
    const unsigned mt = (unsigned)((M + XT - 1) / XT), kt = (unsigned)((K + XT - 1) / XT);
    for (long long v0 = 0; v0 < V; v0 += piece) {
        const long long cols = v0 + piece < V ? piece : V - v0;
        const unsigned nt = (unsigned)((cols + XT - 1) / XT);
        hipLaunchKernelGGL((xe_logits_kernel<T, true>), dim3(nt, mt), dim3(256), 0, stream, x, w, b, labels, M, K, V, v0, v0 + cols,
                           bf16, ignore, nullptr, nullptr, 0ll, nullptr, lse, dloss, dloss_stride, totals, mean, dz, piece);
        DTF_CHECK_LAUNCH();
        if (DX) {
            hipLaunchKernelGGL(xe_dx_kernel<T>, dim3(kt, mt), dim3(256), 0, stream, dz, piece, w, M, K, V, v0, cols, bf16, v0 == 0,
                               v0 + piece >= V, dx32, static_cast<T*>(DX));
            DTF_CHECK_LAUNCH();
        }
        if (DW) {
            hipLaunchKernelGGL(xe_dw_kernel<T>, dim3(nt, kt), dim3(256), 0, stream, x, dz, piece, labels, M, K, V, v0, cols, bf16,
                               ignore, static_cast<T*>(DW));
            DTF_CHECK_LAUNCH();
        }
        if (DB) {
            hipLaunchKernelGGL(xe_db_kernel<T>, dim3((unsigned)((cols + 255) / 256)), dim3(256), 0, stream, dz, piece, M, cols,
                               static_cast<T*>(DB) + v0);
            DTF_CHECK_LAUNCH();
        }
    }
    return 0;
}

bool xe_ok(long long M, long long K, long long V, int type) {
    return M > 0 && K > 0 && V > 0 && (type == 0 || type == 1) && (M + XT - 1) / XT <= 65535 && (K + XT - 1) / XT <= 65535 &&
           V <= (1ll << 30) && M <= (1ll << 24);
}

}  // namespace

DTF_API long long dtf_linear_xent_fwd_workspace_bytes(long long M, long long K, long long V, int type, int bf16) {
    return M * ((V + XT - 1) / XT) * 8;
}
DTF_API long long dtf_linear_xent_bwd_workspace_bytes(long long M, long long K, long long V, int type, int bf16) {
    return (M * xe_piece(M, V) + M * K) * 4;
}

// type: 0 fp32, 1 bf16 (x, w, b alike; b may be null).  bf16 != 0: fp32 operands rounded to bf16 for the products.
// loss, lse, zlab: M floats each; totals: 4 floats (sum, counted rows, mean).
DTF_API int dtf_linear_xent_fwd(const void* X, const void* W, const void* B, const long long* labels, long long M, long long K,
                                long long V, int type, int bf16, long long ignore, float* loss, float* lse, float* zlab,
                                float* totals, void* workspace, hipStream_t stream) {
    if (!xe_ok(M, K, V, type)) return -1;
    float* ws = static_cast<float*>(workspace);
    if (type == 0) return xe_forward<float>(X, W, B, labels, M, K, V, bf16, ignore, loss, lse, zlab, totals, ws, stream);
    return xe_forward<__hip_bfloat16>(X, W, B, labels, M, K, V, 1, ignore, loss, lse, zlab, totals, ws, stream);
}

// dloss: the loss's gradient, one float for all rows (stride 0) or one a row (stride 1); mean != 0: divided by the counted
// rows.  DX, DW, DB may each be null.
DTF_API int dtf_linear_xent_bwd(const void* X, const void* W, const void* B, const long long* labels, long long M, long long K,
                                long long V, int type, int bf16, long long ignore, const float* lse, const float* zlab,
                                const float* totals, int mean, const float* dloss, int dloss_stride, void* DX, void* DW, void* DB,
                                void* workspace, hipStream_t stream) {
    if (!xe_ok(M, K, V, type)) return -1;
    float* ws = static_cast<float*>(workspace);
    if (type == 0)
        return xe_backward<float>(X, W, B, labels, M, K, V, bf16, ignore, lse, totals, mean, dloss, dloss_stride, DX, DW, DB, ws, stream);
    return xe_backward<__hip_bfloat16>(X, W, B, labels, M, K, V, 1, ignore, lse, totals, mean, dloss, dloss_stride, DX, DW, DB, ws,
                                       stream);
}
