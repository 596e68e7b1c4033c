// Softmax cross entropy of z = x w + b over a large vocabulary, without the logits [M, V] in memory:
//
//   lse_m = log sum_v exp z_mv;   loss_m = lse_m - z_m,label;   rows whose label is `ignore` count for nothing
//   dz = g_m (exp(z - lse) - onehot);   dx = dz w^T;   dw = x^T dz;   db = sum_m dz
//
// Forward: one matrix product whose tiles (256 classes wide) never leave registers as logits: a tile leaves every row's maximum,
// its sum of exponentials and, where the label falls into it, the label's logit.  A second kernel joins the tiles' pairs.
//
// Backward, a piece of the vocabulary at a time: e = exp(z - tile maximum) of the piece -> dz of the piece -> its part of dx
// (added up in fp32 over pieces and splits) and its columns of dw, whole.  Where the forward pass was told to, it has kept e
// for the first `kept` classes (as many as fit the caller's memory budget); the logits of the others are computed again.  What
// the forward pass had to pack of x and w (other types than the products', odd strides) stays for the backward pass too if the
// budget has room (2048 x 1024 x 50021 bf16: 896 -> 850 us).
// With everything kept a training step is the three products that it cannot do without.
//
// Numbers.  bf16 operands multiply as they are.  fp32 operands are scaled by a power of two for each tensor (largest value
// in [2^14, 2^15)) and split into two fp16 limbs of 22 bits together, multiplied as three limb products (half_gemm.h): as exact
// as fp32 products for values from 2^-16 of their tensor's largest on (smaller ones are held to 2^-39 of it), at a third of the
// fp16 rate instead of the sixteenth that fp32 matrix instructions have.  All sums and softmax statistics are fp32 or wider.  e is
// kept in bf16 for bf16 operands: one rounding of a factor of dz, which is rounded to bf16 for its products anyway; fp32 for
// fp32.  dz is held in units of a power of two, and without the loss's gradient where that is one number for all rows: (p - 1) at
// a label is then near -1, which bf16 holds well, instead of the same rounding error in every row; and at the label it comes from
// expm1(z_label - lse), not from a rounded p.
//
// What bounds it: the three products (half_gemm.h), tiles of 256 x 256 by workgroups that stay and take the next tile's first stage
// along; tiles of 64 rows up to 128 rows and where the larger ones would not fill the chip, bound by their loads.  Everything
// else is one pass over what it reads.  Measured, loss and gradients of rows x features x classes: 2048 x 1024 x 50021 bf16 834 us
// (logits 298, dx 223, dw 276, dz 76 at 5.4 TB/s, packing 41 us), 4096 x 1024 x 32000 fp32 2.30 ms (860, 716, 734, 213 at 4.9 TB/s), 8192 x 2048 x 65536 bf16
// 6.37 ms (products at 1.12 PFLOP/s), 128 x 512 x 10001 fp32 101 us in twelve launches; the loss of one row, 512 x 32000 bf16,
// 18 us in two.
//
// Masked classes (b = -infinity or the type's lowest value) get probability zero.  A label outside [0, V) that is not `ignore`
// makes the row's loss and gradients NaN.  x may hold anything in ignored rows: it is packed as zeros there, or read in place
// where only the loss is asked for.
#include "common.h"
#include "half_gemm.h"

#include <hip/hip_bf16.h>

namespace {

using hgemm::Gemm;
using hgemm::lds_char;
using hgemm::s16x8;
using hgemm::Tile;

constexpr int XT = 256;                          // classes a tile
constexpr long long XE_PIECE_BYTES = 512ll << 20; // dz of a piece
constexpr long long XE_PACK_BYTES = 512ll << 20;  // w of a piece where it has to be packed
constexpr float XE_DZ_SCALE = 16384.f;           // what dz, below 2 in its units, is multiplied by before it is split

template <int PL>
struct HalfOf {
    typedef __bf16 type;
};
template <>
struct HalfOf<2> {
    typedef _Float16 type;
};

__device__ __forceinline__ float xe_load(const float* p) { return *p; }
__device__ __forceinline__ float xe_load(const __hip_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ short xe_bf16(float v) {
    const __hip_bfloat16 h = __float2bfloat16(v);
    return __builtin_bit_cast(short, h);
}

// power of two that brings a largest magnitude (its bits) into [2^14, 2^15), and its inverse
__device__ __forceinline__ float xe_scale(unsigned amax_bits) {
    const int e = (int)(amax_bits >> 23);                       // biased exponent; subnormal maxima count as the smallest normal
    const int s = 127 + 14 - ((e < 1 ? 1 : e) - 127);
    return amax_bits == 0 ? 1.f : __uint_as_float((unsigned)(s > 253 ? 253 : s) << 23);
}

// ---- scales: the largest finite magnitudes of x (counted rows) and w.  XE_AMAX workgroups leave one partial maximum each for
// x (rows dealt round) and for w (chunks); the kernel that packs x, the next one, joins them and leaves the result.
constexpr int XE_AMAX = 1024;

__device__ __forceinline__ float xe_block_max(float m) {
    __shared__ float part[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    return fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
}

__device__ __forceinline__ float xe_amax_range(const float* __restrict__ p, long long begin, long long end) {
    const float inf = __builtin_inff();
    float m = 0.f;
    auto take = [&](float v) {
        const float a = fabsf(v);
        m = a < inf ? fmaxf(m, a) : m;
    };
    long long i = begin + threadIdx.x * 4;
    for (; i + 3 * 1024 + 3 < end; i += 4096) {                 // 64 bytes a thread in flight
        hgemm::f32x4_any v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const hgemm::f32x4_any*>(p + i + u * 1024);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) take(v[u][e]);
    }
    for (; i < end; i += 1024)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < end) take(p[i + e]);
    return m;
}

__global__ __launch_bounds__(256) void xe_amax_kernel(const float* __restrict__ X, long long M, long long K,
                                                      const long long* __restrict__ labels, long long ignore,
                                                      const float* __restrict__ W, long long KV, float* __restrict__ partial) {
    float m = 0.f;
    for (long long r = blockIdx.x; r < M; r += XE_AMAX)
        if (labels[r] != ignore) m = fmaxf(m, xe_amax_range(X, r * K, (r + 1) * K));
    m = xe_block_max(m);
    if (threadIdx.x == 0) partial[blockIdx.x] = m;
    const long long chunk = ((KV + XE_AMAX - 1) / XE_AMAX + 3) / 4 * 4, begin = blockIdx.x * chunk;
    m = xe_block_max(begin < KV ? xe_amax_range(W, begin, begin + chunk < KV ? begin + chunk : KV) : 0.f);
    if (threadIdx.x == 0) partial[XE_AMAX + blockIdx.x] = m;
}

// ---- packing: [rows, cols] of any alignment -> rows of ld halves, zero behind cols; rows labelled `ignore` as zeros.
// `partial` (x only): the partial maxima, joined here into amax[0] (x) and amax[1] (w).
template <typename T, int PL>
__global__ __launch_bounds__(256) void xe_pack_kernel(const T* __restrict__ src, long long ld_src, long long rows, long long cols,
                                                      short* __restrict__ dst, long long ld, const long long* __restrict__ labels,
                                                      long long ignore, const float* __restrict__ partial, unsigned* __restrict__ amax) {
    const long long per_row = ld / PL / 8;                      // groups of 8 values
    const long long total = rows * per_row;
    float scale = 1.f;
    if (PL == 2) {
        if (partial) {
            float m = 0.f, w = 0.f;
#pragma unroll
            for (int k = 0; k < XE_AMAX / 256; ++k) {
                m = fmaxf(m, partial[k * 256 + threadIdx.x]);
                w = fmaxf(w, partial[XE_AMAX + k * 256 + threadIdx.x]);
            }
            m = xe_block_max(m);
            if (blockIdx.x == 0) {
                w = xe_block_max(w);
                if (threadIdx.x == 0) {
                    amax[0] = __float_as_uint(m);
                    amax[1] = __float_as_uint(w);
                }
            }
            scale = xe_scale(__float_as_uint(m));
        } else {
            scale = xe_scale(*amax);
        }
    }
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / per_row, c = (i - r * per_row) * 8;
        float v[8];
        const bool skip = labels && labels[r] == ignore;
        const T* p = src + r * ld_src + c;
        if (c + 8 <= cols && !skip) {                           // vector loads at the element's alignment
            if (sizeof(T) == 2) {
                const s16x8 q = *reinterpret_cast<const hgemm::s16x8_any*>(p);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = __uint_as_float((unsigned)(unsigned short)q[e] << 16);
            } else {
                const f32x4 a = *reinterpret_cast<const hgemm::f32x4_any*>(p), b = *reinterpret_cast<const hgemm::f32x4_any*>(p + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = a[e];
                    v[4 + e] = b[e];
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = !skip && c + e < cols ? xe_load(p + e) : 0.f;
        }
        s16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (PL == 1) {
                hi[e] = xe_bf16(v[e]);
            } else {
                const float s = v[e] * scale;
                const _Float16 h = (_Float16)s;
                const _Float16 l = fabsf((float)h) < __builtin_inff() ? (_Float16)(s - (float)h) : (_Float16)0.f;
                hi[e] = __builtin_bit_cast(short, h);
                lo[e] = __builtin_bit_cast(short, l);
            }
        }
        short* q = dst + r * ld + (PL == 1 ? c : c / 32 * 64 + c % 32);
        *reinterpret_cast<s16x8*>(q) = hi;
        if (PL == 2) *reinterpret_cast<s16x8*>(q + 32) = lo;
    }
}

// ---- logits of an LN x 256 tile and what the softmax needs of them
template <int PL, int LN, int WL, int WR>
__global__ __launch_bounds__(64 * WL * WR) void xe_logits_kernel(
    const short* __restrict__ X, long long ldx, const short* __restrict__ W, long long ldw, long long w_left,
    const void* __restrict__ bias, int bias_bf16, const long long* __restrict__ labels, long long M, long long K, long long v0,
    long long vend, const unsigned* __restrict__ amax, float* __restrict__ tmax, float* __restrict__ tsum,
    float* __restrict__ zlab, float* __restrict__ beaten, void* __restrict__ E, long long lde, long long e0, long long e_tiles) {
    typedef Gemm<typename HalfOf<PL>::type, PL, LN, XT, WL, WR, false, true, LN == 64 ? 3 : 2> G;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* sbias = reinterpret_cast<float*>(smem + G::LDS_BYTES);   // [256]
    float* smax = sbias + XT;                                   // [WR][LN]
    float* ssum = smax + WR * LN;                               // [WR][LN]
    float* slab = ssum + WR * LN;                               // [LN]: the labels' logits
    unsigned* sbeat = reinterpret_cast<unsigned*>(slab + LN);   // [LN]
    const long long nrow = (M + LN - 1) / LN, ncol = (vend - v0 + XT - 1) / XT;
    auto job_at = [&](long long t, long long& m0, long long& n0) {
        long long rt, ct;
        hgemm::tile_at(t, nrow, ncol, rt, ct);
        m0 = rt * LN, n0 = ct * XT;                             // n0 within the piece
        return typename G::Job{{reinterpret_cast<const char*>(X + m0 * ldx), (M - m0) * ldx * 2, ldx * 2},
                               {reinterpret_cast<const char*>(W + n0 * PL), w_left - n0 * PL * 2, ldw * 2},
                               (int)(ldx / 64)};
    };
    const hgemm::Deal deal(nrow * ncol);
    bool primed = false;
    int buffer = 0;
    for (long long t = deal.first; t < deal.end; t += deal.stride) {
        const bool more = t + deal.stride < deal.end;
        long long m0, n0, next_m0, next_n0;
        const typename G::Job job = job_at(t, m0, n0), next = more ? job_at(t + deal.stride, next_m0, next_n0) : job;
        const long long ct = n0 / XT;
        f32x16 acc[G::TL][G::TR];
        G::run(job, next, more, primed, buffer, (lds_char*)smem, acc);

        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wl = wave / WR, wr = wave % WR;
        for (int i = tid; i < XT; i += G::THREADS) {
            const long long n = v0 + n0 + i;
            sbias[i] = n >= vend ? -__builtin_inff() : !bias ? 0.f : bias_bf16 ? xe_load(static_cast<const __hip_bfloat16*>(bias) + n)
                                                                                : static_cast<const float*>(bias)[n];
        }
        for (int i = tid; i < LN; i += G::THREADS) sbeat[i] = 0u;
        __syncthreads();
        const float ix = PL == 2 ? 1.f / xe_scale(amax[0]) : 1.f, iw = PL == 2 ? 1.f / xe_scale(amax[1]) : 1.f;
        const bool full = v0 + n0 + XT <= vend;
        const int nw = wr * (XT / WR) + 4 * (lane >> 5);            // first class of this lane's, within the tile
        int own[G::TL];                                             // the row's label within the tile, or out of it
        bool any_own = false;
#pragma unroll
        for (int a = 0; a < G::TL; ++a) {
            const int ml = wl * (LN / WL) + a * 32 + (lane & 31);
            const long long l = m0 + ml < M ? labels[m0 + ml] - v0 - n0 : -1;
            own[a] = l >= 0 && l < XT && v0 + n0 + l < vend ? (int)l : -1;
            any_own |= own[a] >= 0;
            float mx = -__builtin_inff();
#pragma unroll
            for (int b = 0; b < G::TR; ++b)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 bz = *reinterpret_cast<const f32x4*>(sbias + nw + b * 32 + q * 8);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float z = acc[a][b][q * 4 + i];
                        if (PL == 2) z = z * ix * iw;
                        z = full || v0 + n0 + nw + b * 32 + q * 8 + i < vend ? z + bz[i] : -__builtin_inff();
                        acc[a][b][q * 4 + i] = z;
                        mx = fmaxf(mx, z);
                    }
                }
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            if (lane < 32) smax[wr * LN + ml] = mx;
        }
        any_own = __any(any_own);
        if (any_own) {                                              // few tiles hold any label of their rows
#pragma unroll
            for (int a = 0; a < G::TL; ++a)
#pragma unroll
                for (int b = 0; b < G::TR; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (nw + b * 32 + (r >> 2) * 8 + (r & 3) == own[a]) slab[wl * (LN / WL) + a * 32 + (lane & 31)] = acc[a][b][r];
        }
        __syncthreads();
        const bool keep = E && ct < e_tiles;
#pragma unroll
        for (int a = 0; a < G::TL; ++a) {
            const int ml = wl * (LN / WL) + a * 32 + (lane & 31);
            float mx = smax[ml];
#pragma unroll
            for (int w = 1; w < WR; ++w) mx = fmaxf(mx, smax[w * LN + ml]);
            const float shift = mx == -__builtin_inff() ? 0.f : mx;
            float s = 0.f;
            if (any_own && own[a] >= 0) {                           // does another class of the tile beat the label's?
                const float zl = slab[ml];
                bool beat = false;
#pragma unroll
                for (int b = 0; b < G::TR; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float z = acc[a][b][r];
                        beat |= z > zl || (z == zl && nw + b * 32 + (r >> 2) * 8 + (r & 3) < own[a]);
                    }
                if (beat) sbeat[ml] = 1u;                           // all write the same
            }
#pragma unroll
            for (int b = 0; b < G::TR; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float e = __expf(acc[a][b][r] - shift);
                    acc[a][b][r] = e;
                    s += e;
                }
            s += __shfl_xor(s, 32, 64);
            if (lane < 32) ssum[wr * LN + ml] = s;
            if (keep && m0 + ml < M) {
#pragma unroll
                for (int b = 0; b < G::TR; ++b) {
                    if (PL == 2) {
                        float* out = static_cast<float*>(E) + (m0 + ml) * lde + e0 + n0 + nw + b * 32;
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            *reinterpret_cast<f32x4*>(out + q * 8) =
                                f32x4{acc[a][b][q * 4], acc[a][b][q * 4 + 1], acc[a][b][q * 4 + 2], acc[a][b][q * 4 + 3]};
                    }
                }
            }
            if (PL == 1 && keep) {
                short* out = static_cast<short*>(E) + (m0 + ml) * lde + e0 + n0 + wr * (XT / WR) + 8 * (lane >> 5);
#pragma unroll
                for (int b = 0; b < G::TR; ++b) hgemm::store_bf16_16(acc[a][b], 1.f, out + b * 32, m0 + ml < M);
            }
        }
        __syncthreads();
        for (int i = tid; i < LN; i += G::THREADS) {
            const long long m = m0 + i;
            if (m >= M) continue;
            float mx = smax[i], s = ssum[i];
#pragma unroll
            for (int w = 1; w < WR; ++w) {
                mx = fmaxf(mx, smax[w * LN + i]);
                s += ssum[w * LN + i];
            }
            const long long tile = v0 / XT + ct;
            if (tsum) {
                tmax[tile * M + m] = mx;
                tsum[tile * M + m] = s;
                const long long l = labels[m] - v0 - n0;
                if (l >= 0 && l < XT && v0 + n0 + l < vend) {
                    zlab[m] = slab[i];
                    beaten[m] = sbeat[i] ? 1.f : 0.f;
                }
            }
        }
        __syncthreads();                                            // the tile's statistics have been read
    }
}

// ---- the tiles' maxima and sums joined: lse, loss, whether the label has the largest logit (ties to the lowest class).
// A workgroup takes `rows` rows (a power of two up to 16: reads of 64 bytes), 256 / rows threads a row.
__global__ __launch_bounds__(256) void xe_merge_kernel(const float* __restrict__ tmax, const float* __restrict__ tsum, long long ntiles,
                                                       const long long* __restrict__ labels, long long M, long long V, long long ignore,
                                                       int rows, const float* __restrict__ zlab, const float* __restrict__ beaten,
                                                       float* __restrict__ lse, float* __restrict__ loss, float* __restrict__ hit) {
    __shared__ float smax[256], ssum[256], slost[256];
    const int lanes = 256 / rows, rl = threadIdx.x % rows, tl = threadIdx.x / rows;
    const long long m = (long long)blockIdx.x * rows + rl;
    const bool live = m < M;
    const long long label = live ? labels[m] : ignore;
    const bool valid = live && label != ignore && label >= 0 && label < V;
    const float zl = valid ? zlab[m] : 0.f;
    const long long own = valid ? label / XT : -1;
    float mx = -__builtin_inff(), s = 0.f, lost = 0.f;
    if (live)
#pragma unroll 4
        for (long long t = tl; t < ntiles; t += lanes) {
            const float v = tmax[t * M + m], w = tsum[t * M + m];
            const float top = fmaxf(mx, v), ref = top == -__builtin_inff() ? 0.f : top;
            s = s * __expf(mx - ref) + w * __expf(v - ref);
            mx = top;
            if (t != own && (v > zl || (v == zl && t < own))) lost = 1.f;
        }
    smax[threadIdx.x] = mx;
    ssum[threadIdx.x] = s;
    slost[threadIdx.x] = lost;
    __syncthreads();
    for (int half = lanes / 2; half > 0; half /= 2) {           // a tree: the order of the sums is that of the sizes alone
        if (tl < half) {
            const int o = threadIdx.x + half * rows;
            const float v = smax[o], top = fmaxf(mx, v), ref = top == -__builtin_inff() ? 0.f : top;
            s = s * __expf(mx - ref) + ssum[o] * __expf(v - ref);
            mx = top;
            lost += slost[o];
            smax[threadIdx.x] = mx;
            ssum[threadIdx.x] = s;
            slost[threadIdx.x] = lost;
        }
        __syncthreads();
    }
    if (tl != 0 || !live) return;
    // a row without any class (all masked) has no loss: NaN, as a sum of zeros gives
    const float l = mx == -__builtin_inff() ? __builtin_nanf("") : mx + logf(s);
    lse[m] = l;
    loss[m] = label == ignore ? 0.f : valid ? l - zl : __builtin_nanf("");
    hit[m] = valid && lost == 0.f && beaten[m] == 0.f ? 1.f : 0.f;
}

// totals: sum of the losses, hits, counted rows, mean over the counted rows (0 where there are none); reduced (may be null): the
// mean (reduction 1) or the sum (2).  One workgroup, fixed order.
__global__ __launch_bounds__(1024) void xe_total_kernel(const float* __restrict__ loss, const float* __restrict__ hit,
                                                        const long long* __restrict__ labels, long long M, long long ignore,
                                                        float* __restrict__ totals, int reduction, float* __restrict__ reduced) {
    __shared__ double part[3][16];
    double s = 0.0, n = 0.0, h = 0.0;
    for (long long m = threadIdx.x; m < M; m += 1024) {
        s += (double)loss[m];
        h += (double)hit[m];
        n += labels[m] != ignore ? 1.0 : 0.0;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        s += __shfl_xor(s, o, 64);
        n += __shfl_xor(n, o, 64);
        h += __shfl_xor(h, o, 64);
    }
    if ((threadIdx.x & 63) == 0) {
        part[0][threadIdx.x >> 6] = s;
        part[1][threadIdx.x >> 6] = n;
        part[2][threadIdx.x >> 6] = h;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = n = h = 0.0;
        for (int k = 0; k < 16; ++k) {
            s += part[0][k];
            n += part[1][k];
            h += part[2][k];
        }
        totals[0] = (float)s;
        totals[1] = (float)h;
        totals[2] = (float)n;
        totals[3] = (float)(s / fmax(n, 1.0));
        if (reduced) *reduced = reduction == 1 ? totals[3] : totals[0];
    }
}

// ---- weights of the rows, one workgroup: rowg[m] *scale = the gradient of row m's loss.
// The largest |dz| of a row is 1 - p_label (the other probabilities add up to it).  *scale holds the power of two of the largest
// one over all rows, so that dz / *scale is below 2 and near 1 somewhere, also where every row is confident: fp16 limbs resolve
// 2^-39 of that.
__global__ __launch_bounds__(1024) void xe_weights_kernel(const float* __restrict__ dloss, int stride, const float* __restrict__ totals,
                                                          int mean, const long long* __restrict__ labels, long long M, long long V,
                                                          long long ignore, const float* __restrict__ lse, const float* __restrict__ zlab,
                                                          float* __restrict__ rowg, float* __restrict__ scale) {
    __shared__ float part[16];
    float m = 0.f;
    for (long long i = threadIdx.x; i < M; i += 1024) {
        const long long l = labels[i];
        const bool valid = l != ignore && l >= 0 && l < V;
        const float w = stride ? dloss[i] : 1.f;
        rowg[i] = l == ignore ? 0.f : valid ? w : __builtin_nanf("");
        const float d = valid ? fabsf(w * expm1f(zlab[i] - lse[i])) : 0.f;
        if (d < __builtin_inff()) m = fmaxf(m, d);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    m = part[0];
    for (int k = 1; k < 16; ++k) m = fmaxf(m, part[k]);
    const int e = (int)(__float_as_uint(m) >> 23) - 127;
    const int unit = m == 0.f ? 0 : e < -100 ? -100 : e > 100 ? 100 : e;
    const float down = __uint_as_float((unsigned)(127 - unit) << 23);
    for (long long i = threadIdx.x; i < M; i += 1024) rowg[i] *= down;
    if (threadIdx.x == 0)
        *scale = (stride ? 1.f : *dloss) * (mean ? 1.f / fmaxf(totals[2], 1.f) : 1.f) * __uint_as_float((unsigned)(127 + unit) << 23);
}

// ---- e of a piece -> its dz, ROWS rows x 256 classes a workgroup; dbp [row blocks][ld]: the columns' sums over its rows.  64 rows
// a workgroup, 16 where that would leave the chip idle.
template <int PL, int ROWS>
__global__ __launch_bounds__(256) void xe_dz_kernel(const void* __restrict__ E, long long lde, long long e0,
                                                    const float* __restrict__ tmax, const float* __restrict__ lse,
                                                    const float* __restrict__ zlab, const float* __restrict__ rowg,
                                                    const long long* __restrict__ labels, long long M, long long v0,
                                                    short* __restrict__ dz, long long ld, float* __restrict__ dbp) {
    __shared__ float f[ROWS], at_label[ROWS];
    __shared__ int own[ROWS];
    __shared__ float sums[8][XT];
    const long long m0 = (long long)blockIdx.y * ROWS, n0 = (long long)blockIdx.x * XT;
    if (threadIdx.x < ROWS) {
        const long long m = m0 + threadIdx.x;
        const float g = m < M ? rowg[m] : 0.f;
        const float mx = m < M ? tmax[(v0 / XT + blockIdx.x) * M + m] : 0.f;
        const float l = m < M ? lse[m] : 0.f;
        f[threadIdx.x] = g != 0.f ? g * __expf(mx == -__builtin_inff() ? -__builtin_inff() : mx - l) : 0.f;
        const long long lab = m < M ? labels[m] - v0 - n0 : -1;
        own[threadIdx.x] = lab >= 0 && lab < XT ? (int)lab : -1;
        at_label[threadIdx.x] = own[threadIdx.x] >= 0 && g != 0.f ? g * expm1f(zlab[m] - l) : 0.f;
    }
    __syncthreads();
    const int cl = (threadIdx.x & 31) * 8, rl = threadIdx.x >> 5;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < ROWS / 8; ++i) {
        const int r = rl + i * 8;
        const long long m = m0 + r;
        if (m >= M) continue;
        float d[8];
        if (PL == 1) {
            const s16x8 e = *reinterpret_cast<const s16x8*>(static_cast<const short*>(E) + m * lde + e0 + n0 + cl);
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = __uint_as_float((unsigned)(unsigned short)e[j] << 16);
        } else {
            const float* p = static_cast<const float*>(E) + m * lde + e0 + n0 + cl;
            const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                d[j] = a[j];
                d[4 + j] = b[j];
            }
        }
        s16x8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float v = cl + j == own[r] ? at_label[r] : d[j] * f[r];
            sum[j] += v;
            if (PL == 1) {
                hi[j] = xe_bf16(v);
            } else {
                const float s = v * XE_DZ_SCALE;
                const _Float16 h = (_Float16)s;
                hi[j] = __builtin_bit_cast(short, h);
                lo[j] = __builtin_bit_cast(short, (_Float16)(s - (float)h));
            }
        }
        short* out = dz + m * ld + (PL == 1 ? n0 + cl : (n0 + cl) / 32 * 64 + cl % 32);
        *reinterpret_cast<s16x8*>(out) = hi;
        if (PL == 2) *reinterpret_cast<s16x8*>(out + 32) = lo;
    }
    if (!dbp) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[rl][cl + j] = sum[j];
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += sums[k][threadIdx.x];
    dbp[(long long)blockIdx.y * (ld / PL) + n0 + threadIdx.x] = s;
}

__device__ __forceinline__ void xe_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void xe_put(__hip_bfloat16* p, float v) { *p = __float2bfloat16(v); }

template <typename T>
__global__ __launch_bounds__(256) void xe_db_kernel(const float* __restrict__ dbp, long long blocks, long long ld, long long cols,
                                                    const float* __restrict__ scale, T* __restrict__ DB) {
    __shared__ double part[8][32];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const long long n = (long long)blockIdx.x * 32 + cl;
    double s = 0.0;
    if (n < cols)
#pragma unroll 4
        for (long long r = rl; r < blocks; r += 8) s += (double)dbp[r * ld + n];
    part[rl][cl] = s;
    __syncthreads();
    if (rl != 0 || n >= cols) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) s += part[k][cl];
    xe_put(DB + n, (float)s * *scale);
}

// ---- slab [split][M][ldk] (+)= dz w^T over a range of the piece's classes
template <int PL, int LN, int WL, int WR>
__global__ __launch_bounds__(64 * WL * WR) void xe_dx_kernel(const short* __restrict__ dz, long long ldz, const short* __restrict__ W,
                                                             long long ldw, long long w_left, long long M, long long K, int blocks,
                                                             int splits, int accumulate, float* __restrict__ slab, long long ldk) {
    typedef Gemm<typename HalfOf<PL>::type, PL, LN, XT, WL, WR, false, false, LN == 64 ? 3 : 2> G;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const long long nrow = (M + LN - 1) / LN, ncol = (K + XT - 1) / XT, tiles = nrow * ncol;
    auto job_at = [&](long long t, long long& m0, long long& k0, int& split) {
        long long rt, ct;
        split = (int)(t / tiles);
        hgemm::tile_at(t - split * tiles, nrow, ncol, rt, ct);
        m0 = rt * LN, k0 = ct * XT;
        const int b0 = (int)((long long)blocks * split / splits), b1 = (int)((long long)blocks * (split + 1) / splits);
        const long long skip = (long long)b0 * 128;
        return typename G::Job{{reinterpret_cast<const char*>(dz + m0 * ldz) + skip, (M - m0) * ldz * 2 - skip, ldz * 2},
                               {reinterpret_cast<const char*>(W + k0 * ldw) + skip, w_left - k0 * ldw * 2 - skip, ldw * 2},
                               b1 - b0};
    };
    const hgemm::Deal deal(tiles * splits);
    bool primed = false;
    int buffer = 0;
    for (long long t = deal.first; t < deal.end; t += deal.stride) {
        const bool more = t + deal.stride < deal.end;
        long long m0, k0, next_m0, next_k0;
        int split, next_split;
        const typename G::Job job = job_at(t, m0, k0, split), next = more ? job_at(t + deal.stride, next_m0, next_k0, next_split) : job;
        f32x16 acc[G::TL][G::TR];
        G::run(job, next, more, primed, buffer, (lds_char*)smem, acc);
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wl = wave / WR, wr = wave % WR;
#pragma unroll
        for (int a = 0; a < G::TL; ++a) {
            const long long m = m0 + wl * (LN / WL) + a * 32 + (lane & 31);
            if (m >= M) continue;
#pragma unroll
            for (int b = 0; b < G::TR; ++b)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const long long k = k0 + wr * (XT / WR) + b * 32 + q * 8 + 4 * (lane >> 5);
                    if (k >= ldk) continue;
                    float* out = slab + ((long long)split * M + m) * ldk + k;
                    f32x4 v = {acc[a][b][q * 4], acc[a][b][q * 4 + 1], acc[a][b][q * 4 + 2], acc[a][b][q * 4 + 3]};
                    if (accumulate) v += *reinterpret_cast<const f32x4*>(out);
                    *reinterpret_cast<f32x4*>(out) = v;
                }
        }
    }
}

template <typename T, int PL>
__global__ __launch_bounds__(256) void xe_dx_finish_kernel(const float* __restrict__ slab, int splits, long long M, long long K,
                                                           long long ldk, const unsigned* __restrict__ amax,
                                                           const float* __restrict__ scale, T* __restrict__ DX) {
    const float iw = PL == 2 ? 1.f / xe_scale(amax[1]) / XE_DZ_SCALE : 1.f;
    const float g = *scale;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < M * K; i += (long long)gridDim.x * 256) {
        const long long m = i / K, k = i - m * K;
        float s = 0.f;
#pragma unroll 8
        for (int p = 0; p < splits; ++p) s += slab[((long long)p * M + m) * ldk + k];
        xe_put(DX + i, s * iw * g);
    }
}

// ---- dw[:, v0 ...] = x^T dz
template <int PL, int OUT_BF16, int LN, int WL, int WR>
__global__ __launch_bounds__(64 * WL * WR) void xe_dw_kernel(const short* __restrict__ X, long long ldx, const short* __restrict__ dz,
                                                             long long ldz, long long dz_left, long long M, long long K,
                                                             long long cols, const unsigned* __restrict__ amax,
                                                             const float* __restrict__ scale, void* __restrict__ DW, long long V,
                                                             long long v0) {
    typedef Gemm<typename HalfOf<PL>::type, PL, LN, XT, WL, WR, true, true, LN == 64 ? 3 : 2> G;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const long long nrow = (K + LN - 1) / LN, ncol = (cols + XT - 1) / XT;
    auto job_at = [&](long long t, long long& k0, long long& n0) {
        long long rt, ct;
        hgemm::tile_at(t, nrow, ncol, rt, ct);
        k0 = rt * LN, n0 = ct * XT;
        return typename G::Job{{reinterpret_cast<const char*>(X + k0 * PL), M * ldx * 2 - k0 * PL * 2, ldx * 2},
                               {reinterpret_cast<const char*>(dz + n0 * PL), dz_left - n0 * PL * 2, ldz * 2},
                               (int)((M + G::CB - 1) / G::CB)};
    };
    const hgemm::Deal deal(nrow * ncol);
    bool primed = false;
    int buffer = 0;
    for (long long t = deal.first; t < deal.end; t += deal.stride) {
        const bool more = t + deal.stride < deal.end;
        long long k0, n0, next_k0, next_n0;
        const typename G::Job job = job_at(t, k0, n0), next = more ? job_at(t + deal.stride, next_k0, next_n0) : job;
        f32x16 acc[G::TL][G::TR];
        G::run(job, next, more, primed, buffer, (lds_char*)smem, acc);
        const float ix = PL == 2 ? 1.f / xe_scale(amax[0]) / XE_DZ_SCALE : 1.f;
        const float g = *scale;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wl = wave / WR, wr = wave % WR;
#pragma unroll
        for (int a = 0; a < G::TL; ++a) {
            const long long k = k0 + wl * (LN / WL) + a * 32 + (lane & 31);
            if (OUT_BF16) {
                short* out = static_cast<short*>(DW) + k * V + v0;
                const long long n = n0 + wr * 64 + 8 * (lane >> 5);
#pragma unroll
                for (int b = 0; b < G::TR; ++b) {
                    if (n0 + wr * 64 + b * 32 + 32 <= cols) {
                        hgemm::store_bf16_16(acc[a][b], g, out + n + b * 32, k < K);
                    } else if (k < K) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const long long c = n0 + wr * 64 + b * 32 + (r >> 2) * 8 + 4 * (lane >> 5) + (r & 3);
                            if (c < cols) out[c] = xe_bf16(acc[a][b][r] * g);
                        }
                    }
                }
            } else {
                float* out = static_cast<float*>(DW) + k * V + v0;
                if (k >= K) continue;
#pragma unroll
                for (int b = 0; b < G::TR; ++b)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const long long c = n0 + wr * 64 + b * 32 + q * 8 + 4 * (lane >> 5);
                        hgemm::f32x4_any v;
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = acc[a][b][q * 4 + i] * ix * g;
                        if (c + 4 <= cols) {
                            *reinterpret_cast<hgemm::f32x4_any*>(out + c) = v;
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (c + i < cols) out[c + i] = v[i];
                        }
                    }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ host
inline long long up(long long v, long long to) { return (v + to - 1) / to * to; }
inline long long lowest(long long a, long long b) { return a < b ? a : b; }

struct Plan {
    long long M, K, V;
    int type, pl;              // 0 fp32, 1 bf16 operands; limbs a value
    bool packs;                // w has to be packed
    bool small, small_dx;      // 64 rows of x a tile: for the logits, for dx
    long long ldx, ldw, piece, tiles;
    long long esize;
    int splits;                // of the classes of a piece for dx
    long long ldk;
};

Plan make_plan(const void* W, long long M, long long K, long long V, int type, int bf16) {
    Plan p;
    p.M = M, p.K = K, p.V = V, p.type = type;
    p.pl = type == 0 && !bf16 ? 2 : 1;
    const int cb = 64 / p.pl;
    p.packs = type == 0 || V % 8 != 0 || (reinterpret_cast<uintptr_t>(W) & 15) != 0;
    p.ldx = up(K, cb) * p.pl;
    p.tiles = (V + XT - 1) / XT;
    // 64 rows a tile where few rows would leave most of a larger one empty, or where the larger ones do not fill the chip: a stage
    // takes some 1.3 us with 64 rows, 2 us with 256, a round 256 workgroups.  (346 rows, 2752 features, 1792 classes, fp32, loss
    // alone: 110 us with 42 tiles, 187 us with 14.)
    const double few = 1.3e-6, many = 2e-6;
    p.small = M <= 128 || (double)(((M + 63) / 64 * p.tiles + 255) / 256) * few < (double)(((M + 255) / 256 * p.tiles + 255) / 256) * many;
    p.esize = p.pl == 2 ? 4 : 2;
    long long piece = XE_PIECE_BYTES / (M * 2 * p.pl);
    if (p.packs) piece = lowest(piece, XE_PACK_BYTES / (K * 2 * p.pl));
    piece = piece / XT * XT;
    if (piece < XT) piece = XT;
    p.piece = lowest(piece, p.tiles * XT);
    p.ldw = p.packs ? p.piece * p.pl : V;
    // dx has few output tiles for its long reduction, which is split: into as many parts as take the least time by the rounds that
    // they need and the traffic of their sums (4.6 TB/s), with tiles of either height; eight stages at least a part.
    // (2048 rows, 1024 features: 32 tiles -> 8 parts.)
    const long long blocks = p.piece / cb;
    double best = 0.0;
    p.splits = 0;
    for (int low = M <= 128 ? 1 : 0; low < 2; ++low) {
        const long long out = ((M + (low ? 63 : 255)) / (low ? 64 : 256)) * ((K + XT - 1) / XT);
        for (int n = 1; n <= 64 && n * 8 <= (blocks < 8 ? 8 : blocks); ++n) {
            const double t = (double)((out * n + 255) / 256) / n * (double)blocks * (low ? few : many) + (double)n * M * K * 8 / 4.6e12;
            if (p.splits == 0 || t < best) {
                best = t;
                p.splits = n;
                p.small_dx = low != 0;
            }
        }
    }
    p.ldk = up(K, 4);
    return p;
}

struct Carver {
    char* base;
    long long used = 0;
    explicit Carver(void* p) : base(static_cast<char*>(p)) {}
    template <typename T>
    T* take(long long n) {
        T* r = reinterpret_cast<T*>(base + used);
        used += up(n * (long long)sizeof(T), 256);
        return r;
    }
};

// The packed operands, where the backward pass takes them over: x, and w if its packed classes are one piece.
struct Packed {
    short *x, *w;
    long long bytes;
    Packed(const Plan& p, void* base) {
        Carver c(base);
        x = c.take<short>(p.M * p.ldx);
        w = p.packs && p.piece >= p.V ? c.take<short>(p.K * p.ldw) : nullptr;
        bytes = c.used;
    }
};

struct FwdBuffers {
    short *x, *w;
    float *tsum, *beaten, *hit, *partial;
    long long bytes;
    FwdBuffers(const Plan& p, void* ws) {
        Carver c(ws);
        x = c.take<short>(p.M * p.ldx);
        w = c.take<short>(p.packs ? p.K * p.ldw : 0);
        tsum = c.take<float>(p.M * p.tiles);
        beaten = c.take<float>(p.M);
        hit = c.take<float>(p.M);
        partial = c.take<float>(2 * XE_AMAX);
        bytes = c.used;
    }
};

struct BwdBuffers {
    short *x, *w, *dz;
    void* e;
    float *slab, *rowg, *scale, *dbp;
    BwdBuffers(const Plan& p, void* ws) {
        Carver c(ws);
        x = c.take<short>(p.M * p.ldx);
        w = c.take<short>(p.packs ? p.K * p.ldw : 0);
        dz = c.take<short>(p.M * p.piece * p.pl);
        e = c.take<char>(p.M * p.piece * p.esize);
        slab = c.take<float>(p.splits * p.M * p.ldk);
        rowg = c.take<float>(p.M);
        scale = c.take<float>(1);
        dbp = c.take<float>((p.M + 15) / 16 * p.piece);
        bytes = c.used;
    }
    long long bytes;
};

// One workgroup a compute unit: the stages take most of its LDS.
unsigned grid_for(long long items) { return (unsigned)lowest(items, 256); }

template <typename F>
int with_lds(F* kernel, int bytes) {
    return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

#define XE_TRY(call)              \
    do {                          \
        const int rc__ = (call);  \
        if (rc__ != 0) return rc__; \
    } while (0)

int pack(const Plan& p, const void* src, long long ld_src, long long rows, long long cols, short* dst, long long ld,
         const long long* labels, long long ignore, const float* partial, unsigned* amax, hipStream_t stream) {
    const long long total = rows * (ld / p.pl / 8);
    const unsigned grid = (unsigned)lowest((total + 255) / 256, 8192);
    if (p.type == 1)
        hipLaunchKernelGGL((xe_pack_kernel<__hip_bfloat16, 1>), dim3(grid), dim3(256), 0, stream,
                           static_cast<const __hip_bfloat16*>(src), ld_src, rows, cols, dst, ld, labels, ignore, partial, amax);
    else if (p.pl == 1)
        hipLaunchKernelGGL((xe_pack_kernel<float, 1>), dim3(grid), dim3(256), 0, stream, static_cast<const float*>(src), ld_src, rows,
                           cols, dst, ld, labels, ignore, partial, amax);
    else
        hipLaunchKernelGGL((xe_pack_kernel<float, 2>), dim3(grid), dim3(256), 0, stream, static_cast<const float*>(src), ld_src, rows,
                           cols, dst, ld, labels, ignore, partial, amax);
    DTF_CHECK_LAUNCH();
    return 0;
}

// w of the classes [v0, v0 + cols): packed into `buf`, or in place.  *left: bytes from there to the end of the operand.
int piece_of_w(const Plan& p, const void* W, long long v0, long long cols, short* buf, unsigned* amax, hipStream_t stream,
               const short** w, long long* left) {
    const char* src = static_cast<const char*>(W) + v0 * (p.type ? 2 : 4);
    if (!p.packs) {
        *w = reinterpret_cast<const short*>(src);
        *left = (p.K * p.V - v0) * 2;
        return 0;
    }
    *w = buf;
    *left = p.K * p.ldw * 2;
    return pack(p, src, p.V, p.K, cols, buf, p.ldw, nullptr, 0, nullptr, amax + 1, stream);
}

// What a forward pass leaves for the backward pass, in one block of floats.
struct State {
    float *lse, *zlab, *totals, *tmax;
    unsigned* amax;
    State(float* base, long long M)
        : lse(base), zlab(base + M), totals(base + 2 * M), tmax(base + 2 * M + 6), amax(reinterpret_cast<unsigned*>(base + 2 * M + 4)) {}
};

struct Call {
    const void *X, *W, *B;
    const long long* labels;
    long long ignore;
    hipStream_t stream;
};

template <int PL, int LN, int WL, int WR>
int launch_logits(const Plan& p, const Call& c, const short* x, const short* w, long long left, long long v0, long long vend,
                  const unsigned* amax, float* tmax, float* tsum, float* zlab, float* beaten, void* E, long long lde, long long e0,
                  long long e_tiles) {
    typedef Gemm<typename HalfOf<PL>::type, PL, LN, XT, WL, WR, false, true, LN == 64 ? 3 : 2> G;
    auto* kernel = &xe_logits_kernel<PL, LN, WL, WR>;
    constexpr int lds = G::LDS_BYTES + (XT + 2 * WR * LN + 2 * LN) * 4;
    XE_TRY(with_lds(kernel, lds));
    const long long tiles = ((p.M + LN - 1) / LN) * ((vend - v0 + XT - 1) / XT);
    hipLaunchKernelGGL(kernel, dim3(grid_for(tiles)), dim3(G::THREADS), lds, c.stream, x, p.ldx, w, p.ldw, left, c.B,
                       p.type, c.labels, p.M, p.K, v0, vend, amax, tmax, tsum, zlab, beaten, E, lde, e0, e_tiles);
    DTF_CHECK_LAUNCH();
    return 0;
}

int logits(const Plan& p, const Call& c, const short* x, const short* w, long long left, long long v0, long long vend,
           const unsigned* amax, float* tmax, float* tsum, float* zlab, float* beaten, void* E, long long lde, long long e0,
           long long e_tiles) {
    auto* launch = p.pl == 1 ? (p.small ? &launch_logits<1, 64, 1, 4> : &launch_logits<1, 256, 2, 4>)
                             : (p.small ? &launch_logits<2, 64, 1, 4> : &launch_logits<2, 256, 2, 4>);
    return launch(p, c, x, w, left, v0, vend, amax, tmax, tsum, zlab, beaten, E, lde, e0, e_tiles);
}

template <int PL, int LN, int WL, int WR>
int launch_dx(const Plan& p, const short* dz, const short* w, long long left, long long cols, int first, float* slab, hipStream_t stream) {
    typedef Gemm<typename HalfOf<PL>::type, PL, LN, XT, WL, WR, false, false, LN == 64 ? 3 : 2> G;
    auto* kernel = &xe_dx_kernel<PL, LN, WL, WR>;
    XE_TRY(with_lds(kernel, G::LDS_BYTES));
    const long long tiles = ((p.M + LN - 1) / LN) * ((p.K + XT - 1) / XT);
    const int blocks = (int)((cols + G::CB - 1) / G::CB), splits = (int)lowest(p.splits, blocks);   // (a last piece may be short)
    hipLaunchKernelGGL(kernel, dim3(grid_for(tiles * splits)), dim3(G::THREADS), G::LDS_BYTES, stream, dz, p.piece * PL, w,
                       p.ldw, left, p.M, p.K, blocks, splits, !first, slab, p.ldk);
    DTF_CHECK_LAUNCH();
    return 0;
}

template <int PL, int OUT_BF16, int LN, int WL, int WR>
int launch_dw_tiles(const Plan& p, const short* x, const short* dz, long long dz_left, long long v0, long long cols,
                    const unsigned* amax, const float* scale, void* DW, hipStream_t stream) {
    typedef Gemm<typename HalfOf<PL>::type, PL, LN, XT, WL, WR, true, true, LN == 64 ? 3 : 2> G;
    auto* kernel = &xe_dw_kernel<PL, OUT_BF16, LN, WL, WR>;
    XE_TRY(with_lds(kernel, G::LDS_BYTES));
    const long long tiles = ((p.K + LN - 1) / LN) * ((cols + XT - 1) / XT);
    hipLaunchKernelGGL(kernel, dim3(grid_for(tiles)), dim3(G::THREADS), G::LDS_BYTES, stream, x, p.ldx, dz, p.piece * PL, dz_left,
                       p.M, p.K, cols, amax, scale, DW, p.V, v0);
    DTF_CHECK_LAUNCH();
    return 0;
}

// dw's tiles of 256 x 256 go out in rounds of 256 workgroups.  What a last round holds goes to tiles of 64 rows if it is at most
// half full: four times as many, a third of a round's time (50021 classes, 1024 features, 2048 rows: 241 + 39 us, and 297 us with
// a last round of 16 tiles.  The logits gained nothing from it: 277 + 27 us for 301.)
long long whole_columns(long long rows, long long cols) {
    const long long nrow = (rows + 255) / 256, ncol = (cols + XT - 1) / XT;
    if (rows <= 128) return 0;                                  // (64-row tiles waste less)
    const long long whole = nrow * ncol / 256 * 256 / nrow;
    return (ncol - whole) * nrow <= 128 ? whole : ncol;
}

template <int PL, int OUT_BF16>
int launch_dw(const Plan& p, const short* x, const short* dz, long long v0, long long cols, const unsigned* amax, const float* scale,
              void* DW, hipStream_t stream) {
    const long long done = lowest(whole_columns(p.K, cols) * XT, cols), left = p.M * p.piece * PL * 2;
    if (done > 0) XE_TRY((launch_dw_tiles<PL, OUT_BF16, 256, 2, 4>(p, x, dz, left, v0, done, amax, scale, DW, stream)));
    if (done < cols)
        XE_TRY((launch_dw_tiles<PL, OUT_BF16, 64, 1, 4>(p, x, dz + done * PL, left - done * PL * 2, v0 + done, cols - done, amax, scale, DW,
                                                        stream)));
    return 0;
}

int forward(const Plan& p, const Call& c, float* loss, const State& st, void* kept, long long kept_cols, void* packed, int reduction,
            float* reduced, void* ws) {
    FwdBuffers b(p, ws);
    if (packed) {
        const Packed to(p, packed);
        b.x = to.x;
        if (to.w) b.w = to.w;
    }
    float *tmax = st.tmax, *zlab = st.zlab;
    unsigned* amax = st.amax;
    if (p.pl == 2) {
        hipLaunchKernelGGL(xe_amax_kernel, dim3(XE_AMAX), dim3(256), 0, c.stream, static_cast<const float*>(c.X), p.M, p.K, c.labels,
                           c.ignore, static_cast<const float*>(c.W), p.K * p.V, b.partial);
        DTF_CHECK_LAUNCH();
    }
    // x in place where the tiles can read it so and no e of an ignored row is kept: such a row's statistics are never looked at
    const bool direct = p.type == 1 && p.K % 64 == 0 && (reinterpret_cast<uintptr_t>(c.X) & 15) == 0 && !kept && !packed;
    const short* x = direct ? static_cast<const short*>(c.X) : b.x;
    if (!direct) XE_TRY(pack(p, c.X, p.K, p.M, p.K, b.x, p.ldx, c.labels, c.ignore, b.partial, amax, c.stream));
    const long long step = p.packs ? p.piece : p.V;             // where w is read in place the whole vocabulary is one launch
    for (long long v0 = 0; v0 < p.V; v0 += step) {
        const long long cols = lowest(step, p.V - v0);
        const short* w;
        long long left;
        XE_TRY(piece_of_w(p, c.W, v0, cols, b.w, amax, c.stream, &w, &left));
        const long long e_tiles = kept_cols > v0 ? (kept_cols - v0) / XT : 0;
        XE_TRY(logits(p, c, x, w, left, v0, v0 + cols, amax, tmax, b.tsum, zlab, b.beaten, kept, kept_cols, v0, e_tiles));
    }
    int rows = 16;
    while (rows > 1 && rows / 2 >= p.M) rows /= 2;
    hipLaunchKernelGGL(xe_merge_kernel, dim3((unsigned)((p.M + rows - 1) / rows)), dim3(256), 0, c.stream, tmax, b.tsum, p.tiles,
                       c.labels, p.M, p.V, c.ignore, rows, zlab, b.beaten, st.lse, loss, b.hit);
    DTF_CHECK_LAUNCH();
    if (reduction) {
        hipLaunchKernelGGL(xe_total_kernel, dim3(1), dim3(1024), 0, c.stream, loss, b.hit, c.labels, p.M, c.ignore, st.totals, reduction,
                           reduced);
        DTF_CHECK_LAUNCH();
    }
    return 0;
}

int backward(const Plan& p, const Call& c, const State& st, const void* kept, long long kept_cols, void* packed, int mean,
             const float* dloss, int stride, void* DX, void* DW, void* DB, void* ws) {
    BwdBuffers b(p, ws);
    bool have_w = false;
    if (packed) {
        const Packed from(p, packed);
        b.x = from.x;
        if (from.w) b.w = from.w, have_w = true;
    }
    float *tmax = st.tmax, *zlab = st.zlab, *lse = st.lse, *totals = st.totals;
    unsigned* amax = st.amax;
    hipLaunchKernelGGL(xe_weights_kernel, dim3(1), dim3(1024), 0, c.stream, dloss, stride, totals, mean, c.labels, p.M, p.V, c.ignore,
                       lse, zlab, b.rowg, b.scale);
    DTF_CHECK_LAUNCH();
    if (!packed && (DW || kept_cols < p.V)) XE_TRY(pack(p, c.X, p.K, p.M, p.K, b.x, p.ldx, c.labels, c.ignore, nullptr, amax, c.stream));
    const int dz_rows = (p.M + 63) / 64 * ((p.piece + XT - 1) / XT) < 1024 ? 16 : 64;
    const long long rowblocks = (p.M + dz_rows - 1) / dz_rows;
    for (long long v0 = 0; v0 < p.V; v0 += p.piece) {
        const long long cols = lowest(p.piece, p.V - v0), ct = (cols + XT - 1) / XT;
        const short* w = nullptr;
        long long left = 0;
        const long long have = kept_cols > v0 ? lowest((kept_cols - v0) / XT, ct) : 0;      // the piece's tiles whose e was kept
        if (have_w)
            w = b.w, left = p.K * p.ldw * 2;
        else if (DX || have < ct)
            XE_TRY(piece_of_w(p, c.W, v0, cols, b.w, amax, c.stream, &w, &left));
        float* dbp = DB ? b.dbp : nullptr;
        for (int part = 0; part < 2; ++part) {
            const long long t0 = part ? have : 0, t1 = part ? ct : have, at = v0 + t0 * XT;
            if (t1 == t0) continue;
            const void* e = kept;
            long long lde = kept_cols, e0 = at;
            if (part) {      // not kept: computed again
                e = b.e, lde = p.piece, e0 = t0 * XT;
                XE_TRY(logits(p, c, b.x, w + t0 * XT * p.pl, left - t0 * XT * p.pl * 2, at, v0 + cols, amax, nullptr, nullptr, nullptr,
                              nullptr, b.e, p.piece, e0, t1 - t0));
            }
            short* dz = b.dz + t0 * XT * p.pl;
            float* sums = dbp ? dbp + t0 * XT : nullptr;
            const dim3 grid((unsigned)(t1 - t0), (unsigned)rowblocks);
            auto* kernel = p.pl == 1 ? (dz_rows == 16 ? &xe_dz_kernel<1, 16> : &xe_dz_kernel<1, 64>)
                                     : (dz_rows == 16 ? &xe_dz_kernel<2, 16> : &xe_dz_kernel<2, 64>);
            hipLaunchKernelGGL(kernel, grid, dim3(256), 0, c.stream, e, lde, e0, tmax, lse, zlab, b.rowg, c.labels, p.M, at, dz,
                               p.piece * p.pl, sums);
            DTF_CHECK_LAUNCH();
        }
        if (DX) {
            const int first = v0 == 0;
            if (p.pl == 1)
                XE_TRY(p.small_dx ? (launch_dx<1, 64, 1, 4>(p, b.dz, w, left, cols, first, b.slab, c.stream))
                               : (launch_dx<1, 256, 2, 4>(p, b.dz, w, left, cols, first, b.slab, c.stream)));
            else
                XE_TRY(p.small_dx ? (launch_dx<2, 64, 1, 4>(p, b.dz, w, left, cols, first, b.slab, c.stream))
                               : (launch_dx<2, 256, 2, 4>(p, b.dz, w, left, cols, first, b.slab, c.stream)));
        }
        if (DW) {
            if (p.pl == 2) XE_TRY((launch_dw<2, 0>(p, b.x, b.dz, v0, cols, amax, b.scale, DW, c.stream)));
            else if (p.type == 1) XE_TRY((launch_dw<1, 1>(p, b.x, b.dz, v0, cols, amax, b.scale, DW, c.stream)));
            else XE_TRY((launch_dw<1, 0>(p, b.x, b.dz, v0, cols, amax, b.scale, DW, c.stream)));
        }
        if (DB) {
            const dim3 grid((unsigned)((cols + 31) / 32));
            if (p.type == 1)
                hipLaunchKernelGGL(xe_db_kernel<__hip_bfloat16>, grid, dim3(256), 0, c.stream, b.dbp, rowblocks, p.piece, cols, b.scale,
                                   static_cast<__hip_bfloat16*>(DB) + v0);
            else
                hipLaunchKernelGGL(xe_db_kernel<float>, grid, dim3(256), 0, c.stream, b.dbp, rowblocks, p.piece, cols, b.scale,
                                   static_cast<float*>(DB) + v0);
            DTF_CHECK_LAUNCH();
        }
    }
    if (DX) {
        const dim3 grid((unsigned)lowest((p.M * p.K + 255) / 256, 16384));
        if (p.pl == 2)
            hipLaunchKernelGGL((xe_dx_finish_kernel<float, 2>), grid, dim3(256), 0, c.stream, b.slab, p.splits, p.M, p.K, p.ldk, amax,
                               b.scale, static_cast<float*>(DX));
        else if (p.type == 1)
            hipLaunchKernelGGL((xe_dx_finish_kernel<__hip_bfloat16, 1>), grid, dim3(256), 0, c.stream, b.slab, p.splits, p.M, p.K, p.ldk,
                               amax, b.scale, static_cast<__hip_bfloat16*>(DX));
        else
            hipLaunchKernelGGL((xe_dx_finish_kernel<float, 1>), grid, dim3(256), 0, c.stream, b.slab, p.splits, p.M, p.K, p.ldk, amax,
                               b.scale, static_cast<float*>(DX));
        DTF_CHECK_LAUNCH();
    }
    return 0;
}

// The largest sizes: 1048560 rows, 1048576 features, 4194304 classes (32-bit offsets within a tile; rows in blocks of 16 as
// the second grid dimension).
bool sizes_ok(long long M, long long K, long long V, int type) {
    return M > 0 && K > 0 && V > 0 && (type == 0 || type == 1) && M <= 65535ll * 16 && K <= (1ll << 20) && V <= (1ll << 22);
}

}  // namespace

DTF_API long long dtf_linear_xent_fwd_workspace_bytes(const void* W, long long M, long long K, long long V, int type, int bf16) {
    return sizes_ok(M, K, V, type) ? FwdBuffers(make_plan(W, M, K, V, type, bf16), nullptr).bytes : -1;
}
DTF_API long long dtf_linear_xent_bwd_workspace_bytes(const void* W, long long M, long long K, long long V, int type, int bf16) {
    return sizes_ok(M, K, V, type) ? BwdBuffers(make_plan(W, M, K, V, type, bf16), nullptr).bytes : -1;
}

// bytes of the packed operands that a forward call may leave for the backward call
DTF_API long long dtf_linear_xent_packed_bytes(const void* W, long long M, long long K, long long V, int type, int bf16) {
    return sizes_ok(M, K, V, type) ? Packed(make_plan(W, M, K, V, type, bf16), nullptr).bytes : -1;
}

// floats of the state between the two passes
DTF_API long long dtf_linear_xent_state_floats(long long M, long long V) { return 2 * M + 6 + (V + XT - 1) / XT * M; }

// type: 0 fp32, 1 bf16 (x, w, b alike; b may be null).  bf16 != 0: fp32 operands rounded to bf16 for the products.
// loss: M floats.  state: [2 M, 2 M + 4) holds the sum of the losses, the rows whose label has the largest logit, the counted
// rows and the mean, if reduction is not 0; reduced (may be null): the mean (reduction 1) or the sum (2).  kept (may be null):
// [M, kept_cols] fp32 - bf16 where the products take bf16 -, kept_cols a multiple of 256.  packed (may be null): as above.
DTF_API int dtf_linear_xent_fwd(const void* X, const void* W, const void* B, const long long* labels, long long M, long long K,
                                long long V, int type, int bf16, long long ignore, float* loss, float* state, void* kept,
                                long long kept_cols, void* packed, int reduction, float* reduced, void* workspace,
                                hipStream_t stream) {
    if (!sizes_ok(M, K, V, type) || kept_cols % XT) return -1;
    const Call c = {X, W, B, labels, ignore, stream};
    return forward(make_plan(W, M, K, V, type, bf16), c, loss, State(state, M), kept, kept ? kept_cols : 0, packed, reduction, reduced,
                   workspace);
}

// dloss: the loss's gradient, one float for all rows (stride 0) or one a row (stride 1); mean != 0: divided by the counted
// rows (the forward pass had a reduction).  DX, DW, DB may each be null.
DTF_API int dtf_linear_xent_bwd(const void* X, const void* W, const void* B, const long long* labels, long long M, long long K,
                                long long V, int type, int bf16, long long ignore, float* state, const void* kept, long long kept_cols,
                                void* packed, int mean, const float* dloss, int dloss_stride, void* DX, void* DW, void* DB,
                                void* workspace, hipStream_t stream) {
    if (!sizes_ok(M, K, V, type) || kept_cols % XT) return -1;
    const Call c = {X, W, B, labels, ignore, stream};
    return backward(make_plan(W, M, K, V, type, bf16), c, State(state, M), kept, kept ? kept_cols : 0, packed, mean, dloss,
                    dloss_stride, DX, DW, DB, workspace);
}
