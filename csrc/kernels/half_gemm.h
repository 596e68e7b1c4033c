// Matrix products of 16-bit operands on the gfx950 matrix cores, as a main loop for kernels that bring their own epilogue:
//
//   acc[l, r] = sum_k L[l, k] R[r, k]          (fp32 accumulation)
//
// Each operand lies in memory either along k (rows l, k contiguous: "RC") or across it (rows k, l contiguous: "RS"), so no
// operand is ever transposed in memory: RS tiles are read from LDS with the transposing 64-bit read.
//
// PL = 2 serves fp32 operands, kept as two fp16 limbs x = hi + lo (22 bits; what is lost is below fp32's own rounding of a
// product): 32 values of a row are stored as 32 hi limbs, then 32 lo limbs, so that a tile of 2-limb values has the shape of
// a tile of 16-bit values with half as many k.  Three limb products make one product: hi hi, hi lo, lo hi.
//
// A workgroup of WL x WR waves computes LN x RN tiles one after another; a wave holds (LN / WL) x (RN / WR) in accumulators.  A stage is
// 64 halves of the reduction an operand row: 128 bytes a row, loaded straight into LDS (16 bytes a lane); while one stage
// is multiplied the next one arrives in the other buffer, one barrier a stage.
//
// What bounds it (8192 x 8192 x 2048, bf16): power and the loads into LDS.  The matrix pipes are busy 58 % of the cycles at a
// clock that the load drives down to 1.9 GHz; without the loads in the loop the same instructions reach 1400 TFLOP/s, without
// LDS reads 1200, without both 1550.  At it for a second, logits / dx / dw reach 1250 / 1250 / 1220 TFLOP/s and two limbs 450 / 450 /
// 440; over the vocabularies below, with their longer strides, 1040 - 1140.  Measured and dropped: a ring of four half stages (64
// bytes a row: 1070), four waves of 128 x 128 (8 % slower), padded rows (no effect: the strides do not meet in one channel),
// raised priority for the waves that multiply (no effect).
//
// LDS layouts.  RC: row of 128 bytes = 8 chunks of 16; chunk c of row i lies at c ^ ((i >> 1) & 7): LDS delivers 256 bytes a
// cycle, 16 lanes of a fragment read, whose 16 rows at one c are then on 16 different chunks of two rows' width (with i & 7
// every second chunk would be hit twice: measured as one conflict cycle for each useful one).  RS: row k of N * PL halves in
// granules of 32 bytes; granule q of row k lies at q ^ 2 (k & 3): a transposing read takes 4 rows x 2 granules at once, which are
// then 8 distinct ones of 256 bytes.
// The direct load writes LDS linearly, so the permutation is applied to the addresses it loads from.
#pragma once
#include "common.h"

namespace hgemm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

template <typename H>
struct Mma;
template <>
struct Mma<__bf16> {
    static __device__ __forceinline__ f32x16 run(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mma<_Float16> {
    static __device__ __forceinline__ f32x16 run(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

typedef __attribute__((address_space(3))) char lds_char;

// vectors at any element's address: global memory takes 16-byte accesses that are aligned to the element only
typedef s16x8 s16x8_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(unsigned, v);
}

// 32 accumulator columns of a row, times `g`, as bf16 at `out` (of this lane: 8 (lane >> 5) behind the row's first): a lane holds
// 4 neighbours of every 8, its partner 32 lanes on the other 4; after the exchange each holds 8 of every 16 and writes 16 bytes.
__device__ __forceinline__ void store_bf16_16(const f32x16& acc, float g, short* out, bool live) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        unsigned a0 = pack_bf16(acc[h * 8 + 0] * g, acc[h * 8 + 1] * g), a1 = pack_bf16(acc[h * 8 + 2] * g, acc[h * 8 + 3] * g);
        unsigned b0 = pack_bf16(acc[h * 8 + 4] * g, acc[h * 8 + 5] * g), b1 = pack_bf16(acc[h * 8 + 6] * g, acc[h * 8 + 7] * g);
        const auto p = __builtin_amdgcn_permlane32_swap(a0, b0, false, false), q = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        const u32x4 v = {p[0], q[0], p[1], q[1]};
        if (live) *reinterpret_cast<s16x8_any*>(out + h * 16) = __builtin_bit_cast(s16x8, v);
    }
}

// Transposing read: of every 16 lanes, lane i receives value i of 4 rows, from the 4 lanes that address each row (4 values a lane).
// __restrict__ gives the read a scope of its own; without one the compiler waits for all loads into LDS that are in flight
// before it, also for those into the other buffer.  (The waits that are needed are written out in the loop.)
__device__ __forceinline__ s16x4 read_tr(const lds_char* __restrict__ p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}

// One operand's tile in memory: `base` is its first element, `left` the bytes from there to the end of the operand (what lies
// behind reads as zero), `ld` the bytes of a row.
struct Tile {
    const char* base;
    long long left, ld;
};

template <typename H, int PL, int LN, int RN, int WL, int WR, bool L_RS, bool R_RS, int STAGES = 2>
struct Gemm {
    static constexpr int THREADS = 64 * WL * WR, WAVES = WL * WR;
    static constexpr int CB = 64 / PL;                       // values of the reduction a stage
    static constexpr int TL = LN / WL / 32, TR = RN / WR / 32;
    static constexpr int L_BYTES = LN * 128, R_BYTES = RN * 128, STAGE = L_BYTES + R_BYTES;
    static constexpr int LDS_BYTES = STAGES * STAGE;
    static constexpr int LOADS = (LN + RN) / 8 / WAVES;      // a wave and stage, 1 KB each
    static constexpr int KS = CB / 16;                       // MFMA steps a stage and limb product
    static_assert(LN % (32 * WL) == 0 && RN % (32 * WR) == 0 && (LN / 8) % WAVES == 0 && (RN / 8) % WAVES == 0, "tile");
    static_assert((!L_RS || LN == 256 || LN == 64) && (!R_RS || RN == 256), "the RS layout's banks are worked out for these rows");

    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const char* base, long long left) {
        const long long n = left < 0 ? 0 : left > 0xffffffffll ? 0xffffffffll : left;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, (int)(unsigned)n, 0x00020000);
    }

    // granule permutation of row k of an RS tile of N values: 4 rows by 2 granules on 8 granules of 256 bytes; rows of 128 bytes
    // (64 values, one limb) lie two to 256 bytes
    template <int N>
    static __device__ __forceinline__ int rs_swap(int k) {
        return N * PL == 64 ? k & 2 : 2 * (k & 3);
    }

    // An operand's memory from stage `blk` on.
    template <bool RS>
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t from(const Tile& t, int blk) {
        const long long skip = RS ? (long long)blk * CB * t.ld : (long long)blk * 128;
        return resource(t.base + skip, t.left - skip);
    }

    // LDS <- a stage of one operand, the first of `rs`
    template <int N, bool RS>
    static __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, unsigned ld, lds_char* dst) {
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));                       // the offsets are worked out anew each stage: kept, they would spill
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        constexpr int LOADS = N / 8 / WAVES;                 // 1 KB each
        if (!RS) {
            static_assert(LOADS % 2 == 0, "the chunk permutation of a load depends on its parity");
            const unsigned row0 = (unsigned)(wave * LOADS * 8 + (lane >> 3)) * ld;
            const unsigned chunk = (unsigned)((lane & 7) ^ (lane >> 4)) * 16;
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(dst + (wave * LOADS + i) * 1024), 16,
                                                         (int)(row0 + 8 * i * ld + (i & 1 ? chunk ^ 64 : chunk)), 0, 0, 0);
        } else {
            constexpr int SLOTS = N * PL / 8;                // 16-byte chunks a row: 8 to 64
            constexpr int ROWS = 64 / SLOTS;                 // rows a load: 8 to 1
            static_assert(LOADS * ROWS % 4 == 0, "a wave's first row is a multiple of 4");
            const unsigned row0 = (unsigned)(wave * LOADS * ROWS + lane / SLOTS) * ld;
            const unsigned chunk = (unsigned)((lane % SLOTS) ^ (2 * rs_swap<N>(lane / SLOTS))) * 16;
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(dst + (wave * LOADS + i) * 1024), 16,
                                                         (int)(row0 + ROWS * i * ld + (chunk ^ (32 * rs_swap<N>(ROWS * i)))), 0, 0, 0);
        }
    }

    // Fragment of 32 values x 16 steps of k: lane holds value lane & 31, steps 8 (lane >> 5) ... + 7.
    template <bool RS, int N>
    static __device__ __forceinline__ s16x8 frag(const lds_char* src, int tile32, int plane, int kk) {
        const int lane = threadIdx.x & 63;
        if (!RS) {
            const int chunk = plane * 4 + kk * 2 + (lane >> 5);
            const lds_char* p = src + (tile32 * 32 + (lane & 31)) * 128 + (chunk ^ ((lane >> 1) & 7)) * 16;
            return *(const __attribute__((address_space(3))) s16x8*)p;
        }
        constexpr int ROW = N * PL * 2;
        const int granule = tile32 * 2 * PL + plane * 2 + ((lane >> 4) & 1);
        const int row = kk * 16 + (lane >> 5) * 8 + ((lane >> 2) & 3);
        const lds_char* p = src + row * ROW + ((granule ^ rs_swap<N>((lane >> 2) & 3)) * 32) + (lane & 3) * 8;
        const s16x4 lo = read_tr(p), hi = read_tr(p + 4 * ROW);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }

    struct Frags {
        s16x8 l[PL][TL], r[PL][TR];
    };

    static __device__ __forceinline__ void load_stage(const Tile& tl, const Tile& tr, int blk, lds_char* dst) {
        load<LN, L_RS>(from<L_RS>(tl, blk), (unsigned)tl.ld, dst);
        load<RN, R_RS>(from<R_RS>(tr, blk), (unsigned)tr.ld, dst + L_BYTES);
    }

    static __device__ __forceinline__ void fetch(const lds_char* src, int kk, int wl, int wr, Frags& f) {
#pragma unroll
        for (int p = 0; p < PL; ++p) {
#pragma unroll
            for (int b = 0; b < TR; ++b) f.r[p][b] = frag<R_RS, RN>(src + L_BYTES, wr * TR + b, p, kk);
#pragma unroll
            for (int a = 0; a < TL; ++a) f.l[p][a] = frag<L_RS, LN>(src, wl * TL + a, p, kk);
        }
    }

    template <int A0 = 0, int A1 = TL>
    static __device__ __forceinline__ void multiply(const Frags& f, f32x16 (&acc)[TL][TR]) {
#pragma unroll
        for (int a = A0; a < A1; ++a)
#pragma unroll
            for (int b = 0; b < TR; ++b) {
                if (PL == 2) {
                    acc[a][b] = Mma<H>::run(f.r[PL - 1][b], f.l[0][a], acc[a][b]);
                    acc[a][b] = Mma<H>::run(f.r[0][b], f.l[PL - 1][a], acc[a][b]);
                }
                acc[a][b] = Mma<H>::run(f.r[0][b], f.l[0][a], acc[a][b]);
            }
    }

    // This wave's loads into LDS have landed and its reads have returned; then everybody's.
    static __device__ __forceinline__ void meet() {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
    }

    // What a workgroup multiplies now, and what next (`more`): the next tile's first stage is loaded during the last one of this.
    struct Job {
        Tile l, r;
        int blocks;
    };
    // LDS <- stage `blk` of the job, or the next job's first one behind the last; out of bounds (zeros) if there is none, so that no
    // branch stands in the way.
    static __device__ __forceinline__ void load_ahead(const Job& job, const Job& next, bool more, int blk, lds_char* dst) {
        const bool in = blk < job.blocks;
        const Tile l = {in ? job.l.base : next.l.base, in ? job.l.left : more ? next.l.left : 0, in ? job.l.ld : next.l.ld};
        const Tile r = {in ? job.r.base : next.r.base, in ? job.r.left : more ? next.r.left : 0, in ? job.r.ld : next.r.ld};
        load_stage(l, r, in ? blk : 0, dst);
    }

    // Tiles of few rows: so little to multiply that a stage takes as long as its loads' way, so STAGES - 1 stages are on their way at
    // a time.  64 rows against 128 tiles of columns, 4096 features, two stages / three: fp32 156 / 112 us, bf16 60 / 51 us (5.3 TB/s);
    // 512 features: 16.6 / 16.0 and 8.3 / 8.7 us; four stages are no faster than three.  The loads of stages behind the last
    // one are issued all the same, out of bounds, so that the number in flight is a constant.
    static __device__ __forceinline__ void ring(const Job& job, int wl, int wr, lds_char* smem, f32x16 (&acc)[TL][TR]) {
        const Tile none_l = {job.l.base, 0, job.l.ld}, none_r = {job.r.base, 0, job.r.ld};
        auto issue = [&](int blk, int at) {
            if (blk < job.blocks) load_stage(job.l, job.r, blk, smem + at * STAGE);
            else load_stage(none_l, none_r, 0, smem + at * STAGE);
        };
        meet();                                              // nobody reads a buffer of an earlier job any more
#pragma unroll
        for (int k = 0; k < STAGES - 1; ++k) issue(k, k);
        int now = 0, ahead = STAGES - 1;
        for (int blk = 0; blk < job.blocks; ++blk) {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * LOADS) : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            Frags f[KS];                                     // one wave a SIMD: all reads of a stage first, not step by step
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) fetch(smem + now * STAGE, kk, wl, wr, f[kk]);
            issue(blk + STAGES - 1, ahead);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) multiply(f[kk], acc);
            __builtin_amdgcn_sched_barrier(0);
            now = now + 1 == STAGES ? 0 : now + 1;
            ahead = ahead + 1 == STAGES ? 0 : ahead + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // nothing is on its way into LDS when the workgroup ends
    }

    // Fragments a step ahead (8192 x 8192 x 2048: 1128 TFLOP/s where both operands are RC, against 1066 without; the others
    // within 2 %).  Two limbs' fragments do not fit the registers twice, so they are read step by step (1230 against 1148).
    static constexpr bool AHEAD = PL == 1 && STAGES == 2;

    // Where a stage's loads are issued.  One limb: at the meeting, as early as the buffer is free (2048 x 1024 x 50021, the whole
    // training step: 831 us; behind a stage's first matrix instructions 866 us).  Two limbs, with three times as many matrix
    // instructions a byte: behind the first row of them, so that not all eight waves stand in the queue of the loads at once
    // (4096 x 1024 x 32000: 2275 us; at the meeting 2300 us).  Dealt over several steps they are no faster.

    // `buffer`: where the job's first stage is (or goes, unless `primed`); both are carried from job to job.  blocks >= 1.
    static __device__ __forceinline__ void run(const Job& job, const Job& next, bool more, bool& primed, int& buffer, lds_char* smem,
                                               f32x16 (&acc)[TL][TR]) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wl = wave / WR, wr = wave % WR;
#pragma unroll
        for (int a = 0; a < TL; ++a)
#pragma unroll
            for (int b = 0; b < TR; ++b) acc[a][b] = f32x16{};
        if (STAGES > 2) {
            ring(job, wl, wr, smem, acc);
            return;
        }
        lds_char* cur = smem + buffer * STAGE;
        lds_char* oth = smem + (buffer ^ 1) * STAGE;
        static_assert(!AHEAD || KS % 2 == 0, "a stage's first fragments are those of f[0]");
        Frags f[AHEAD ? 2 : 1];
        if (!primed) load_stage(job.l, job.r, 0, cur);
        meet();
        if (AHEAD) {
            load_ahead(job, next, more, 1, oth);
            fetch(cur, 0, wl, wr, f[0]);
        }
        for (int blk = 0; blk < job.blocks; ++blk) {
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                if (AHEAD) {
                    // the meeting between two stages lies before the last multiplications of the first: they cover it and the reads
                    if (kk + 1 < KS) {
                        fetch(cur, kk + 1, wl, wr, f[(kk + 1) & 1]);
                    } else if (blk + 1 < job.blocks) {
                        meet();
                        load_ahead(job, next, more, blk + 2, cur);
                        fetch(oth, 0, wl, wr, f[0]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    multiply(f[kk & 1], acc);
                    __builtin_amdgcn_sched_barrier(0);
                } else {
                    fetch(cur, kk, wl, wr, f[0]);
                    multiply<0, 1>(f[0], acc);
                    if (kk == 0) {
                        __builtin_amdgcn_sched_barrier(0);
                        load_ahead(job, next, more, blk + 1, oth);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    multiply<1, TL>(f[0], acc);
                }
            }
            if (!AHEAD && blk + 1 < job.blocks) meet();
            lds_char* const t = cur;
            cur = oth;
            oth = t;
        }
        if (!more) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing is on its way into LDS when the workgroup ends
        primed = more;
        buffer ^= job.blocks & 1;
    }
};

// Work items of a launch, dealt to its workgroups: those go round the 8 XCDs one after another, so each XCD gets a contiguous run
// of items and its workgroups take turns in it.
struct Deal {
    long long first, end;
    int stride;
    __device__ __forceinline__ Deal(long long count) {
        const long long x = blockIdx.x & 7, base = count >> 3, extra = count & 7;
        const long long start = x * base + (x < extra ? x : extra);
        first = start + (blockIdx.x >> 3);
        end = start + base + (x < extra ? 1 : 0);
        stride = (int)((gridDim.x + 7 - x) >> 3);
    }
};

// Tile `t` of nrow x ncol: down 8 rows of tiles before the next column, so that the operands of neighbours meet in the L2.
__device__ __forceinline__ void tile_at(long long t, long long nrow, long long ncol, long long& row, long long& col) {
    const long long group = t / (8 * ncol), first = group * 8;
    const long long rows = nrow - first < 8 ? nrow - first : 8;
    const long long in = t - group * 8 * ncol;
    row = first + in % rows;
    col = in / rows;
}

}  // namespace hgemm
