// Tiles of 16-bit matrix products on v_mfma_f32_16x16x32_{bf16,f16}, fed from LDS that global_load_lds fills.
//
//   acc[m][n] += sum_k A(m, k) B(n, k)
//
// Each operand is stored in one of two ways:
//   rows     [m][k], k contiguous: a fragment is one ds_read_b128 of 8 consecutive k
//   columns  [k][m], m contiguous: a fragment is two ds_read_b64_tr_b16 (the hardware's 4 x 16 transposition)
// One K step is 32 wide.  A workgroup holds STAGES steps in LDS: later steps are requested while step s is multiplied,
// one barrier a step, and the waits count outstanding requests (vmcnt) instead of draining them.
//
// M rows are permuted inside blocks of 64 so that a lane's 16 accumulators of a block are 16 CONSECUTIVE m of one n:
// matrix row i = 4 p + j of tile t of a block is m = 16 p + 4 t + j (rows) or 16 p + 4 (t ^ (p & 1)) + j (columns).  For "rows" the
// permutation costs nothing (it picks which global row is fetched into which LDS row), for "columns" it is the address of the
// transposed read.  An epilogue then stores 32 bytes of 16-bit results (64 of fp32) per lane and 128 (256) contiguous bytes
// per n.
//
// LDS bank conflicts: 16-byte chunks of a row are XORed with row bits (the fetch applies the same XOR to its source address,
// since global_load_lds writes lanes linearly), so that every 8-lane pass of a b128 read touches each bank once.  A transposed
// read takes 8 bytes per lane from 8 rows x 4 places in a pass of 32 lanes; the XOR of t above puts its even and odd p into
// different halves of the chunks, so it too touches each bank once (without: two passes, SQ_LDS_BANK_CONFLICT half of
// SQ_LDS_IDX_ACTIVE).
#pragma once
#include "common.h"

namespace mfma16 {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void glob_void;

constexpr int BK = 32;          // K of a matrix instruction

// lane and wave of this thread; the lane is counted anew wherever it is needed instead of occupying a register in the main loop
__device__ __forceinline__ int my_lane() { return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); }
__device__ __forceinline__ int my_wave() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

template <bool F16>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c)
{
    if (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 16 bytes per lane from base + off into LDS at dst + 16 lane, counted by vmcnt.  In assembly, because the compiler drains vmcnt
// in front of every transposed read that follows the builtin (it has no alias information for either); it has no
// result register, and every wait for it is written out in Tile::run.
__device__ __forceinline__ void request16(const unsigned char *base, unsigned off, unsigned char *dst)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"((unsigned)(uintptr_t)(lds_void *)dst), "v"(off), "s"(base)
                 : "memory");
}

// the same from 64-bit addresses of the lanes' own
__device__ __forceinline__ void request16_far(const unsigned char *src, unsigned char *dst)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"((unsigned)(uintptr_t)(lds_void *)dst), "v"(src)
                 : "memory");
}
__device__ const u32x4 no_k = {0u, 0u, 0u, 0u};       // what rows hold behind their last k

// An operand as the tile sees it: `base` points at its first element (row 0 or column 0 of the tile, k = first k),
// `ld` in elements.  rows: `lim` = last valid row of the tile's rows (later ones read that row again; their results are
// not used).  columns: `lim` = last valid column chunk (8 columns), likewise.
struct Operand {
    const unsigned short *base;
    int64_t plane;              // elements between the parts of a split fp32 operand
    int64_t ld;
    int lim;
    int k_rows;                 // valid k.  rows: later ones are zero (a multiple of 8); columns: they read the last row again (the
                                // other operand is zero there)
};

// the six products of two three-part operands, small ones first: (part of A, part of B)
__device__ __forceinline__ int seg_a(int s, int nseg) { return nseg == 1 ? 0 : (0x012010 >> (4 * (5 - s))) & 0xf; }
__device__ __forceinline__ int seg_b(int s, int nseg) { return nseg == 1 ? 0 : (0x210100 >> (4 * (5 - s))) & 0xf; }

// SPREAD != 0: of every SPREAD rows (columns) only a block of 64 is fetched, from `first` on
template <bool COLS, int B, bool PERM, int WAVES, int KD, int SPREAD = 0>
struct Loader {
    static constexpr int INSTR = B * KD * 2 / 1024;              // 1 KB requests per step
    static constexpr int PER_WAVE = (INSTR + WAVES - 1) / WAVES; // (the last may be idle for some waves)
    static constexpr int CHUNKS = COLS ? B / 8 : KD / 8;         // 16-byte chunks per LDS row
    static_assert(!COLS || B == 64 || B == 128 || B == 256, "columns operand width");

    __device__ static __forceinline__ int swz(int row)
    {
        if (!COLS) return (row >> 1) & (CHUNKS - 1);
        return B >= 128 ? ((row & 3) | (row & 8)) : (((row >> 1) & 1) | ((row >> 2) & 2));
    }

    unsigned off[PER_WAVE];          // bytes from the step's first element
    const unsigned char *cur;        // the step's first element
    unsigned row_bytes;              // columns: of one k

    __device__ __forceinline__ void init(const Operand &o, int wave, int lane, int first = 0)
    {
        row_bytes = (unsigned)(o.ld * 2);
#pragma unroll
        for (int j = 0; j < PER_WAVE; ++j) {
            const int slot = (j * WAVES + wave) * 64 + lane;
            const int row = slot / CHUNKS, c = (slot % CHUNKS) ^ swz(row);
            if (!COLS) {
                int m = row;
                if (PERM) m = (row & ~63) | (((row & 15) >> 2) << 4) | (((row >> 4) & 3) << 2) | (row & 3);
                if (SPREAD) m = (m >> 6) * SPREAD + first + (m & 63);
                m = m < o.lim ? m : o.lim;
                off[j] = (unsigned)m * row_bytes + c * 16;
            } else {
                const int cc = SPREAD ? (c >> 3) * (SPREAD / 8) + first / 8 + (c & 7) : c;
                off[j] = (unsigned)row * row_bytes + (cc < o.lim ? cc : o.lim) * 16;
            }
        }
    }
    // to step kk of part `part`
    __device__ __forceinline__ void seek(const Operand &o, int part, int64_t kk)
    {
        cur = (const unsigned char *)(o.base + part * o.plane + (COLS ? kk * KD * o.ld : kk * KD));
    }
    __device__ __forceinline__ void next() { cur += COLS ? (int64_t)KD * row_bytes : KD * 2; }

    // request this step into the LDS image `dst`; k_left >= 1: valid k from here on
    __device__ __forceinline__ void issue(unsigned char *dst, int k_left, int wave) const
    {
        if (!COLS && k_left < KD) {
#pragma unroll
            for (int j = 0; j < PER_WAVE; ++j) {
                const int i = j * WAVES + wave, slot = i * 64 + my_lane(), row = slot / CHUNKS, c = (slot % CHUNKS) ^ swz(row);
                if (INSTR % WAVES != 0 && i >= INSTR) continue;
                request16_far(c * 8 < k_left ? cur + off[j] : (const unsigned char *)&no_k, dst + i * 1024);
            }
            return;
        }
        unsigned bo[PER_WAVE];
#pragma unroll
        for (int j = 0; j < PER_WAVE; ++j) bo[j] = off[j];
        if (COLS && k_left < KD) {
#pragma unroll
            for (int j = 0; j < PER_WAVE; ++j) {
                const int row = ((j * WAVES + wave) * 64 + my_lane()) / CHUNKS;
                if (row >= k_left) bo[j] -= (unsigned)(row - (k_left - 1)) * row_bytes;
            }
        }
#pragma unroll
        for (int j = 0; j < PER_WAVE; ++j) {
            const int i = j * WAVES + wave;
            if (INSTR % WAVES != 0 && i >= INSTR) continue;
            request16(cur, bo[j], dst + i * 1024);
        }
    }
};

// fragment of the 16 rows (columns) from 16 tile16 on, k from BK sub on
template <bool COLS, int B, bool PERM, int KD>
__device__ __forceinline__ u32x4 fragment(const unsigned char *img, int tile16, int sub, int lane)
{
    using L = Loader<COLS, B, PERM, 4, KD>;
    if (!COLS) {
        const int row = tile16 * 16 + (lane & 15);
        return *(const u32x4 *)(img + row * (KD * 2) + (((sub * 4 + (lane >> 4)) ^ L::swz(row)) << 4));
    }
    const int g = lane >> 4, q = (lane & 15) >> 2, p = lane & 3, k = sub * BK + 8 * g + q;
    const int blk = tile16 >> 2, t = tile16 & 3;
    const int tp = t ^ (p & 1);
    const int c = (blk * 8 + 2 * p + (tp >> 1)) ^ L::swz(k);
    const unsigned char *a = img + k * (B * 2) + c * 16 + (tp & 1) * 8;
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16 *)a);
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16 *)(a + 4 * (B * 2)));
    const unsigned long long l = __builtin_bit_cast(unsigned long long, lo), h = __builtin_bit_cast(unsigned long long, hi);
    return u32x4{(unsigned)l, (unsigned)(l >> 32), (unsigned)h, (unsigned)(h >> 32)};
}

template <int BM_, int BN_, int WM_, int WN_, bool ACOLS_, bool BCOLS_, bool F16_, int STAGES_ = 3>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;             // waves along m and n
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int KD = BK, STAGES = STAGES_;                          // depth of a step, steps in LDS
    static constexpr bool ACOLS = ACOLS_, BCOLS = BCOLS_, F16 = F16_;
    static constexpr int TM = BM / WM, TN = BN / WN;                         // per wave
    static constexpr int MT = TM / 16, NT = TN / 16;
    static constexpr int A_BYTES = BM * KD * 2, B_BYTES = BN * KD * 2, STAGE = A_BYTES + B_BYTES;
    static constexpr int LDS = STAGES * STAGE;
    static constexpr int OCCUPANCY = (LDS > 80 * 1024 ? 1 : 2) * WAVES / 4;  // waves per SIMD: one or two workgroups per CU
    using LA = Loader<ACOLS, BM, true, WAVES, KD>;
    using LB = Loader<BCOLS, BN, BCOLS, WAVES, KD>;
    static_assert(TM % 64 == 0, "a wave holds whole permuted blocks");
    static_assert(!BCOLS || TN % 64 == 0, "transposed reads go by blocks of 64");

    using Acc = f32x4[MT][NT];
    struct Frags { u32x4 a[MT], b[NT]; };

    __device__ static __forceinline__ void read(Frags &f, const unsigned char *ia, int wm, int wn, int lane)
    {
        const unsigned char *ib = ia + A_BYTES;
#pragma unroll
        for (int n = 0; n < NT; ++n) f.b[n] = fragment<BCOLS, BN, BCOLS, KD>(ib, wn * NT + n, 0, lane);
#pragma unroll
        for (int m = 0; m < MT; ++m) f.a[m] = fragment<ACOLS, BM, true, KD>(ia, wm * MT + m, 0, lane);
    }
    __device__ static __forceinline__ void multiply(Acc &acc, const Frags &f)
    {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[m][n] = mma<F16>(f.a[m], f.b[n], acc[m][n]);
    }
    // vmcnt(N) lgkmcnt(0), then the barrier
    template <int N>
    __device__ static __forceinline__ void sync()
    {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }

    // with `later` steps requested behind this one
    template <int N, int PER>
    __device__ static __forceinline__ void tail_sync(int later)
    {
        if constexpr (N > 0) {
            if (later >= N) sync<N * PER>();
            else tail_sync<N - 1, PER>(later);
        } else {
            sync<0>();
        }
    }

    // steps [s0, s1) of the nseg * ksteps steps
    __device__ static __forceinline__ void run(Acc &acc, const Operand &A, const Operand &Bo, int nseg, int64_t ksteps, int64_t s0,
                                               int64_t s1, unsigned char *lds)
    {
        const int lane = my_lane(), wave = my_wave();
        const int wm = wave / WN, wn = wave % WN;
        LA la;
        LB lb;
        la.init(A, wave, lane);
        lb.init(Bo, wave, lane);
        int seg = (int)(s0 / ksteps);
        int kk = (int)(s0 % ksteps);
        const int last_k = (int)ksteps, steps = (int)(s1 - s0);
        unsigned char *put = lds, *get = lds;     // images
        la.seek(A, seg_a(seg, nseg), kk);
        lb.seek(Bo, seg_b(seg, nseg), kk);
        auto request = [&]() {
            la.issue(put, A.k_rows - kk * KD, wave);
            lb.issue(put + A_BYTES, Bo.k_rows - kk * KD, wave);
            put = put == lds + (STAGES - 1) * STAGE ? lds : put + STAGE;
            la.next();
            lb.next();
            if (++kk == last_k) {
                kk = 0;
                ++seg;
                if (seg < nseg) {
                    la.seek(A, seg_a(seg, nseg), 0);
                    lb.seek(Bo, seg_b(seg, nseg), 0);
                }
            }
        };
        // requests of one step by the wave that has the fewest (the others wait for a few more than they must)
        constexpr int PER = LA::INSTR / WAVES + LB::INSTR / WAVES;
        constexpr int DEPTH = STAGES - 1;         // steps requested ahead
        static_assert((DEPTH - 1) * PER < 64, "vmcnt has six bits");
        const int pre = steps < DEPTH ? steps : DEPTH;
        for (int i = 0; i < pre; ++i) request();
        // step s has arrived when only the later steps' requests are outstanding; lgkmcnt(0): this wave's reads of the image that
        // the next request overwrites are back
        int s = 0;
        Frags f;
        for (; s + DEPTH < steps; ++s) {
            sync<(DEPTH - 1) * PER>();
            read(f, get, wm, wn, lane);
            request();
            __builtin_amdgcn_sched_barrier(0);
            multiply(acc, f);
            get = get == lds + (STAGES - 1) * STAGE ? lds : get + STAGE;
        }
        for (; s < steps; ++s) {
            tail_sync<DEPTH - 1, PER>(steps - 1 - s);
            read(f, get, wm, wn, lane);
            multiply(acc, f);
            get = get == lds + (STAGES - 1) * STAGE ? lds : get + STAGE;
        }
        asm volatile("" ::: "memory");
        __syncthreads();                          // (an epilogue may use the LDS)
    }

    // first m (inside the tile) of the 16 consecutive ones that acc[4 blk .. 4 blk + 3] hold, and the n of acc[.][nt]
    __device__ static __forceinline__ int m_of(int blk)
    {
        return (my_wave() / WN) * TM + blk * 64 + (my_lane() >> 4) * 16;
    }
    __device__ static __forceinline__ int n_of(int nt)
    {
        const int i = my_lane() & 15, base = (my_wave() % WN) * TN;
        return BCOLS ? base + (nt >> 2) * 64 + (i >> 2) * 16 + (((nt & 3) ^ ((i >> 2) & 1)) << 2) + (i & 3) : base + nt * 16 + i;
    }
    // the four results at m_of(blk) + 4 j
    __device__ static __forceinline__ f32x4 quad(const Acc &acc, int blk, int j, int nt)
    {
        if (!ACOLS) return acc[4 * blk + j][nt];
        const bool odd = (my_lane() >> 4) & 1;
        const f32x4 a = acc[4 * blk + j][nt], b = acc[4 * blk + (j ^ 1)][nt];
        return f32x4{odd ? b[0] : a[0], odd ? b[1] : a[1], odd ? b[2] : a[2], odd ? b[3] : a[3]};
    }
};

// The same product by two groups of four waves (one of each per SIMD) that alternate: while one group multiplies, the other
// reads the fragments of its next products, and a barrier swaps them, so that the matrix units are never without a wave that has
// its operands.  A step in LDS is 64 deep (rows are fetched by whole cache lines), two of them are there, and a wave's share of
// m is two blocks of 64: it reads n and the lower block, multiplies, reads the upper block, multiplies.  So n and the
// lower half of m are free for the step after next as soon as both groups have read them, half a step before the rest, and
// 64 to 112 KB are always on their way (measured, dw of 4096 x 32768 x 512 bf16: requests alone took 104 of 132 us when a
// step was only requested once the one before it was in).  One workgroup per CU.
template <int BM_, int BN_, int WM_, int WN_, bool ACOLS_, bool BCOLS_, bool F16_>
struct DuoTile : Tile<BM_, BN_, WM_, WN_, ACOLS_, BCOLS_, F16_> {
    using Base = Tile<BM_, BN_, WM_, WN_, ACOLS_, BCOLS_, F16_>;
    using Acc = typename Base::Acc;
    static constexpr int BM = BM_, BN = BN_, WN = WN_, MT = Base::MT, NT = Base::NT, WAVES = Base::WAVES;
    static constexpr int KD = 2 * BK, OCCUPANCY = WAVES / 4;
    static constexpr int HALF = BM / 2 * KD * 2, B_BYTES = BN * KD * 2, STAGE = 2 * HALF + B_BYTES, LDS = 2 * STAGE;
    static constexpr int TM = Base::TM;
    using LA = Loader<ACOLS_, BM / 2, true, WAVES, KD, TM>;
    using LB = Loader<BCOLS_, BN, BCOLS_, WAVES, KD>;
    static_assert(WAVES == 8 && TM == 128 && LA::INSTR % WAVES == 0 && LB::INSTR % WAVES == 0, "two groups of four waves");
    static constexpr int LOW = LB::PER_WAVE + LA::PER_WAVE, HIGH = LA::PER_WAVE;     // requests of a wave

    __device__ static __forceinline__ void swap()         // end of a phase: this wave's reads are back
    {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xC07F);               // lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }
    template <int N>
    __device__ static __forceinline__ void arrived() { __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14)); }   // vmcnt(N)

    // What a wave keeps between its requests.  begin() asks for the first steps of a product (the images must be free), finish()
    // runs it; between the two a kernel may do other work (the results of the product before).
    struct Pipe {
        LA lo, hi;
        LB lb;
        Operand A, B;
        int nseg, last_k, steps, seg_lo, k_lo, seg_hi, k_hi;
        int wave;
        unsigned char *lds;

        // step s of n and the lower half of m; of the upper half: both are called for s = 0, 1, ...
        __device__ __forceinline__ void request_low(unsigned char *img)
        {
            lb.issue(img + 2 * HALF, B.k_rows - k_lo * KD, wave);
            lo.issue(img, A.k_rows - k_lo * KD, wave);
            lb.next();
            lo.next();
            if (++k_lo == last_k && ++seg_lo < nseg) {
                k_lo = 0;
                lo.seek(A, seg_a(seg_lo, nseg), 0);
                lb.seek(B, seg_b(seg_lo, nseg), 0);
            }
        }
        __device__ __forceinline__ void request_high(unsigned char *img)
        {
            hi.issue(img + HALF, A.k_rows - k_hi * KD, wave);
            hi.next();
            if (++k_hi == last_k && ++seg_hi < nseg) {
                k_hi = 0;
                hi.seek(A, seg_a(seg_hi, nseg), 0);
            }
        }

        // steps [s0, s1) of the nseg * ksteps steps of 64
        __device__ __forceinline__ void begin(const Operand &A_, const Operand &B_, int nseg_, int64_t ksteps, int64_t s0, int64_t s1,
                                              unsigned char *lds_)
        {
            A = A_; B = B_; nseg = nseg_; lds = lds_;
            wave = my_wave();
            const int lane = my_lane();
            last_k = (int)ksteps;
            steps = (int)(s1 - s0);
            lo.init(A, wave, lane, 0);
            hi.init(A, wave, lane, 64);
            lb.init(B, wave, lane);
            seg_lo = seg_hi = (int)(s0 / ksteps);
            k_lo = k_hi = (int)(s0 % ksteps);
            lo.seek(A, seg_a(seg_lo, nseg), k_lo);
            hi.seek(A, seg_a(seg_lo, nseg), k_lo);
            lb.seek(B, seg_b(seg_lo, nseg), k_lo);
            if (steps > 0) {
                request_low(lds);
                request_high(lds);
            }
            if (steps > 1) request_low(lds + STAGE);
        }

        // AFTER: requests to memory (stores) of this wave between begin() and here, if `after_begin`: the waits for what begin() asked
        // for need not wait for them
        template <int AFTER = 0>
        __device__ __forceinline__ void finish(Acc &acc, bool after_begin = false)
        {
            const int lane = my_lane(), wm = wave / WN, wn = wave % WN;
            const bool second = wave >= 4;
            u32x4 a[2][4], b[2][NT];
            auto read_a = [&](const unsigned char *half) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int m = 0; m < 4; ++m) a[k][m] = fragment<ACOLS_, BM / 2, true, KD>(half, wm * 4 + m, k, lane);
            };
            auto multiply = [&](int base) {
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int m = 0; m < 4; ++m)
#pragma unroll
                        for (int n = 0; n < NT; ++n) acc[base + m][n] = mma<F16_>(a[k][m], b[k][n], acc[base + m][n]);
                __builtin_amdgcn_s_setprio(0);
            };
            unsigned char *img = lds, *other = lds + STAGE;
            auto in_but = [&](bool more, bool first) {           // all but the last LOW + HIGH requests (and the stores) are in
                if (!more) arrived<0>();
                else if (first) arrived<LOW + HIGH + AFTER>();
                else arrived<LOW + HIGH>();
            };
            in_but(steps > 1, after_begin);
            swap();
            if (second) swap();                               // one phase behind
            for (int s = 0; s < steps; ++s) {
                const bool next = s + 1 < steps, after = s + 2 < steps, first = after_begin && s == 0;
                // upper m of the other image: step s - 1 was read there a phase ago by both groups
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int n = 0; n < NT; ++n) b[k][n] = fragment<BCOLS_, BN, BCOLS_, KD>(img + 2 * HALF, wn * NT + n, k, lane);
                read_a(img);
                if (next) request_high(other);
                // what the first group reads in its next phase has to be in by the end of the phase before it: the first group's
                // own products, the second group's reads
                if (second) in_but(next, first);
                swap();
                multiply(0);
                if (!second) in_but(next, first);
                swap();
                read_a(img + HALF);
                if (after) request_low(img);                  // n and lower m of this image: both groups have read them
                if (second) in_but(after, first);
                swap();
                multiply(4);
                if (!second) in_but(after, first);
                swap();
                unsigned char *t = img;
                img = other;
                other = t;
            }
            if (!second) swap();
            swap();                                           // (the images are free)
        }
    };

    __device__ static __forceinline__ void run(Acc &acc, const Operand &A, const Operand &Bo, int nseg, int64_t ksteps, int64_t s0,
                                               int64_t s1, unsigned char *lds)
    {
        Pipe p;
        p.begin(A, Bo, nseg, ksteps, s0, s1, lds);
        p.finish(acc);
    }
};

}  // namespace mfma16
