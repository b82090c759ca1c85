// Tiles of 16-bit matrix products on v_mfma_f32_16x16x32_{bf16,f16}, fed from LDS that global_load_lds fills.
//
//   acc[m][n] += sum_k A(m, k) B(n, k)
//
// Each operand is stored in one of two ways:
//   rows     [m][k], k contiguous: a fragment is one ds_read_b128 of 8 consecutive k
//   columns  [k][m], m contiguous: a fragment is two ds_read_b64_tr_b16 (the hardware's 4 x 16 transposition)
// One K step is 32 wide.  A workgroup of 4 waves holds STAGES steps in LDS: step s + 2 is requested while step s is multiplied,
// one barrier a step, and the waits count outstanding requests (vmcnt) instead of draining them.
//
// M rows are permuted inside blocks of 64 so that a lane's 16 accumulators of a block are 16 CONSECUTIVE m of one n:
// matrix row i of tile t of a block is m = 16 (i / 4) + 4 t + (i & 3).  For "rows" the permutation costs nothing (it picks which
// global row is fetched into which LDS row), for "columns" it is the address of the transposed read.  An epilogue then
// stores 32 bytes of 16-bit results (64 of fp32) per lane and 128 (256) contiguous bytes per n.
//
// LDS bank conflicts: 16-byte chunks of a row are XORed with row bits (the fetch applies the same XOR to its source address,
// since global_load_lds writes lanes linearly), so that every 8-lane pass of a b128 read and every 16-lane pass of a
// transposed read touches each bank once.
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

constexpr int BK = 32;          // K step
constexpr int STAGES = 3;       // steps in LDS
constexpr int WAVES = 4;
constexpr int THREADS = 64 * WAVES;

template <bool F16>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c)
{
    if (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// An operand as the tile sees it: `base` points at its first element (row 0 or column 0 of the tile, k = first k),
// `ld` in elements.  rows: `lim` = last valid row of the tile's rows (later ones read that row again; their results are
// not used).  columns: `lim` = last valid column chunk (8 columns), likewise.
struct Operand {
    const unsigned short *base;
    int64_t plane;              // elements between the parts of a split fp32 operand
    int64_t ld;
    int lim;
    int64_t k_rows;             // columns only: valid k (later ones read the last row again: the other operand is zero there)
};

// the six products of two three-part operands, small ones first: (part of A, part of B)
__device__ __forceinline__ int seg_a(int s, int nseg) { return nseg == 1 ? 0 : (0x012010 >> (4 * (5 - s))) & 0xf; }
__device__ __forceinline__ int seg_b(int s, int nseg) { return nseg == 1 ? 0 : (0x210100 >> (4 * (5 - s))) & 0xf; }

template <bool COLS, int B, bool PERM>
struct Loader {
    static constexpr int INSTR = B * BK * 2 / 1024;              // 1 KB requests per step
    static constexpr int PER_WAVE = (INSTR + WAVES - 1) / WAVES; // (the last may be idle for some waves)
    static constexpr int CHUNKS = COLS ? B / 8 : 4;              // 16-byte chunks per LDS row
    static_assert(!COLS || B == 64 || B == 128 || B == 256, "columns operand width");

    __device__ static __forceinline__ int swz(int row)
    {
        if (!COLS) return (row >> 1) & 3;
        return B >= 128 ? ((row & 1) | ((row & 2) << 2)) : ((row >> 1) & 1);
    }

    // offset (rows: bytes from the step's base; columns: LDS row in the high half, byte column in the low)
    unsigned off[PER_WAVE];

    __device__ __forceinline__ void init(const Operand &o, int wave, int lane)
    {
#pragma unroll
        for (int j = 0; j < PER_WAVE; ++j) {
            const int slot = (j * WAVES + wave) * 64 + lane;
            const int row = slot / CHUNKS, c = (slot % CHUNKS) ^ swz(row);
            if (!COLS) {
                int m = row;
                if (PERM) m = (row & ~63) | (((row & 15) >> 2) << 4) | (((row >> 4) & 3) << 2) | (row & 3);
                m = m < o.lim ? m : o.lim;
                off[j] = (unsigned)(m * (int)o.ld * 2 + c * 16);
            } else {
                const int cc = c < o.lim ? c : o.lim;
                off[j] = ((unsigned)row << 16) | (unsigned)(cc * 16);
            }
        }
    }

    // request step kk of part `part` into the LDS image `dst`
    __device__ __forceinline__ void issue(const Operand &o, int part, int64_t kk, unsigned char *dst, int wave) const
    {
        const unsigned char *b = (const unsigned char *)(o.base + part * o.plane + (COLS ? kk * BK * o.ld : kk * BK));
        const int64_t left = o.k_rows - 1 - kk * BK;
        const int last = COLS ? (int)(left < BK - 1 ? left : BK - 1) : 0;
#pragma unroll
        for (int j = 0; j < PER_WAVE; ++j) {
            const int i = j * WAVES + wave;
            if (INSTR % WAVES != 0 && i >= INSTR) continue;
            unsigned bo = off[j];
            if (COLS) {
                int r = (int)(bo >> 16);
                r = r < last ? r : last;
                bo = (unsigned)r * (unsigned)(o.ld * 2) + (bo & 0xffffu);
            }
            __builtin_amdgcn_global_load_lds((glob_void *)(b + bo), (lds_void *)(dst + i * 1024), 16, 0, 0);
        }
    }
};

// fragment t (16 wide) of 64-block blk
template <bool COLS, int B, bool PERM>
__device__ __forceinline__ u32x4 fragment(const unsigned char *img, int tile16, int lane)
{
    using L = Loader<COLS, B, PERM>;
    if (!COLS) {
        const int row = tile16 * 16 + (lane & 15);
        return *(const u32x4 *)(img + row * 64 + (((lane >> 4) ^ L::swz(row)) << 4));
    }
    const int g = lane >> 4, q = (lane & 15) >> 2, p = lane & 3, k = 8 * g + q;
    const int blk = tile16 >> 2, t = tile16 & 3;
    const int c = (blk * 8 + 2 * p + (t >> 1)) ^ L::swz(k);
    const unsigned char *a = img + k * (B * 2) + c * 16 + (t & 1) * 8;
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16 *)a);
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16 *)(a + 4 * (B * 2)));
    const unsigned long long l = __builtin_bit_cast(unsigned long long, lo), h = __builtin_bit_cast(unsigned long long, hi);
    return u32x4{(unsigned)l, (unsigned)(l >> 32), (unsigned)h, (unsigned)(h >> 32)};
}

template <int BM_, int BN_, int WM_, bool ACOLS_, bool BCOLS_, bool F16_>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WAVES / WM_;     // waves along m and n
    static constexpr bool ACOLS = ACOLS_, BCOLS = BCOLS_, F16 = F16_;
    static constexpr int TM = BM / WM, TN = BN / WN;                         // per wave
    static constexpr int MT = TM / 16, NT = TN / 16;
    static constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, STAGE = A_BYTES + B_BYTES;
    static constexpr int LDS = STAGES * STAGE;
    using LA = Loader<ACOLS, BM, true>;
    using LB = Loader<BCOLS, BN, BCOLS>;
    static_assert(TM % 64 == 0, "a wave holds whole permuted blocks");
    static_assert(!BCOLS || TN % 64 == 0, "transposed reads go by blocks of 64");

    // steps [s0, s1) of the nseg * ksteps steps
    __device__ static __forceinline__ void run(f32x4 (&acc)[MT][NT], const Operand &A, const Operand &Bo, int nseg, int64_t ksteps,
                                               int64_t s0, int64_t s1, unsigned char *lds)
    {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wm = wave / WN, wn = wave % WN;
        LA la;
        LB lb;
        la.init(A, wave, lane);
        lb.init(Bo, wave, lane);
        int seg = (int)(s0 / ksteps);
        int64_t kk = s0 % ksteps;
        auto request = [&](int64_t s) {
            unsigned char *st = lds + (int)((s - s0) % STAGES) * STAGE;
            la.issue(A, seg_a(seg, nseg), kk, st, wave);
            lb.issue(Bo, seg_b(seg, nseg), kk, st + A_BYTES, wave);
            if (++kk == ksteps) { kk = 0; ++seg; }
        };
        if (s0 < s1) request(s0);
        if (s0 + 1 < s1) request(s0 + 1);
        for (int64_t s = s0; s < s1; ++s) {
            // step s has arrived when only step s + 1's requests are outstanding; lgkmcnt(0): this wave's reads of the image
            // that step s + 2 overwrites are back
            asm volatile("" ::: "memory");
            if (s + 1 < s1 && LA::INSTR % WAVES == 0 && LB::INSTR % WAVES == 0)
                __builtin_amdgcn_s_waitcnt(0x0070 | (LA::PER_WAVE + LB::PER_WAVE));
            else
                __builtin_amdgcn_s_waitcnt(0x0070);
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (s + 2 < s1) request(s + 2);       // into the image that every wave has finished reading
            const unsigned char *ia = lds + (int)((s - s0) % STAGES) * STAGE, *ib = ia + A_BYTES;
            u32x4 b[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) b[n] = fragment<BCOLS, BN, BCOLS>(ib, wn * NT + n, lane);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const u32x4 a = fragment<ACOLS, BM, true>(ia, wm * MT + m, lane);
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[m][n] = mma<F16>(a, b[n], acc[m][n]);
            }
        }
        asm volatile("" ::: "memory");
        __syncthreads();                          // (an epilogue may use the LDS)
    }

    // first m (inside the tile) of the 16 consecutive ones that acc[4 blk .. 4 blk + 3] hold, and the n of acc[.][nt]
    __device__ static __forceinline__ int m_of(int blk)
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        return (wave / WN) * TM + blk * 64 + (lane >> 4) * 16;
    }
    __device__ static __forceinline__ int n_of(int nt)
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15;
        const int base = (wave % WN) * TN;
        return BCOLS ? base + (nt >> 2) * 64 + (i >> 2) * 16 + (nt & 3) * 4 + (i & 3) : base + nt * 16 + i;
    }
};

}  // namespace mfma16
