// A linear head over many classes and its losses, without the logits in memory:
//
//   z = x w^T                                          x [N, D] features, w [V, D] class codes
//   cross entropy   l_n = lse_n - z_{n, y_n}
//   distillation    l_n = T^2 sum_k q_nk (log q_nk - z_{n, i_nk} / T + lse_n),   q = softmax of the teacher's listed logits / T
//                   lse_n = log sum_j exp(z_nj / T)
//   gradient        dz = T g_n (softmax(z / T) - q),   dx = dz w,   dw = dz^T x
//
// Cross entropy is the distillation of one entry with q = 1 and T = 1, so one set of kernels serves both.
//
// Forward: the tiles of z never leave the registers: each writes its rows' maximum and sum of exponentials, and one wave per row
// joins them and takes the logits of the K listed classes as K dot products.  The first listed class (the label) is left out of
// the tiles' sums and joined from its dot product: with R the sum over the others, lse - z_y = log(1 + R exp(-z_y)) and
// 1 - p_y = 1 / (1 + exp(z_y) / R) keep all their digits where the head is sure of itself, and both uses of z_y see one rounding.
// Backward, in pieces of the classes: the tiles are computed again and leave as 16-bit dz [rows][piece]; two products read it
// (dx over the piece, dw of the piece).  A piece is at most DZ_BYTES, unless 256 classes of all the rows are more (beyond 2^18 rows, fp32 87381):
// it is still in the last-level cache when it is read (products at V = 131072: 1005 us; with 64 MB pieces, twice as many launches, 1267, with 256 MB 1273).
//
// Bound by the matrix units, and by what runs between products.  4096 x 32768 x 512 bf16: z 152 us (0.90 PF/s, about a quarter of
// it the exponentials), dz 174, the two products 275 (1.0 PF/s); matrix units busy 43, 36 and 48 % of the cycles, at 1.7-1.8 GHz.  32 rows or less are
// bound by reading the codes: 16 x 65536 x 512 bf16 13.7 us (4.9 TB/s).
//
// Number formats.  bf16 and fp16 operands enter the matrix unit as they are, sums are fp32.  fp32 operands are split into three
// bf16 parts (24 significant bits) and six products are summed, small ones first.  dz is rounded once to the operands' type
// (fp32: to three parts): softmax(z) - q lies in [-1, 1], an error of half a step per entry averages out over the sums that
// follow and stays below the rounding of the results.  fp16 holds it times 2^12, so that probabilities down to 1.5e-8 are
// normal numbers.  The rows' weights T g_n go into dz before its rounding, relative to the largest one (equal weights: a factor
// of exactly 1; in a copy of x they would cost a second rounding: fp16 dw 0.00037 instead of 0.00027 from the 64-bit result).
//
// Rows that take part in nothing (an ignored label, no listed entry) are exactly zero in every output, whatever x holds.
// No atomics on floats: every sum has a fixed order and results repeat bit for bit.
#include "mfma16.h"

using namespace mfma16;

namespace {

constexpr int T_F32 = 0, T_BF16 = 1, T_F16 = 2;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float F16_DZ = 4096.0f;
constexpr int64_t DZ_BYTES = 128ll << 20;      // of one piece of dz
// us of a step (64 deep) of a job of the products, and steps that a job costs beyond its own.  With 256 x 256 tiles alone 1000 x 10000 x
// 200 bf16 took 90 us (here 76), with 128 x 128 ones 4096 x 32768 x 512 607 us (here 558); 0.45 to 0.65 chose alike but for long rows.
constexpr double STEP_256 = 1.0, STEP_128 = 0.57, JOB_STEPS = 6.0;
constexpr double PIECE = 15.0;
constexpr int CUS = 256;                        // MI355X
constexpr int64_t WPACK_BYTES = 128ll << 20;   // of the packed class codes of one piece

__device__ __forceinline__ float bf2f(unsigned short u) { return __builtin_bit_cast(float, (unsigned)u << 16); }
__device__ __forceinline__ float hf2f(unsigned short u) { return (float)__builtin_bit_cast(_Float16, u); }
__device__ __forceinline__ unsigned short f2bf(float f) { return __builtin_bit_cast(unsigned short, (__bf16)f); }
__device__ __forceinline__ unsigned short f2hf(float f) { return __builtin_bit_cast(unsigned short, (_Float16)f); }
template <bool F16> __device__ __forceinline__ unsigned short to16(float f) { return F16 ? f2hf(f) : f2bf(f); }

// two at once, the first in the low half
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <bool F16> __device__ __forceinline__ unsigned to16_two(float a, float b)
{
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {a, b};
    return F16 ? __builtin_bit_cast(unsigned, __builtin_convertvector(v, h2)) : __builtin_bit_cast(unsigned, __builtin_convertvector(v, b2));
}

template <int DT> __device__ __forceinline__ float load1(const void *p, int64_t i)
{
    if (DT == T_F32) return ((const float *)p)[i];
    const unsigned short u = ((const unsigned short *)p)[i];
    return DT == T_BF16 ? bf2f(u) : hf2f(u);
}
template <int DT> __device__ __forceinline__ void store1(void *p, int64_t i, float v)
{
    if (DT == T_F32) ((float *)p)[i] = v;
    else ((unsigned short *)p)[i] = DT == T_BF16 ? f2bf(v) : f2hf(v);
}

// vectors at any address of an element (rows of an odd length start anywhere)
template <class V, int ALIGN> struct __attribute__((packed, aligned(ALIGN))) Anywhere { V v; };
template <class V, int DT> __device__ __forceinline__ V load_at(const void *p, int64_t i)
{
    constexpr int SIZE = DT == T_F32 ? 4 : 2;
    return ((const Anywhere<V, SIZE> *)((const unsigned char *)p + i * SIZE))->v;
}
template <int DT, class V> __device__ __forceinline__ void store_at(void *p, int64_t i, V v)
{
    constexpr int SIZE = DT == T_F32 ? 4 : 2;
    ((Anywhere<V, SIZE> *)((unsigned char *)p + i * SIZE))->v = v;
}

// three bf16 parts of an fp32 number (an infinity or NaN stays in the first part)
__device__ __forceinline__ void split3(float v, unsigned short (&h)[3])
{
    h[0] = f2bf(v);
    const float a = bf2f(h[0]);
    const bool fin = fabsf(a) < __builtin_inff();
    const float r1 = fin ? v - a : 0.0f;
    h[1] = f2bf(r1);
    h[2] = f2bf(r1 - bf2f(h[1]));
}

// of two finite numbers (others become NaN)
__device__ __forceinline__ void split3_two(float a, float b, unsigned *h)
{
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        h[k] = to16_two<false>(a, b);
        a -= __builtin_bit_cast(float, h[k] << 16);
        b -= __builtin_bit_cast(float, h[k] & 0xffff0000u);
    }
}

// (maximum, sum of 2^(. - maximum)) of two sets; a set without a finite element has maximum -inf and a sum of 0 or NaN
__device__ __forceinline__ float2 join_stats(float2 a, float2 b)
{
    const float m = fmaxf(a.x, b.x);
    const float fa = a.x > -__builtin_inff() ? __builtin_amdgcn_exp2f(a.x - m) : 1.0f;
    const float fb = b.x > -__builtin_inff() ? __builtin_amdgcn_exp2f(b.x - m) : 1.0f;
    return float2{m, a.y * fa + b.y * fb};
}

// logical tile of a block: each of the 8 XCDs (its own 4 MB L2) walks a contiguous range of tiles
__device__ __forceinline__ int64_t xcd_tile(int64_t total)
{
    const int64_t b = blockIdx.x, per = (total + 7) / 8;
    const int64_t i = b / 8 + (b & 7) * per;
    return (b / 8 < per && i < total) ? i : -1;
}

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// ---- before a pass, in one launch: operands as 16-bit parts, row weights -----------------------------------------------------
// [rows][d] of any type -> [P][rows_pad][dp], zero padded.  lse (may be NULL): the rows are those of the gradient; one that takes
// part in nothing, or has no weight, becomes zero whatever it holds.
struct Pack { const void *src; int64_t rows, rows_pad; unsigned short *dst; };
struct PrepArgs {
    Pack p[2];
    int64_t chunks[2];           // 8-element chunks of the two
    int d, dp;
    // weight of a row in the gradient: T g_n (mean: / count), 0 where it takes part in nothing; top[0] = the largest |weight|
    const float *lse, *g, *count;
    int g_per_row;
    float temperature;
    int64_t n;
    float *weight, *top;         // NULL: a forward pass
};
constexpr int PREP = 1024;

template <int DT>
__global__ void __launch_bounds__(PREP) prep_kernel(PrepArgs a)
{
    if (a.weight != nullptr && blockIdx.x == 0) {
        __shared__ float sm[PREP / 64];
        const float f = a.count != nullptr ? a.temperature / a.count[0] : a.temperature;
        float m = 0.0f;
        for (int64_t i = threadIdx.x; i < a.n; i += PREP) {
            const float wr = a.lse[i] != __builtin_inff() ? a.g[a.g_per_row ? i : 0] * f : 0.0f;
            a.weight[i] = wr;
            m = fmaxf(m, fabsf(wr) < __builtin_inff() ? fabsf(wr) : 0.0f);      // (an infinite or NaN one spoils its own row)
        }
        m = wave_max(m);
        if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int i = 0; i < PREP / 64; ++i) m = fmaxf(m, sm[i]);
            a.top[0] = m > 0.0f ? m : 1.0f;
        }
        return;
    }
    const int64_t blocks = gridDim.x - (a.weight != nullptr), block = blockIdx.x - (a.weight != nullptr);
    const int per = a.dp / 8;
    for (int64_t j = block * PREP + threadIdx.x; j < a.chunks[0] + a.chunks[1]; j += blocks * PREP) {
        const bool second = j >= a.chunks[0];
        const Pack &p = a.p[second];
        const int64_t i = second ? j - a.chunks[0] : j, r = i / per;
        const int c = (int)(i % per) * 8;
        bool live = r < p.rows;
        if (live && !second && a.lse != nullptr) live = a.lse[r] != __builtin_inff() && a.g[a.g_per_row ? r : 0] != 0.0f;
        float x[8];
        if (live && c + 8 <= a.d) {
            u32x4 raw[2];
            raw[0] = load_at<u32x4, DT>(p.src, r * a.d + c);
            if (DT == T_F32) raw[1] = load_at<u32x4, DT>(p.src, r * a.d + c + 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = load1<DT>(raw, e);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = live && c + e < a.d ? load1<DT>(p.src, r * a.d + c + e) : 0.0f;
        }
        unsigned short o[3][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = x[e];
            if (DT == T_F32) {
                unsigned short h[3];
                split3(v, h);
                o[0][e] = h[0]; o[1][e] = h[1]; o[2][e] = h[2];
            } else {
                o[0][e] = to16<DT == T_F16>(v);
            }
        }
#pragma unroll
        for (int k = 0; k < (DT == T_F32 ? 3 : 1); ++k) *(u32x4 *)(p.dst + (k * p.rows_pad + r) * a.dp + c) = *(const u32x4 *)o[k];
    }
}

// ---- z = x w^T by tiles: statistics, or dz ----------------------------------------------------------------------------------
struct HeadArgs {
    Operand w, x;                // base of the piece's first class / of row 0
    int64_t n, vc;               // rows, classes of the piece
    int nseg;
    int64_t depth;               // K: a multiple of 64 (zeros behind the features)
    float c;                     // log2(e) / T
    int64_t tiles_n, tiles;
    // statistics
    float2 *stats;               // [class tile][n]: maximum and sum of 2^(c z - maximum)
    int64_t tile0;               // first class tile of the piece
    // dz
    const float *lse;            // [n] in powers of two; +inf: a row that takes part in nothing; [n] 1 - p of the first listed class
    const float *weight, *top;   // [n], [1]
    const int64_t *label;        // first listed class of a row, label_step apart (dz: labels, or NULL)
    int64_t label_step;
    int64_t v0;
    unsigned short *dz;          // [parts][n_pad][ldz]
    int64_t n_pad, ldz;
};

// operands of tile t and where it lies
template <class TL>
__device__ __forceinline__ void head_tile(const HeadArgs &a, int64_t t, Operand &W, Operand &X, int64_t &m0, int64_t &n0)
{
    m0 = t / a.tiles_n * TL::BM;
    n0 = t % a.tiles_n * TL::BN;
    W = a.w;
    X = a.x;
    if (m0 >= a.vc || n0 >= a.n) return;        // (nothing to read: a tile of zeros)
    W.base += m0 * W.ld;
    W.lim = (int)(a.vc - 1 - m0 < TL::BM - 1 ? a.vc - 1 - m0 : TL::BM - 1);
    X.base += n0 * X.ld;
    X.lim = (int)(a.n - 1 - n0 < TL::BN - 1 ? a.n - 1 - n0 : TL::BN - 1);
}

// per row: the weight f relative to the largest (0: the row takes part in nothing, whatever its logits are), lse - log2 |f| (the weight goes
// into the exponent), the label's class relative to the tile's first
template <class TL>
struct RowState {
    float lse[TL::NT], f[TL::NT];
    int label[TL::NT];
    __device__ __forceinline__ void load(const HeadArgs &a, int64_t m0, int64_t n0)
    {
        const int rows = (int)(a.n - n0 < TL::BN ? a.n - n0 : TL::BN);
        const float *pl = a.lse + n0, *pw = a.weight + n0;
        const int *pt = a.label != nullptr ? (const int *)(a.label + n0) : (const int *)pl;
        const int two = a.label != nullptr ? 2 : 1;
#pragma unroll
        for (int nt = 0; nt < TL::NT; ++nt) {
            int n = TL::n_of(nt);
            n = n < rows ? n : (rows > 0 ? rows - 1 : 0);
            lse[nt] = rows > 0 ? pl[n] : __builtin_inff();
            f[nt] = rows > 0 ? pw[n] : 0.0f;
            label[nt] = rows > 0 ? pt[n * two] : 0;      // (the low half: a row that takes part has a label of this head)
        }
        const float top = a.top[0];
        // here, and not behind the requests of the next tile: the loads' wait would wait for those too
#pragma unroll
        for (int nt = 0; nt < TL::NT; ++nt) asm volatile("" ::"v"(lse[nt]), "v"(f[nt]), "v"(label[nt]));
        const int first = (int)(a.v0 + m0);
#pragma unroll
        for (int nt = 0; nt < TL::NT; ++nt) {
            const bool live = TL::n_of(nt) < rows && lse[nt] != __builtin_inff();
            f[nt] = live ? f[nt] / top * (TL::F16 ? F16_DZ : 1.0f) : 0.0f;      // (equal weights: exactly 1)
            lse[nt] -= __builtin_amdgcn_logf(fabsf(f[nt]));
            label[nt] = f[nt] != 0.0f && a.label != nullptr ? label[nt] - first : -1;
        }
    }
};

// what a tile needs of its rows: the state above for dz, for statistics the class that is left out, relative to the head's first
// (one that is not there: -1)
template <class TL, bool DZ>
struct TileRows : RowState<TL> {};
template <class TL>
struct TileRows<TL, false> {
    int label[TL::NT];
    int2 raw[TL::NT];
    __device__ __forceinline__ void request(const HeadArgs &a, int64_t n0)
    {
#pragma unroll
        for (int nt = 0; nt < TL::NT; ++nt) {
            const int64_t n = n0 + TL::n_of(nt);
            raw[nt] = *(const int2 *)(a.label + (n < a.n ? n : a.n - 1) * a.label_step);
        }
    }
    __device__ __forceinline__ void load(const HeadArgs &, int64_t, int64_t)
    {
#pragma unroll
        for (int nt = 0; nt < TL::NT; ++nt) {
            label[nt] = raw[nt].y == 0 ? raw[nt].x : -1;
            asm volatile("" ::"v"(label[nt]));       // (here, as above)
        }
    }
};

template <class TL, bool DZ, int PARTS>
__device__ __forceinline__ void head_results(const HeadArgs &a, typename TL::Acc &acc, const TileRows<TL, DZ> &rows, int64_t m0, int64_t n0,
                                             float2 *part /* [WM][BN], LDS */)
{
    const bool whole = a.vc - m0 >= TL::BM;     // else the last classes of the tile are not there
    const int left = whole ? TL::BM : (int)(a.vc - m0);      // (0 or less: a tile of zeros)
    if constexpr (!DZ) {
        const int lane = my_lane(), wm = my_wave() / TL::WN;
        if (!whole) {
#pragma unroll
            for (int mt = 0; mt < TL::MT; ++mt) {
                const int m = TL::m_of(mt >> 2) + (mt & 3) * 4;
#pragma unroll
                for (int nt = 0; nt < TL::NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[mt][nt][r] = m + r < left ? acc[mt][nt][r] : -__builtin_inff();
            }
        }
        const int wave_m = (int)(a.v0 + m0) + wm * TL::TM;
#pragma unroll
        for (int nt = 0; nt < TL::NT; ++nt) {
            const int label = rows.label[nt] - wave_m;
            if (label >= 0 && label < TL::TM) {
#pragma unroll
                for (int b = 0; b < TL::MT / 4; ++b) {
                    const int l = label - (TL::m_of(b) - wm * TL::TM);
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[4 * b + (e >> 2)][nt][e & 3] = e == l ? -__builtin_inff() : acc[4 * b + (e >> 2)][nt][e & 3];
                }
            }
            // (c > 0: the maximum of z is that of c z; one fma, one exponential and one sum per logit)
            float mx = -__builtin_inff();
#pragma unroll
            for (int mt = 0; mt < TL::MT; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[mt][nt][r]);
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            mx *= a.c;
            const float ref = mx > -__builtin_inff() ? mx : 0.0f;
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int mt = 0; mt < TL::MT; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[r] += __builtin_amdgcn_exp2f(fmaf(acc[mt][nt][r], a.c, -ref));
            float t = (s[0] + s[1]) + (s[2] + s[3]);
            t += __shfl_xor(t, 16, 64);
            t += __shfl_xor(t, 32, 64);
            if (lane < 16) part[wm * TL::BN + TL::n_of(nt)] = float2{mx, t};
        }
        __syncthreads();
        for (int n = threadIdx.x; n < TL::BN; n += TL::THREADS) {
            if (n0 + n >= a.n) continue;
            float2 p = part[n];
#pragma unroll
            for (int k = 1; k < TL::WM; ++k) p = join_stats(p, part[k * TL::BN + n]);
            a.stats[(a.tile0 + m0 / TL::BM) * a.n + n0 + n] = p;
        }
    } else {
        constexpr bool F16 = TL::F16;
#pragma unroll
        for (int nt = 0; nt < TL::NT; ++nt) {
            const float lse = rows.lse[nt], f = rows.f[nt];
            unsigned short *to = a.dz + (n0 + TL::n_of(nt)) * a.ldz + m0;
#pragma unroll
            for (int b = 0; b < TL::MT / 4; ++b) {
                const int m = TL::m_of(b), label = rows.label[nt] - m;
                float p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(acc[4 * b + (e >> 2)][nt][e & 3], a.c, -lse));
                if (f < 0.0f) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) p[e] = -p[e];
                }
                if (label >= 0 && label < 16) {
                    const float miss = a.lse[a.n + n0 + TL::n_of(nt)];      // (in a walk this waits for the next tile's requests too)
#pragma unroll
                    for (int e = 0; e < 16; ++e) p[e] = e == label ? -miss * f : p[e];
                }
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) p[e] = e < left - m ? p[e] : 0.0f;
                }
                u32x4 o[PARTS][2];
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    unsigned h[PARTS];
                    if (PARTS == 3) split3_two(p[e], p[e + 1], h);
                    else h[0] = to16_two<F16>(p[e], p[e + 1]);
#pragma unroll
                    for (int k = 0; k < PARTS; ++k) o[k][e >> 3][(e >> 1) & 3] = h[k];
                }
                if (f == 0.0f) {
#pragma unroll
                    for (int k = 0; k < PARTS; ++k) o[k][0] = o[k][1] = u32x4{0u, 0u, 0u, 0u};
                }
#pragma unroll
                for (int k = 0; k < PARTS; ++k) {
                    u32x4 *d = (u32x4 *)(to + k * a.n_pad * a.ldz + m);
                    d[0] = o[k][0];
                    d[1] = o[k][1];
                }
            }
        }
    }
}

template <class TL>
__device__ __forceinline__ void clear(typename TL::Acc &acc)
{
#pragma unroll
    for (int i = 0; i < TL::MT; ++i)
#pragma unroll
        for (int j = 0; j < TL::NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// one tile per workgroup
template <class TL, bool DZ, int PARTS>
__global__ void __launch_bounds__(TL::THREADS, TL::OCCUPANCY) head_kernel(HeadArgs a)
{
    __shared__ __attribute__((aligned(1024))) unsigned char lds[TL::LDS];
    const int64_t t = xcd_tile(a.tiles);
    if (t < 0) return;
    Operand W, X;
    int64_t m0, n0;
    head_tile<TL>(a, t, W, X, m0, n0);
    typename TL::Acc acc;
    clear<TL>(acc);
    const int64_t ksteps = a.depth / TL::KD;
    const bool there = m0 < a.vc && n0 < a.n;
    TileRows<TL, DZ> rows;
    if constexpr (!DZ) rows.request(a, n0);
    TL::run(acc, W, X, a.nseg, ksteps, 0, there ? a.nseg * ksteps : 0, lds);
    rows.load(a, m0, n0);
    head_results<TL, DZ, PARTS>(a, acc, rows, m0, n0, (float2 *)lds);
}

// One workgroup per CU walks its tiles; the first steps of the next tile are on their way while the results of this one are
// worked out.  Each XCD has a contiguous eighth of the tiles (rows run fastest) and its workgroups take neighbouring ones:
// they share the class codes in the XCD's L2.
template <class TL, bool DZ, int PARTS>
__global__ void __launch_bounds__(TL::THREADS, TL::OCCUPANCY) head_walk_kernel(HeadArgs a)
{
    __shared__ __attribute__((aligned(1024))) unsigned char lds[TL::LDS];
    __shared__ float2 part[TL::WM * TL::BN];
    const int64_t per = (a.tiles + 7) / 8, first = (blockIdx.x & 7) * per, stride = gridDim.x >> 3;
    const int64_t end = first + per < a.tiles ? first + per : a.tiles;
    const int64_t ksteps = a.depth / TL::KD, steps = a.nseg * ksteps;
    int64_t t = first + (blockIdx.x >> 3);
    if (t >= end) return;
    Operand W, X;
    int64_t m0, n0;
    typename TL::Pipe pipe;
    TileRows<TL, DZ> rows;
    head_tile<TL>(a, t, W, X, m0, n0);
    if constexpr (!DZ) rows.request(a, n0);           // (before the tile's requests: the waits count what comes after)
    pipe.begin(W, X, a.nseg, ksteps, 0, steps, lds);
    // stores of dz by a wave behind the requests of its next tile (head_results: two per part, block of 64 classes and 16 rows)
    constexpr int STORES = DZ ? 2 * PARTS * (TL::MT / 4) * TL::NT : 0;
    static_assert(TL::LOW + TL::HIGH + STORES < 64, "vmcnt has six bits");
    for (bool later = false;; later = true) {
        typename TL::Acc acc;
        clear<TL>(acc);
        pipe.template finish<STORES>(acc, later);
        rows.load(a, m0, n0);
        const int64_t m = m0, n = n0;
        t += stride;
        if (t < end) {
            head_tile<TL>(a, t, W, X, m0, n0);
            if constexpr (!DZ) rows.request(a, n0);
            pipe.begin(W, X, a.nseg, ksteps, 0, steps, lds);
        }
        head_results<TL, DZ, PARTS>(a, acc, rows, m, n, part);
        if (t >= end) return;
    }
}

// ---- rows: statistics of the tiles -> lse, listed logits, loss -----------------------------------------------------------------
struct RowArgs {
    const void *x, *w;
    int64_t n, v;
    int d, k;
    const float2 *stats;
    int64_t tiles;
    const int64_t *ids;          // [n][k]
    const float *logits;         // [n][k], NULL: cross entropy (k = 1)
    int64_t ignore;              // cross entropy: the label that is left out; distillation leaves out every id < 0
    float temperature;
    float *loss, *lse, *q, *zt;  // [n], [2][n], [n][k] (NULL: cross entropy), [n][k] (NULL likewise)
    int *status;                 // counts ids outside [0, v); may be NULL
};

// G dot products of row x with G rows of w by one wave: lane l gets number (l >> 3) & 7 of them.  The eight sums are folded
// together, so that they cost 10 exchanges instead of 48.
constexpr int G = 8;
template <int E> struct Words { using type = u32x4; };
template <> struct Words<8> { using type = __attribute__((ext_vector_type(2))) unsigned; };
template <> struct Words<4> { using type = unsigned; };
template <int DT, int BYTES>
__device__ __forceinline__ float dots(const void *x, const void *w, int64_t xo, const int64_t (&wo)[G], int d)
{
    constexpr int E = BYTES / (DT == T_F32 ? 4 : 2);
    using V = typename Words<BYTES>::type;
    const int lane = threadIdx.x & 63;
    float s[G];
#pragma unroll
    for (int j = 0; j < G; ++j) s[j] = 0.0f;
    int i = lane * E;
    for (; i + E <= d; i += 64 * E) {
        const V a = load_at<V, DT>(x, xo + i);
        V b[G];
#pragma unroll
        for (int j = 0; j < G; ++j) b[j] = load_at<V, DT>(w, wo[j] + i);
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) s[j] = fmaf(load1<DT>(&a, e), load1<DT>(&b[j], e), s[j]);
    }
    i = d / E * E + lane;
    if (E > 1 && i < d) {
        const float a = load1<DT>(x, xo + i);
#pragma unroll
        for (int j = 0; j < G; ++j) s[j] = fmaf(a, load1<DT>(w, wo[j] + i), s[j]);
    }
#pragma unroll
    for (int o = 32, m = G / 2; m >= 1; o >>= 1, m >>= 1)
#pragma unroll
        for (int j = 0; j < m; ++j) {
            const bool up = lane & o;
            s[j] = (up ? s[j + m] : s[j]) + __shfl_xor(up ? s[j] : s[j + m], o, 64);
        }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) s[0] += __shfl_xor(s[0], o, 64);
    return s[0];
}

// one dot product by one wave
template <int DT, int BYTES>
__device__ __forceinline__ float dot(const void *x, const void *w, int64_t xo, int64_t wo, int d)
{
    constexpr int E = BYTES / (DT == T_F32 ? 4 : 2);
    using V = typename Words<BYTES>::type;
    const int lane = threadIdx.x & 63;
    float s = 0.0f;
    int i = lane * E;
    for (; i + E <= d; i += 64 * E) {
        const V a = load_at<V, DT>(x, xo + i), b = load_at<V, DT>(w, wo + i);
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(load1<DT>(&a, e), load1<DT>(&b, e), s);
    }
    i = d / E * E + lane;
    if (E > 1 && i < d) s = fmaf(load1<DT>(x, xo + i), load1<DT>(w, wo + i), s);
    return wave_sum(s);
}

// LR rows per workgroup (4; 1 where a teacher's rows are few).  The tiles' statistics are read with rows running
// fastest, then each wave takes whole rows (1 row: its waves share the listed classes).
template <int DT, int BYTES, int LR>
__global__ void __launch_bounds__(256) rows_kernel(RowArgs a)
{
    __shared__ float2 st[256];
    __shared__ float part[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r0 = (int64_t)blockIdx.x * LR;
    const int rr = LR == 1 ? 0 : wave;
    const int64_t r = r0 + rr;
    const bool there = r < a.n;                     // (LR 1: always)
    const float inv_t = 1.0f / a.temperature, c = LOG2E * inv_t;
    // the statistics are on their way while the first class's logit is computed
    const int sr = tid % LR;
    int64_t t = tid / LR;
    const int64_t stat_rows = r0 + sr < a.n ? a.tiles : 0;
    float2 s = t < stat_rows ? a.stats[t * a.n + r0 + sr] : float2{-__builtin_inff(), 0.0f};
    const int64_t first = there ? a.ids[r * a.k] : -1;
    const bool pivot = first >= 0 && first < a.v && (a.logits != nullptr || first != a.ignore);
    const float zp = pivot ? dot<DT, BYTES>(a.x, a.w, r * a.d, first * a.d, a.d) : 0.0f;
    for (t += 256 / LR; t < stat_rows; t += 256 / LR) s = join_stats(s, a.stats[t * a.n + r0 + sr]);
    st[tid] = s;
    __syncthreads();
    for (int o = 128; o >= LR; o >>= 1) {
        if (tid < o) st[tid] = join_stats(st[tid], st[tid + o]);
        __syncthreads();
    }
    if (!there) return;
    // lse = ref + over in powers of two, kept apart: with a first class, over = log(1 + what is smaller, it or the others)
    const float rest = st[rr].x + __builtin_amdgcn_logf(st[rr].y);    // v_log_f32: base 2
    const float u = zp * c - rest, near = __builtin_amdgcn_exp2f(-fabsf(u));
    const float ref = pivot ? fmaxf(zp * c, rest) : st[rr].x;
    const float over = pivot ? log1pf(near) * LOG2E : __builtin_amdgcn_logf(st[rr].y);
    const float miss = pivot ? 1.0f / (1.0f + __builtin_amdgcn_exp2f(u)) : 1.0f;
    float lse = ref + over;
    if (!(fabsf(lse) < __builtin_inff())) lse = __builtin_nanf("");   // (+inf means something else)
    float loss = 0.0f;
    bool alive = false, bad = false;
    if (a.logits == nullptr) {
        bad = first != a.ignore && !pivot;
        alive = pivot;
        if (alive) loss = ((ref - zp * c) + over) * LN2 + (lse - lse);
    } else {
        const int64_t *ids = a.ids + r * a.k;
        const float *lg = a.logits + r * a.k;
        float *q = a.q + r * a.k, *zt = a.zt + r * a.k;
        float tm = -__builtin_inff();
        bool nan = false;
        for (int k = lane; k < a.k; k += 64) {
            if (ids[k] < 0) continue;           // (whatever its logit holds)
            bad |= ids[k] >= a.v;
            nan |= lg[k] != lg[k];
            tm = fmaxf(tm, lg[k]);
        }
        tm = wave_max(tm);
        bad = __any(bad);
        alive = (tm > -__builtin_inff() || __any(nan)) && !bad;
        float sum = 0.0f;
        if (alive)
            for (int k = lane; k < a.k; k += 64)
                if (ids[k] >= 0) sum += expf((lg[k] - tm) * inv_t);   // (the difference first: logits at the type's ends)
        sum = wave_sum(sum);
        const float ls = logf(sum);
        int listed = 0;                                               // of 64 entries; for an absent one a class that is there
        for (int k0 = LR == 1 ? wave * G : 0; k0 < a.k; k0 += LR == 1 ? 4 * G : G) {
            if ((k0 & 63) < (LR == 1 ? 4 * G : G)) {
                const int k = (k0 & ~63) + lane;
                const int64_t id = k < a.k ? ids[k] : -1;
                listed = alive && id >= 0 ? (int)id : 0;
            }
            int64_t wo[G];
#pragma unroll
            for (int j = 0; j < G; ++j) wo[j] = (int64_t)__builtin_amdgcn_readlane(listed, (k0 & 63) + j) * a.d;
            float z = alive ? dots<DT, BYTES>(a.x, a.w, r * a.d, wo, a.d) : 0.0f;
            const int k = k0 + ((lane >> 3) & 7);
            if (k < a.k && (lane & 7) == 0) {
                float qk = 0.0f;
                if (alive && ids[k] >= 0) {
                    if (ids[k] == first) z = zp;
                    const float lq = (lg[k] - tm) * inv_t - ls;
                    qk = expf(lq);
                    if (!(qk == 0.0f)) loss += qk * (lq + ((ref - z * c) + over) * LN2) + (lse - lse);
                } else {
                    z = 0.0f;
                }
                q[k] = qk;
                zt[k] = z;
            }
        }
        loss = wave_sum(loss);
        if (LR == 1) {
            if (lane == 0) part[wave] = loss;
            __syncthreads();
            loss = (part[0] + part[1]) + (part[2] + part[3]);
            if (wave != 0) return;
        }
        loss *= a.temperature * a.temperature;
    }
    if (lane == 0) {
        if (bad) loss = __builtin_nanf("");
        if (bad && a.status != nullptr) atomicAdd(a.status, 1);
        a.loss[r] = loss;
        a.lse[r] = alive ? lse : __builtin_inff();
        a.lse[a.n + r] = miss;
    }
}

// sum of the rows' losses (and their number) in a fixed order: one block
__global__ void __launch_bounds__(1024) sum_kernel(const float *__restrict__ loss, const float *__restrict__ lse, int64_t n, int mean,
                                                   float *__restrict__ out, float *__restrict__ count)
{
    __shared__ double sl[16];
    __shared__ double sc[16];
    double l = 0.0, c = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        l += (double)loss[i];
        c += (lse[i] != __builtin_inff() || loss[i] != loss[i]) ? 1.0 : 0.0;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { l += __shfl_xor(l, o, 64); c += __shfl_xor(c, o, 64); }
    if ((threadIdx.x & 63) == 0) { sl[threadIdx.x >> 6] = l; sc[threadIdx.x >> 6] = c; }
    __syncthreads();
    if (threadIdx.x == 0) {
        l = c = 0.0;
        for (int i = 0; i < 16; ++i) { l += sl[i]; c += sc[i]; }
        c = c > 1.0 ? c : 1.0;
        out[0] = (float)(mean ? l / c : l);
        if (count != nullptr) count[0] = (float)c;
    }
}

// The listed classes' entries of dz: p - (sum of the q of that class in this row); a class listed twice is written twice alike.  The first
// class of a row that is sure of it: (1 - q) - (1 - p).
// One wave per row, its entries 64 at a time in the lanes.
template <bool F16, int PARTS>
__global__ void __launch_bounds__(256) listed_kernel(const int64_t *__restrict__ ids, const float *__restrict__ q,
                                                     const float *__restrict__ zt, const float *__restrict__ lse,
                                                     const float *__restrict__ weight, const float *__restrict__ top, int64_t n, int k,
                                                     float c, int64_t v0, int64_t vc, int64_t n_pad, unsigned short *__restrict__ dz)
{
    const int lane = threadIdx.x & 63;
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= n) return;
    const float l = lse[r], miss = lse[n + r];
    const int64_t first = ids[r * k];
    if (l == __builtin_inff()) return;
    const float f = weight[r] / top[0] * (F16 ? F16_DZ : 1.0f);
    for (int k0 = 0; k0 < k; k0 += 64) {
        const int i = k0 + lane;
        const int64_t id = i < k ? ids[r * k + i] : -1;
        float s = 0.0f;
        for (int j0 = 0; j0 < k; j0 += 64) {
            const int64_t jd = j0 == k0 ? id : (j0 + lane < k ? ids[r * k + j0 + lane] : -1);
            const float jq = j0 + lane < k ? q[r * k + j0 + lane] : 0.0f;
            const int here = k - j0 < 64 ? k - j0 : 64;
            for (int j = 0; j < here; ++j) {        // (ids of this head fit 32 bits; absent ones match nothing that is written)
                const float t = __shfl(jq, j, 64);
                s += __shfl((int)jd, j, 64) == (int)id ? t : 0.0f;
            }
        }
        if (id < v0 || id >= v0 + vc || s == 0.0f) continue;
        const float pq = id == first && miss < 0.5f ? (1.0f - s) - miss : __builtin_amdgcn_exp2f(zt[r * k + i] * c - l) - s;
        const float p = f != 0.0f ? pq * f : 0.0f;
        unsigned short h[3];
        if (PARTS == 3) split3(p, h);
        else h[0] = to16<F16>(p);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) dz[(part * n_pad + r) * vc + id - v0] = h[part];
    }
}

// ---- products with dz: out[n][m] = sum_k A(k, m) B(n, k), A by columns ---------------------------------------------------------
// split over k; partial sums to `part` [split][rows][ldp] (+= with `add`), or, unsplit, the result itself
struct ProdArgs {
    Operand a, b;
    int64_t rows;                // n side
    int d;                       // m side
    int nseg;
    int64_t depth;               // K: the last step may reach beyond it, into zeros of dz
    int64_t tiles_m, tiles, splits;
    float *part;
    int64_t ldp, part_stride;
    int add;
    void *out;                   // part == NULL: [rows][d]
    const float *top;
    float scale;
};

template <class TL, int DT>
__device__ __forceinline__ void product(const ProdArgs &a, int64_t job, unsigned char *lds)
{
    const int64_t sp = job / a.tiles, t = job % a.tiles;
    const int64_t tm = t % a.tiles_m, tn = t / a.tiles_m;
    const int64_t m0 = tm * TL::BM, n0 = tn * TL::BN;
    const int64_t ksteps = (a.depth + TL::KD - 1) / TL::KD, steps = a.nseg * ksteps;
    const int64_t s0 = steps * sp / a.splits, s1 = steps * (sp + 1) / a.splits;
    Operand A = a.a, B = a.b;
    A.base += m0;
    A.lim = (int)((A.ld - m0) / 8 - 1);
    if (TL::BCOLS) {
        B.base += n0;
        B.lim = (int)((B.ld - n0) / 8 - 1);
    } else {
        B.base += n0 * B.ld;
        B.lim = TL::BN - 1;                     // (rows are padded to whole tiles)
    }
    typename TL::Acc acc;
#pragma unroll
    for (int i = 0; i < TL::MT; ++i)
#pragma unroll
        for (int j = 0; j < TL::NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    TL::run(acc, A, B, a.nseg, ksteps, s0, s1, lds);

    const float f = a.part == nullptr ? a.top[0] * a.scale : 1.0f;
#pragma unroll
    for (int nt = 0; nt < TL::NT; ++nt) {
        const int64_t n = n0 + TL::n_of(nt);
        if (n >= a.rows) continue;
#pragma unroll
        for (int b = 0; b < TL::MT / 4; ++b) {
            const int64_t m = m0 + TL::m_of(b);
            if (a.part != nullptr) {
                if (m >= a.ldp) continue;       // ldp is a multiple of 16
                float4 *p = (float4 *)(a.part + sp * a.part_stride + n * a.ldp + m);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 r = TL::quad(acc, b, j, nt);
                    float4 v = {r[0], r[1], r[2], r[3]};
                    if (a.add) {
                        const float4 o = p[j];
                        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
                    }
                    p[j] = v;
                }
                continue;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t at = m + 8 * h, to = n * a.d + at;
                if (at >= a.d) continue;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = TL::quad(acc, b, 2 * h + (e >> 2), nt)[e & 3] * f;
                if (at + 8 > a.d) {
#pragma unroll
                    for (int e = 0; e < 7; ++e)
                        if (at + e < a.d) store1<DT>(a.out, to + e, v[e]);
                } else if (DT == T_F32) {
                    store_at<DT>(a.out, to, f32x4{v[0], v[1], v[2], v[3]});
                    store_at<DT>(a.out, to + 4, f32x4{v[4], v[5], v[6], v[7]});
                } else {
                    unsigned short u[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) u[e] = to16<DT == T_F16>(v[e]);
                    store_at<DT>(a.out, to, *(const u32x4 *)u);
                }
            }
        }
    }
}

// dw of a piece (TW) and its share of dx (TX) in one launch: together they fill the chip with workgroups of about the same number
// of steps (4096 x 32768 x 512 bf16: 137 us a piece of 16384 classes), and dz is read by both while it is in the last-level cache
template <class TW, class TX, int DT>
__global__ void __launch_bounds__(TW::THREADS, TW::OCCUPANCY) products_kernel(ProdArgs w, ProdArgs x, int x_first)
{
    static_assert(TW::LDS == TX::LDS && TW::THREADS == TX::THREADS, "one workgroup shape");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[TW::LDS];
    // each XCD: a contiguous eighth of either list, the longer jobs first
    const int64_t xcd = blockIdx.x & 7;
    const int64_t jobs_w = w.tiles * w.splits, jobs_x = x.tiles * x.splits, per_w = (jobs_w + 7) / 8, per_x = (jobs_x + 7) / 8;
    int64_t i = blockIdx.x >> 3;
    const bool is_x = x_first ? i < per_x : i >= per_w;
    if (x_first ? !is_x : is_x) i -= x_first ? per_x : per_w;
    if (is_x) {
        if (i < per_x && xcd * per_x + i < jobs_x) product<TX, DT>(x, xcd * per_x + i, lds);
    } else {
        if (i < per_w && xcd * per_w + i < jobs_w) product<TW, DT>(w, xcd * per_w + i, lds);
    }
}

// out[r][c] = (sum over the splits) * top * scale, for up to two results; rows of weight 0 (weight may be NULL: none) are zero
struct Join {
    const float *part;
    int64_t part_stride, rows;
    int splits;
    const float *weight;
    void *out;
};
template <int DT>
__global__ void __launch_bounds__(256) join_kernel(Join ja, Join jb, int d, int64_t ldp, const float *__restrict__ top, float scale)
{
    const int per = (int)(ldp / 4);
    const int64_t first = ja.rows * per, total = first + jb.rows * per;
    const float g = top[0] * scale;
    for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < total; j += (int64_t)gridDim.x * 256) {
        const bool second = j >= first;
        const Join &a = second ? jb : ja;
        const int64_t i = second ? j - first : j, r = i / per;
        const int c = (int)(i % per) * 4;
        if (c >= d) continue;
        float4 s = {0.f, 0.f, 0.f, 0.f};
        if (a.weight == nullptr || a.weight[r] != 0.0f) {
            const float *p = a.part + r * ldp + c;
#pragma unroll 4
            for (int k = 0; k < a.splits; ++k) {
                const float4 v = *(const float4 *)(p + k * a.part_stride);
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
        }
        const float v[4] = {s.x * g, s.y * g, s.z * g, s.w * g};
        if (c + 4 > d) {
            for (int e = 0; e < 3; ++e)
                if (c + e < d) store1<DT>(a.out, r * d + c + e, v[e]);
        } else if (DT == T_F32) {
            store_at<DT>(a.out, r * d + c, f32x4{v[0], v[1], v[2], v[3]});
        } else {
            unsigned short u[4];
            for (int e = 0; e < 4; ++e) u[e] = to16<DT == T_F16>(v[e]);
            store_at<DT>(a.out, r * d + c, *(const unsigned long long *)u);
        }
    }
}

// ---- host: sizes, workspace, launches -----------------------------------------------------------------------------------------
int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

struct Plan {
    int sbm;                         // classes of a forward tile
    bool quarter_fwd, quarter_bwd;   // z by 128 x 128 tiles
    int64_t n, v, n_pad, vf, vc;     // vf, vc: classes of a piece, forward and backward (whole piece stride)
    int d, dp, parts, dtype;
    bool direct;                     // operands are read where they are
    bool small;                      // few rows: tiles of 32 rows
    int bm;                          // the products' tiles are bm x bm
    int split_dx, split_dw;
    bool x_first;                    // the jobs of dx are the longer ones
};

// Tiles of z: 256 x 256, one per CU, or 128 x 128, two per CU.  Estimated us of a launch from what steps (64 deep) and results of a
// tile took (dz writes its results too): the large ones come in whole rounds, the small ones fill the last one better (1000 x 20000 x
// 256 bf16: forward 18.4 against 22.9 us with large ones, backward 24.6 and 30.5; 1000 x 3000 x 100 fp32 11.2 and 21.4; but 4096 x
// 4096 x 256 fp32 57.5 and 40.8).
struct Tiling { bool quarter; double us; };
Tiling tiling(int64_t n, int64_t classes, int64_t steps, int dz_parts)
{
    const int64_t large = (n + 255) / 256 * ((classes + 255) / 256), small = (n + 127) / 128 * ((classes + 127) / 128);
    const double t256 = (double)((large + CUS - 1) / CUS) * (1.4 * steps + 5.0 + 5.0 * dz_parts);
    const double t128 = small <= CUS ? 0.7 * steps + 2.5 + 2.0 * dz_parts
                                     : (small <= 2 * CUS ? 1.0 : small / (2.0 * CUS) + 0.5) * (0.9 * steps + 2.5 + 2.0 * dz_parts);
    return Tiling{t128 < t256, t128 < t256 ? t128 : t256};
}

Plan make_plan(int64_t n, int64_t v, int d, int dtype)
{
    Plan p;
    p.n = n; p.v = v; p.d = d; p.dtype = dtype;
    p.parts = dtype == T_F32 ? 3 : 1;
    p.dp = (int)up(d, 64);
    p.direct = dtype != T_F32 && d % 8 == 0;      // (16 x 65536 x 512 bf16: 19 us; packed first 41; 4096 x 32768 x 512 + gradients 612 and 637)
    p.n_pad = up(n, 256);
    p.small = n <= 32;                            // (32 x 65536 x 512 bf16: tiles and rows 19.5 us, with 128 x 128 tiles 22.4)
    int64_t most = DZ_BYTES / (p.n_pad * 2 * p.parts), packed = WPACK_BYTES / ((int64_t)p.dp * 2 * p.parts) / 256 * 256;
    if (packed < 256) packed = 256;
    if (!p.direct && packed < most) most = packed;
    most = most / 256 * 256;
    if (most < 256) most = 256;
    // forward: nothing is kept of a piece but the packed codes; direct, one launch takes them all (bounded by the grid)
    p.vf = p.direct ? 256ll * ((1ll << 22) / ((n + 31) / 32)) : packed;
    if (p.vf < 256) p.vf = 256;
    p.vf = p.vf < up(v, 256) ? p.vf : up(v, 256);
    const int64_t steps = (int64_t)(p.parts == 3 ? 6 : 1) * (p.dp / 64);
    p.quarter_fwd = tiling(n, p.vf < v ? p.vf : v, steps, 0).quarter;
    // backward: as few pieces as fit, or more where their tiles come in whole rounds (PIECE us: the launches around a piece).  With gradients,
    // against as few as fit: 3000 x 131000 x 256 bf16 1050 and 1109 us, 1644 x 72779 x 176 fp32 1452 and 1486, 7000 x 70000 x 64 fp16 879 and 906
    const int64_t blocks = (v + 255) / 256, fewest = (v + most - 1) / most;
    double least = 0.0;
    for (int64_t pieces = fewest; pieces <= 2 * fewest && pieces <= fewest + 32; ++pieces) {
        const int64_t each = (blocks + pieces - 1) / pieces;
        const Tiling t = tiling(n, each * 256 < v ? each * 256 : v, steps, p.parts);
        const double us = (double)((blocks + each - 1) / each) * (t.us + PIECE);
        if (least == 0.0 || us < least) {
            least = us;
            p.vc = each * 256;
            p.quarter_bwd = t.quarter;
        }
    }
    p.sbm = p.quarter_fwd && !p.small ? 128 : 256;
    // The products of a piece are cut over k into jobs of about `job` steps (64 deep), by tiles of 256 x 256 (one per CU) or
    // 128 x 128 (two); what has the least estimated time is taken.  In us: a job's steps and its own cost (its first
    // requests, its results), what the partial sums cost to write and read again, and for more jobs than the chip holds
    // at once their average plus half a long one.
    double best = 0.0;
    for (int bm = 128; bm <= 256; bm *= 2) {
        const int64_t tm = (p.dp + bm - 1) / bm, seg = p.parts == 3 ? 6 : 1;
        const int64_t tiles_w = tm * ((p.vc + bm - 1) / bm), tiles_x = tm * ((n + bm - 1) / bm);
        const int64_t steps_w = seg * (up(n, 64) / 64), steps_x = seg * (p.vc / 64);
        const int64_t slots = bm == 256 ? CUS : 2 * CUS;
        const double step = bm == 256 ? STEP_256 : STEP_128;
        for (int64_t job = 4;; job += job / 4 + 1) {
            auto cut = [&](int64_t steps) {
                const int64_t s = (steps + job - 1) / job;
                return s < 1 ? (int64_t)1 : (s > 64 ? (int64_t)64 : s);
            };
            const int64_t sw = cut(steps_w), sx = cut(steps_x);
            const double lw = (double)((steps_w + sw - 1) / sw) + JOB_STEPS, lx = (double)((steps_x + sx - 1) / sx) + JOB_STEPS;
            const double jobs = (double)(tiles_w * sw + tiles_x * sx), all = tiles_w * sw * lw + tiles_x * sx * lx;
            const double longest = lw > lx ? lw : lx;
            double t = jobs <= slots ? longest : all / slots + longest / 2;
            t = (t > longest ? t : longest) * step;
            t += 8.0 * p.dp * (double)(sx * n + (sw > 1 ? sw * p.vc : 0)) / 6.4e6;
            if (best == 0.0 || t < best) {
                best = t;
                p.bm = bm;
                p.split_dw = (int)sw;
                p.split_dx = (int)sx;
                p.x_first = lx > lw;
            }
            if (sw == 1 && sx == 1) break;
        }
    }
    return p;
}

struct Space {          // hands out 256-byte aligned ranges; with base == NULL only counts
    unsigned char *base;
    int64_t at = 0;
    void *take(int64_t bytes)
    {
        void *r = base != nullptr ? base + at : nullptr;
        at = up(at + bytes, 256);
        return r;
    }
};

struct FwdSpace { unsigned short *xp, *wp; float2 *stats; float *loss; };
struct BwdSpace { unsigned short *xs, *wp, *dz; float *dxp, *dwp, *weight, *top; };

FwdSpace fwd_space(const Plan &p, Space &s)
{
    FwdSpace f;
    f.xp = p.direct ? nullptr : (unsigned short *)s.take(p.n_pad * p.dp * 2 * p.parts);
    f.wp = p.direct ? nullptr : (unsigned short *)s.take(p.vf * p.dp * 2 * p.parts);
    f.stats = (float2 *)s.take((p.v + p.sbm - 1) / p.sbm * p.n * 8);
    f.loss = (float *)s.take(p.n * 4);
    return f;
}
BwdSpace bwd_space(const Plan &p, Space &s, bool dx, bool dw)
{
    BwdSpace b;
    b.weight = (float *)s.take(p.n * 4);
    b.top = (float *)s.take(4);
    b.wp = p.direct ? nullptr : (unsigned short *)s.take(p.vc * p.dp * 2 * p.parts);
    b.xs = dw || !p.direct ? (unsigned short *)s.take(p.n_pad * p.dp * 2 * p.parts) : nullptr;
    b.dz = (unsigned short *)s.take(p.n_pad * p.vc * 2 * p.parts);
    b.dxp = dx ? (float *)s.take(p.split_dx * p.n * (int64_t)p.dp * 4) : nullptr;
    b.dwp = dw && p.split_dw > 1 ? (float *)s.take(p.split_dw * p.vc * (int64_t)p.dp * 4) : nullptr;
    return b;
}

void prep(int dtype, const PrepArgs &a, hipStream_t st)
{
    int64_t g = (a.chunks[0] + a.chunks[1] + PREP - 1) / PREP;
    g = (g > 4 * CUS ? 4 * CUS : g) + (a.weight != nullptr);
    if (g == 0) return;
    if (dtype == T_F32) prep_kernel<T_F32><<<(unsigned)g, PREP, 0, st>>>(a);
    else if (dtype == T_BF16) prep_kernel<T_BF16><<<(unsigned)g, PREP, 0, st>>>(a);
    else prep_kernel<T_F16><<<(unsigned)g, PREP, 0, st>>>(a);
}
void add_pack(PrepArgs &a, int i, const void *src, int64_t rows, int64_t rows_pad, unsigned short *dst)
{
    a.p[i] = Pack{src, rows, rows_pad, dst};
    a.chunks[i] = rows_pad * (a.dp / 8);
}

template <class TL, bool DZ, int PARTS>
void launch_head(HeadArgs a, hipStream_t st)
{
    // dz: the products read whole blocks of 256 rows and classes, so the tiles beyond the last ones write zeros
    a.tiles_n = ((DZ ? a.n_pad : a.n) + TL::BN - 1) / TL::BN;
    a.tiles = ((DZ ? up(a.vc, 256) : a.vc) + TL::BM - 1) / TL::BM * a.tiles_n;
    head_kernel<TL, DZ, PARTS><<<(unsigned)up(a.tiles, 8), TL::THREADS, 0, st>>>(a);
}
template <class TL, bool DZ, int PARTS>
void launch_head_walk(HeadArgs a, hipStream_t st)
{
    a.tiles_n = (a.n + TL::BN - 1) / TL::BN;        // (dz: n_pad / BN, the padding rows are written too)
    a.tiles = (a.vc + TL::BM - 1) / TL::BM * a.tiles_n;
    const int64_t g = up(a.tiles, 8);
    head_walk_kernel<TL, DZ, PARTS><<<(unsigned)(g < CUS ? g : CUS), TL::THREADS, 0, st>>>(a);
}

template <bool DZ, bool F16, int PARTS>
void head_of(const Plan &p, const HeadArgs &a, hipStream_t st)
{
    // (four stages of the small tile: 1 x 32768 x 512 bf16 8.4 us, three 9.6, seven with one workgroup per CU 10.2)
    if (!DZ && p.small) launch_head<Tile<256, 32, 4, 1, false, false, F16, 4>, false, PARTS>(a, st);
    else if (DZ ? p.quarter_bwd : p.quarter_fwd) launch_head<Tile<128, 128, 2, 2, false, false, F16>, DZ, PARTS>(a, st);
    else launch_head_walk<DuoTile<256, 256, 2, 4, false, false, F16>, DZ, PARTS>(a, st);
}
template <bool DZ>
void head(const Plan &p, const HeadArgs &a, hipStream_t st)
{
    if (p.dtype == T_F16) head_of<DZ, true, 1>(p, a, st);
    else if (p.dtype == T_BF16) head_of<DZ, false, 1>(p, a, st);
    else head_of<DZ, false, 3>(p, a, st);
}

template <class TW, class TX>
void launch_products(const Plan &p, ProdArgs w, ProdArgs x, hipStream_t st)
{
    w.tiles_m = x.tiles_m = (p.dp + TW::BM - 1) / TW::BM;
    w.tiles = w.rows > 0 ? w.tiles_m * ((w.rows + TW::BN - 1) / TW::BN) : 0;
    x.tiles = x.rows > 0 ? x.tiles_m * ((x.rows + TX::BN - 1) / TX::BN) : 0;
    const unsigned g = (unsigned)(8 * ((w.tiles * w.splits + 7) / 8 + (x.tiles * x.splits + 7) / 8));
    if (p.dtype == T_F32) products_kernel<TW, TX, T_F32><<<g, TW::THREADS, 0, st>>>(w, x, p.x_first);
    else if (TW::F16) products_kernel<TW, TX, T_F16><<<g, TW::THREADS, 0, st>>>(w, x, p.x_first);
    else products_kernel<TW, TX, T_BF16><<<g, TW::THREADS, 0, st>>>(w, x, p.x_first);
}
template <bool F16>
void products_of(const Plan &p, const ProdArgs &w, const ProdArgs &x, hipStream_t st)
{
    if (p.bm == 128) launch_products<Tile<128, 128, 2, 2, true, true, F16>, Tile<128, 128, 2, 2, true, false, F16>>(p, w, x, st);
    else launch_products<DuoTile<256, 256, 2, 4, true, true, F16>, DuoTile<256, 256, 2, 4, true, false, F16>>(p, w, x, st);
}
void products(const Plan &p, const ProdArgs &w, const ProdArgs &x, hipStream_t st)
{
    if (p.dtype == T_F16) products_of<true>(p, w, x, st);
    else products_of<false>(p, w, x, st);
}

void join(const Plan &p, const Join &a, const Join &b, const float *top, float scale, hipStream_t st)
{
    const int64_t items = (a.rows + b.rows) * (p.dp / 4);
    if (items == 0) return;
    const int64_t blocks = (items + 255) / 256;
    const unsigned g = (unsigned)(blocks > 8192 ? 8192 : blocks);
    if (p.dtype == T_F32) join_kernel<T_F32><<<g, 256, 0, st>>>(a, b, p.d, p.dp, top, scale);
    else if (p.dtype == T_BF16) join_kernel<T_BF16><<<g, 256, 0, st>>>(a, b, p.d, p.dp, top, scale);
    else join_kernel<T_F16><<<g, 256, 0, st>>>(a, b, p.d, p.dp, top, scale);
}

template <int DT, int BYTES>
void launch_rows(const RowArgs &r, hipStream_t st)
{
    // a teacher's classes are shared by the waves of a workgroup where whole rows would leave the chip idle (us shared / by rows: 16 x 512 with
    // 64 classes 13 / 39, 855 x 122 with 110 20 / 38, 2000 x 256 with 64 23 / 28 and with 8 12.8 / 7.4, 4096 x 512 with 32 43 / 32)
    const bool share = r.logits != nullptr && r.n < (r.k > 16 ? 16 : 2) * CUS;
    if (share) rows_kernel<DT, BYTES, 1><<<(unsigned)r.n, 256, 0, st>>>(r);
    else rows_kernel<DT, BYTES, 4><<<(unsigned)((r.n + 3) / 4), 256, 0, st>>>(r);
}
template <int DT>
void launch_rows_of(const RowArgs &r, hipStream_t st)
{
    // loads no wider than 64 lanes need for a row (855 x 122 fp16, 110 classes: 20 us, with 16-byte loads 23; 8192 x 64 bf16, 32: 32 and 39)
    const int need = (r.d + 63) / 64 * (DT == T_F32 ? 4 : 2);
    if (need > 8) launch_rows<DT, 16>(r, st);
    else if (need > 4) launch_rows<DT, 8>(r, st);
    else launch_rows<DT, 4>(r, st);
}
void rows_pass(int dtype, const RowArgs &r, hipStream_t st)
{
    if (dtype == T_F32) launch_rows_of<T_F32>(r, st);
    else if (dtype == T_BF16) launch_rows_of<T_BF16>(r, st);
    else launch_rows_of<T_F16>(r, st);
}

const char *bad_head(int64_t n, int64_t v, int d, int dtype, int k, const void *x, const void *w)
{
    if (dtype < T_F32 || dtype > T_F16) return "class head: dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)";
    if (n < 1 || v < 1 || n > (1 << 24) || v > (1 << 28)) return "class head: rows must be in [1, 2^24], classes in [1, 2^28]";
    if (d < 1 || d > (1 << 15)) return "class head: features must be in [1, 2^15]";
    if (k < 1 || k > 4096) return "class head: listed classes per row must be in [1, 4096]";
    if (((uintptr_t)x | (uintptr_t)w) & 15) return "class head: x and w must be 16-byte aligned";
    return nullptr;
}

// (k: valid elements of a row)
Operand rows_of(const void *p, int64_t plane, int64_t ld, int64_t k) { return Operand{(const unsigned short *)p, plane, ld, 0, (int)k}; }

const unsigned char *row_ptr(const void *p, int64_t row, int d, int dtype)
{
    return (const unsigned char *)p + row * d * (dtype == T_F32 ? 4 : 2);
}

}  // namespace

extern "C" {

int64_t rsdf_class_head_workspace_bytes(int64_t n, int64_t v, int d, int dtype, int pass)
{
    const char *bad = bad_head(n, v, d, dtype, 1, nullptr, nullptr);
    if (bad != nullptr) { rsdf_set_error(bad); return -1; }
    const Plan p = make_plan(n, v, d, dtype);
    Space s{nullptr};
    if (pass == 0) fwd_space(p, s);
    else bwd_space(p, s, pass & 1, pass & 2);
    return s.at;
}

int rsdf_class_head_plan(int64_t n, int64_t v, int d, int dtype, int32_t *plan)
{
    const char *bad = bad_head(n, v, d, dtype, 1, nullptr, nullptr);
    RSDF_CHECK_ARG(bad == nullptr, bad);
    RSDF_CHECK_ARG(plan != nullptr, "class_head_plan: plan must not be NULL");
    const Plan p = make_plan(n, v, d, dtype);
    const int32_t out[8] = {p.small ? 32 : (p.quarter_fwd ? 128 : 256), p.quarter_bwd ? 128 : 256, p.bm,
                            (int32_t)((v + p.vf - 1) / p.vf), (int32_t)((v + p.vc - 1) / p.vc), p.split_dw, p.split_dx, p.direct};
    for (int i = 0; i < 8; ++i) plan[i] = out[i];
    return 0;
}

int rsdf_class_head_fwd(const void *x, const void *w, int64_t n, int64_t v, int d, int dtype, const int64_t *ids,
                        const float *teacher_logits, int k, int64_t ignore_id, float temperature, int reduction, float *loss,
                        float *lse, float *count, float *q, float *listed_z, int32_t *bad_ids, void *workspace,
                        int64_t workspace_bytes, void *stream)
{
    const char *bad = bad_head(n, v, d, dtype, k, x, w);
    RSDF_CHECK_ARG(bad == nullptr, bad);
    RSDF_CHECK_ARG(temperature >= 0.999e-6f && temperature <= 1.001e6f, "class_head_fwd: temperature must be in [1e-6, 1e6]");
    RSDF_CHECK_ARG(teacher_logits != nullptr ? (q != nullptr && listed_z != nullptr) : k == 1,
                   "class_head_fwd: a teacher needs q and listed_z, labels need k = 1");
    RSDF_CHECK_ARG(reduction >= 0 && reduction <= 2, "class_head_fwd: reduction must be 0 (none), 1 (mean) or 2 (sum)");
    RSDF_CHECK_ARG(x != nullptr && w != nullptr && ids != nullptr && loss != nullptr && lse != nullptr && (count != nullptr || reduction != 1),
                   "class_head_fwd: x, w, ids, loss, lse, and for a mean count, must not be NULL");
    const Plan p = make_plan(n, v, d, dtype);
    Space s{(unsigned char *)workspace};
    const FwdSpace f = fwd_space(p, s);
    RSDF_CHECK_ARG(workspace != nullptr && s.at <= workspace_bytes, "class_head_fwd: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    const int64_t xplane = p.n_pad * p.dp, wplane = p.vf * p.dp;
    for (int64_t v0 = 0; v0 < v; v0 += p.vf) {
        const int64_t here = v - v0 < p.vf ? v - v0 : p.vf;
        HeadArgs a = {};
        if (!p.direct) {
            PrepArgs r = {};
            r.d = d; r.dp = p.dp;
            if (v0 == 0) add_pack(r, 0, x, n, p.n_pad, f.xp);
            add_pack(r, 1, row_ptr(w, v0, d, dtype), here, p.vf, f.wp);
            prep(dtype, r, st);
        }
        a.x = p.direct ? rows_of(x, 0, d, d) : rows_of(f.xp, xplane, p.dp, p.dp);
        a.w = p.direct ? rows_of(row_ptr(w, v0, d, dtype), 0, d, d) : rows_of(f.wp, wplane, p.dp, p.dp);
        a.n = n; a.vc = here;
        a.nseg = p.parts == 3 ? 6 : 1;
        a.depth = p.dp;
        a.c = LOG2E / temperature;
        a.stats = f.stats;
        a.tile0 = v0 / p.sbm;
        a.v0 = v0;
        a.label = ids; a.label_step = k;
        head<false>(p, a, st);
    }
    RowArgs r = {x, w, n, v, d, k, f.stats, (v + p.sbm - 1) / p.sbm, ids, teacher_logits, ignore_id, temperature,
                 reduction == 0 ? loss : f.loss, lse, q, listed_z, bad_ids};
    rows_pass(dtype, r, st);
    if (reduction != 0) sum_kernel<<<1, 1024, 0, st>>>(f.loss, lse, n, reduction == 1, loss, count);
    RSDF_RETURN_LAUNCH();
}

int rsdf_class_head_bwd(const void *x, const void *w, int64_t n, int64_t v, int d, int dtype, const int64_t *ids, const float *q,
                        const float *listed_z, int k, float temperature, const float *lse, const float *count, const float *grad,
                        int grad_per_row, void *dx, void *dw, void *workspace, int64_t workspace_bytes, void *stream)
{
    const char *bad = bad_head(n, v, d, dtype, k, x, w);
    RSDF_CHECK_ARG(bad == nullptr, bad);
    RSDF_CHECK_ARG((q == nullptr) == (listed_z == nullptr) && (q != nullptr || k == 1),
                   "class_head_bwd: a teacher needs q and listed_z, labels need k = 1");
    RSDF_CHECK_ARG(x != nullptr && w != nullptr && ids != nullptr && lse != nullptr && grad != nullptr,
                   "class_head_bwd: x, w, ids, lse and grad must not be NULL");
    RSDF_CHECK_ARG((((uintptr_t)dx | (uintptr_t)dw) & 15) == 0, "class_head_bwd: dx and dw must be 16-byte aligned");
    if (dx == nullptr && dw == nullptr) return 0;
    const Plan p = make_plan(n, v, d, dtype);
    Space s{(unsigned char *)workspace};
    const BwdSpace b = bwd_space(p, s, dx != nullptr, dw != nullptr);
    RSDF_CHECK_ARG(workspace != nullptr && s.at <= workspace_bytes, "class_head_bwd: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    const int nseg = p.parts == 3 ? 6 : 1;
    const int64_t xplane = p.n_pad * p.dp, wplane = p.vc * p.dp, zplane = p.n_pad * p.vc;
    const float scale = dtype == T_F16 ? 1.0f / F16_DZ : 1.0f;
    for (int64_t v0 = 0; v0 < v; v0 += p.vc) {
        const int64_t here = v - v0 < p.vc ? v - v0 : p.vc;
        HeadArgs a = {};
        if (v0 == 0 || !p.direct) {
            PrepArgs r = {};
            r.d = d; r.dp = p.dp;
            if (v0 == 0) {
                r.lse = lse; r.g = grad; r.count = count; r.g_per_row = grad_per_row;
                r.temperature = temperature; r.n = n;
                r.weight = b.weight; r.top = b.top;
                if (b.xs != nullptr) add_pack(r, 0, x, n, p.n_pad, b.xs);
            }
            if (!p.direct) add_pack(r, 1, row_ptr(w, v0, d, dtype), here, p.vc, b.wp);
            prep(dtype, r, st);
        }
        a.x = p.direct ? rows_of(x, 0, d, d) : rows_of(b.xs, xplane, p.dp, p.dp);
        a.w = p.direct ? rows_of(row_ptr(w, v0, d, dtype), 0, d, d) : rows_of(b.wp, wplane, p.dp, p.dp);
        a.n = n; a.n_pad = p.n_pad; a.vc = here; a.ldz = p.vc;
        a.nseg = nseg;
        a.depth = p.dp;
        a.c = LOG2E / temperature;
        a.lse = lse;
        a.weight = b.weight; a.top = b.top;
        a.label = q == nullptr ? ids : nullptr; a.label_step = 1;
        a.v0 = v0;
        a.dz = b.dz;
        head<true>(p, a, st);
        if (q != nullptr) {
            const unsigned g = (unsigned)((n + 3) / 4);
            if (dtype == T_F32) listed_kernel<false, 3><<<g, 256, 0, st>>>(ids, q, listed_z, lse, b.weight, b.top, n, k, a.c, v0, p.vc, p.n_pad, b.dz);
            else if (dtype == T_BF16) listed_kernel<false, 1><<<g, 256, 0, st>>>(ids, q, listed_z, lse, b.weight, b.top, n, k, a.c, v0, p.vc, p.n_pad, b.dz);
            else listed_kernel<true, 1><<<g, 256, 0, st>>>(ids, q, listed_z, lse, b.weight, b.top, n, k, a.c, v0, p.vc, p.n_pad, b.dz);
        }
        ProdArgs px = {}, pw = {};
        px.splits = pw.splits = 1;
        if (dx != nullptr) {
            px.a = a.w;
            px.a.k_rows = (int)(p.direct ? here : p.vc);
            px.b = rows_of(b.dz, zplane, p.vc, p.vc);
            px.rows = n; px.d = d; px.nseg = nseg;
            px.depth = here;
            px.splits = p.split_dx;
            px.part = b.dxp; px.ldp = p.dp; px.part_stride = n * p.dp; px.add = v0 > 0;
        }
        if (dw != nullptr) {
            pw.a = rows_of(b.xs, xplane, p.dp, p.dp);
            pw.a.k_rows = (int)p.n_pad;
            pw.b = rows_of(b.dz, zplane, p.vc, p.vc);
            pw.b.k_rows = (int)p.n_pad;
            pw.rows = here; pw.d = d; pw.nseg = nseg;
            pw.depth = n;
            pw.splits = p.split_dw;
            pw.part = b.dwp; pw.ldp = p.dp; pw.part_stride = p.vc * p.dp;
            pw.out = (unsigned char *)dw + v0 * d * (dtype == T_F32 ? 4 : 2);
            pw.top = b.top;
            pw.scale = scale;
        }
        products(p, pw, px, st);
        Join ja = {}, jb = {};
        if (b.dwp != nullptr) ja = Join{b.dwp, pw.part_stride, here, p.split_dw, nullptr, pw.out};
        if (dx != nullptr && v0 + p.vc >= v) jb = Join{b.dxp, n * p.dp, n, p.split_dx, b.weight, dx};
        join(p, ja, jb, b.top, scale, st);
    }
    RSDF_RETURN_LAUNCH();
}

}  // extern "C"
