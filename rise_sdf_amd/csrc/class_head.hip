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
// Forward: the tiles of z (256 classes x 128 rows) never leave the registers: each writes its rows' maximum and sum of
// exponentials, and one wave per row joins them and takes the logits of the K listed classes as K dot products.
// Backward, in pieces of the classes: the tiles are computed again and leave as 16-bit dz [rows][piece]; two products read it
// (dx over the piece, dw of the piece).  A piece is at most DZ_BYTES, so the memory does not grow with V.
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
constexpr int64_t DZ_BYTES = 256ll << 20;      // of one piece of dz
constexpr int64_t WPACK_BYTES = 128ll << 20;   // of the packed class codes of one piece

__device__ __forceinline__ float bf2f(unsigned short u) { return __builtin_bit_cast(float, (unsigned)u << 16); }
__device__ __forceinline__ float hf2f(unsigned short u) { return (float)__builtin_bit_cast(_Float16, u); }
__device__ __forceinline__ unsigned short f2bf(float f) { return __builtin_bit_cast(unsigned short, (__bf16)f); }
__device__ __forceinline__ unsigned short f2hf(float f) { return __builtin_bit_cast(unsigned short, (_Float16)f); }
template <bool F16> __device__ __forceinline__ unsigned short to16(float f) { return F16 ? f2hf(f) : f2bf(f); }

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

// ---- operands: [rows][d] of any type -> 16-bit parts [P][rows_pad][dp], zero padded -----------------------------------------
// weight (may be NULL): a row of weight 0 becomes zero whatever it holds
template <int DT>
__global__ void __launch_bounds__(256) pack_kernel(const void *__restrict__ src, int64_t rows, int d, int64_t rows_pad, int dp,
                                                   const float *__restrict__ weight, unsigned short *__restrict__ dst)
{
    const int per = dp / 8;
    const int64_t total = rows_pad * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per;
        const int c = (int)(i % per) * 8;
        const bool live = r < rows && (weight == nullptr || weight[r] != 0.0f);
        unsigned short o[3][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = 0.0f;
            if (live && c + e < d) v = load1<DT>(src, r * d + c + e);
            if (DT == T_F32) {
                unsigned short h[3];
                split3(v, h);
                o[0][e] = h[0]; o[1][e] = h[1]; o[2][e] = h[2];
            } else {
                o[0][e] = to16<DT == T_F16>(v);
            }
        }
#pragma unroll
        for (int p = 0; p < (DT == T_F32 ? 3 : 1); ++p) *(u32x4 *)(dst + (p * rows_pad + r) * dp + c) = *(const u32x4 *)o[p];
    }
}

// ---- z = x w^T by tiles: statistics, or dz ----------------------------------------------------------------------------------
struct HeadArgs {
    Operand w, x;                // base of the piece's first class / of row 0
    int64_t n, vc;               // rows, classes of the piece
    int nseg;
    int64_t ksteps;
    float c;                     // log2(e) / T
    int64_t tiles_n, tiles;
    // statistics
    float2 *stats;               // [class tile][n]: maximum and sum of 2^(c z - maximum)
    int64_t tile0;               // first class tile of the piece
    // dz
    const float *lse;            // [n] in powers of two; +inf: a row that takes part in nothing
    const float *weight, *top;   // [n], [1]
    const int64_t *label;        // [n] or NULL
    int64_t v0;
    unsigned short *dz;          // [parts][n_pad][ldz]
    int64_t n_pad, ldz;
};

template <class TL, bool DZ, int PARTS>
__global__ void __launch_bounds__(THREADS, 2) head_kernel(HeadArgs a)
{
    __shared__ __attribute__((aligned(1024))) unsigned char lds[TL::LDS];
    const int64_t t = xcd_tile(a.tiles);
    if (t < 0) return;
    const int64_t tm = t / a.tiles_n, tn = t % a.tiles_n;
    const int64_t m0 = tm * TL::BM, n0 = tn * TL::BN;
    Operand W = a.w, X = a.x;
    const bool rows_here = n0 < a.n;            // (dz: the tiles of padding rows only write zeros)
    W.base += m0 * W.ld;
    W.lim = (int)(a.vc - 1 - m0 < TL::BM - 1 ? a.vc - 1 - m0 : TL::BM - 1);
    if (rows_here) X.base += n0 * X.ld;
    X.lim = rows_here ? (int)(a.n - 1 - n0 < TL::BN - 1 ? a.n - 1 - n0 : TL::BN - 1) : 0;
    f32x4 acc[TL::MT][TL::NT];
#pragma unroll
    for (int i = 0; i < TL::MT; ++i)
#pragma unroll
        for (int j = 0; j < TL::NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    TL::run(acc, W, X, a.nseg, a.ksteps, 0, rows_here ? a.nseg * a.ksteps : 0, lds);

    const int64_t left = a.vc - m0;         // valid classes of this tile
    if (!DZ) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / TL::WN;
        float2 *part = (float2 *)lds;           // [WM][BN]
#pragma unroll
        for (int nt = 0; nt < TL::NT; ++nt) {
            float mx = -__builtin_inff();
#pragma unroll
            for (int mt = 0; mt < TL::MT; ++mt) {
                const int m = TL::m_of(mt >> 2) + (mt & 3) * 4;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float z = acc[mt][nt][r] * a.c;
                    z = m + r < left ? z : -__builtin_inff();
                    acc[mt][nt][r] = z;
                    mx = fmaxf(mx, z);
                }
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float ref = mx > -__builtin_inff() ? mx : 0.0f;
            float s = 0.0f;
#pragma unroll
            for (int mt = 0; mt < TL::MT; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f(acc[mt][nt][r] - ref);
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
            if (lane < 16) part[wm * TL::BN + TL::n_of(nt)] = float2{mx, s};
        }
        __syncthreads();
        for (int n = threadIdx.x; n < TL::BN; n += THREADS) {
            if (n0 + n >= a.n) continue;
            float2 p = part[n];
#pragma unroll
            for (int k = 1; k < TL::WM; ++k) p = join_stats(p, part[k * TL::BN + n]);
            a.stats[(a.tile0 + tm) * a.n + n0 + n] = p;
        }
    } else {
        constexpr bool F16 = TL::F16;
#pragma unroll
        for (int nt = 0; nt < TL::NT; ++nt) {
            const int64_t n = n0 + TL::n_of(nt);
            const float lse = n < a.n ? a.lse[n] : __builtin_inff();
            const bool live = lse != __builtin_inff();
            const float f = live ? a.weight[n] / a.top[0] * (F16 ? F16_DZ : 1.0f) : 0.0f;
            const int64_t label = (live && a.label != nullptr) ? a.label[n] - a.v0 - m0 : -1;
#pragma unroll
            for (int b = 0; b < TL::MT / 4; ++b) {
                const int m = TL::m_of(b);
                unsigned short o[PARTS][16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float p = __builtin_amdgcn_exp2f(acc[4 * b + (e >> 2)][nt][e & 3] * a.c - lse);
                    p = m + e == label ? p - 1.0f : p;
                    p = f != 0.0f && m + e < left ? p * f : 0.0f;
                    if (PARTS == 3) {
                        unsigned short h[3];
                        split3(p, h);
#pragma unroll
                        for (int k = 0; k < PARTS; ++k) o[k][e] = h[k];
                    } else {
                        o[0][e] = to16<F16>(p);
                    }
                }
#pragma unroll
                for (int k = 0; k < PARTS; ++k) {
                    u32x4 *d = (u32x4 *)(a.dz + (k * a.n_pad + n) * a.ldz + m0 + m);
                    d[0] = ((const u32x4 *)o[k])[0];
                    d[1] = ((const u32x4 *)o[k])[1];
                }
            }
        }
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
    float *loss, *lse, *q, *zt;  // [n], [n], [n][k] (NULL: cross entropy), [n][k] (NULL likewise)
    int *status;                 // counts ids outside [0, v); may be NULL
};

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

template <int DT>
__device__ __forceinline__ float dot_row(const void *x, const void *w, int64_t xo, int64_t wo, int d)
{
    float s = 0.0f;
    for (int i = threadIdx.x & 63; i < d; i += 64) s = fmaf(load1<DT>(x, xo + i), load1<DT>(w, wo + i), s);
    return wave_sum(s);
}

template <int DT>
__global__ void __launch_bounds__(256) rows_kernel(RowArgs a)
{
    const int lane = threadIdx.x & 63;
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= a.n) return;
    float2 st = {-__builtin_inff(), 0.0f};
    for (int64_t t = lane; t < a.tiles; t += 64) st = join_stats(st, a.stats[t * a.n + r]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) st = join_stats(st, float2{__shfl_xor(st.x, o, 64), __shfl_xor(st.y, o, 64)});
    const float lse = st.x + __builtin_amdgcn_logf(st.y);     // v_log_f32: base 2
    const float inv_t = 1.0f / a.temperature;
    float loss = 0.0f;
    bool alive = false, bad = false;
    if (a.logits == nullptr) {
        const int64_t id = a.ids[r];
        bad = id != a.ignore && (id < 0 || id >= a.v);
        alive = id != a.ignore && !bad;
        if (alive) loss = lse * LN2 - dot_row<DT>(a.x, a.w, r * a.d, id * a.d, a.d);
    } else {
        const int64_t *ids = a.ids + r * a.k;
        const float *lg = a.logits + r * a.k;
        float *q = a.q + r * a.k, *zt = a.zt + r * a.k;
        float tm = -__builtin_inff();
        bool nan = false;
        for (int k = lane; k < a.k; k += 64) {
            if (ids[k] < 0) continue;               // (whatever its logit holds)
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
                if (ids[k] >= 0) sum += expf((lg[k] - tm) * inv_t);     // (the difference first: logits at the type's ends)
        sum = wave_sum(sum);
        const float lse_e = lse * LN2, ls = logf(sum);
        for (int k = 0; k < a.k; ++k) {
            const int64_t id = ids[k];
            float qk = 0.0f, z = 0.0f;
            if (alive && id >= 0) {
                const float lq = (lg[k] - tm) * inv_t - ls;
                qk = expf(lq);
                z = dot_row<DT>(a.x, a.w, r * a.d, id * a.d, a.d);
                if (!(qk == 0.0f)) loss += qk * (lq - z * inv_t + lse_e);
            }
            if (lane == 0) { q[k] = qk; zt[k] = z; }
        }
        loss *= a.temperature * a.temperature;
    }
    if (lane != 0) return;
    if (bad) loss = __builtin_nanf("");
    if (bad && a.status != nullptr) atomicAdd(a.status, 1);
    a.loss[r] = loss;
    a.lse[r] = alive ? lse : __builtin_inff();
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
        count[0] = (float)c;
    }
}

// weight of a row in the gradient: T g_n (mean: / count), 0 where it takes part in nothing; top[0] = the largest |weight|
__global__ void __launch_bounds__(1024) weights_kernel(const float *__restrict__ lse, const float *__restrict__ g, int g_per_row,
                                                       const float *__restrict__ count, float temperature, int64_t n,
                                                       float *__restrict__ weight, float *__restrict__ top)
{
    __shared__ float sm[16];
    const float f = count != nullptr ? temperature / count[0] : temperature;
    float m = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        const float wr = lse[i] != __builtin_inff() ? g[g_per_row ? i : 0] * f : 0.0f;
        weight[i] = wr;
        m = fmaxf(m, fabsf(wr));
    }
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 0; i < 16; ++i) m = fmaxf(m, sm[i]);
        top[0] = m > 0.0f ? m : 1.0f;
    }
}

// the listed classes' entries of dz: p - (sum of the q of that class in this row); a class listed twice is written twice alike
template <bool F16, int PARTS>
__global__ void __launch_bounds__(256) listed_kernel(const int64_t *__restrict__ ids, const float *__restrict__ q,
                                                     const float *__restrict__ zt, const float *__restrict__ lse,
                                                     const float *__restrict__ weight, const float *__restrict__ top, int64_t n, int k,
                                                     float c, int64_t v0, int64_t vc, int64_t n_pad, unsigned short *__restrict__ dz)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n * k) return;
    const int64_t r = i / k, id = ids[i];
    const float l = lse[r];
    if (id < v0 || id >= v0 + vc || l == __builtin_inff()) return;
    float s = 0.0f;
    for (int j = 0; j < k; ++j) s += ids[r * k + j] == id ? q[r * k + j] : 0.0f;
    if (s == 0.0f) return;
    const float p = (__builtin_amdgcn_exp2f(zt[i] * c - l) - s) * (weight[r] / top[0] * (F16 ? F16_DZ : 1.0f));
    unsigned short h[3];
    if (PARTS == 3) split3(p, h);
    else h[0] = to16<F16>(p);
#pragma unroll
    for (int part = 0; part < PARTS; ++part) dz[(part * n_pad + r) * vc + id - v0] = h[part];
}

// ---- products with dz: out[n][m] = sum_k A(k, m) B(n, k), A by columns ---------------------------------------------------------
// split over k into gridDim.y ranges; partial sums to `part` [split][rows][ldp] (+= with `add`), or, unsplit, the result itself
struct ProdArgs {
    Operand a, b;
    int64_t rows;                // n side
    int d;                       // m side
    int nseg;
    int64_t ksteps;
    int64_t tiles_m, tiles;
    float *part;
    int64_t ldp, part_stride;
    int add;
    void *out;                   // part == NULL: [rows][d]
    const float *top;
    float scale;
};

template <class TL, int DT>
__global__ void __launch_bounds__(THREADS, 2) product_kernel(ProdArgs a)
{
    __shared__ __attribute__((aligned(1024))) unsigned char lds[TL::LDS];
    const int64_t t = xcd_tile(a.tiles);
    if (t < 0) return;
    const int64_t tm = t % a.tiles_m, tn = t / a.tiles_m;
    const int64_t m0 = tm * TL::BM, n0 = tn * TL::BN;
    const int64_t steps = a.nseg * a.ksteps, splits = gridDim.y, sp = blockIdx.y;
    const int64_t s0 = steps * sp / splits, s1 = steps * (sp + 1) / splits;
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
    f32x4 acc[TL::MT][TL::NT];
#pragma unroll
    for (int i = 0; i < TL::MT; ++i)
#pragma unroll
        for (int j = 0; j < TL::NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    TL::run(acc, A, B, a.nseg, a.ksteps, s0, s1, lds);

    const float f = a.part == nullptr ? a.top[0] * a.scale : 1.0f;
    const bool wide = (a.d & 7) == 0;
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
                    float4 v = {acc[4 * b + j][nt][0], acc[4 * b + j][nt][1], acc[4 * b + j][nt][2], acc[4 * b + j][nt][3]};
                    if (a.add) {
                        const float4 o = p[j];
                        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
                    }
                    p[j] = v;
                }
                continue;
            }
            if (wide) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (m + 8 * h >= a.d) continue;
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = acc[4 * b + 2 * h + (e >> 2)][nt][e & 3] * f;
                    if (DT == T_F32) {
                        float4 *o = (float4 *)((float *)a.out + n * a.d + m + 8 * h);
                        o[0] = float4{v[0], v[1], v[2], v[3]};
                        o[1] = float4{v[4], v[5], v[6], v[7]};
                    } else {
                        unsigned short u[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) u[e] = to16<DT == T_F16>(v[e]);
                        *(u32x4 *)((unsigned short *)a.out + n * a.d + m + 8 * h) = *(const u32x4 *)u;
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (m + e < a.d) store1<DT>(a.out, n * a.d + m + e, acc[4 * b + (e >> 2)][nt][e & 3] * f);
            }
        }
    }
}

// out[r][c] = (sum over the splits) * top * scale; rows of weight 0 (weight may be NULL: none) are zero
template <int DT>
__global__ void __launch_bounds__(256) join_kernel(const float *__restrict__ part, int64_t part_stride, int splits, int64_t rows, int d,
                                                   int64_t ldp, const float *__restrict__ weight, const float *__restrict__ top,
                                                   float scale, void *__restrict__ out)
{
    const int per = (int)(ldp / 4);
    const int64_t total = rows * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per;
        const int c = (int)(i % per) * 4;
        if (c >= d) continue;
        float4 s = {0.f, 0.f, 0.f, 0.f};
        if (weight == nullptr || weight[r] != 0.0f) {
            for (int k = 0; k < splits; ++k) {
                const float4 p = *(const float4 *)(part + k * part_stride + r * ldp + c);
                s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
            }
            const float g = top[0] * scale;
            s.x *= g; s.y *= g; s.z *= g; s.w *= g;
        }
        const float v[4] = {s.x, s.y, s.z, s.w};
        for (int e = 0; e < 4; ++e)
            if (c + e < d) store1<DT>(out, r * d + c + e, v[e]);
    }
}

// ---- host: sizes, workspace, launches -----------------------------------------------------------------------------------------
int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

struct Plan {
    int64_t n, v, n_pad, vc;         // vc: classes of a piece (whole piece stride)
    int d, dp, parts, dtype;
    bool direct;                     // operands are read where they are
    bool small;                      // few rows: tiles of 32 rows
    int bm;                          // width of the d side of the products' tiles
    int64_t k_dx, k_dw;              // K steps per segment
    int split_dx, split_dw;
};

Plan make_plan(int64_t n, int64_t v, int d, int dtype)
{
    Plan p;
    p.n = n; p.v = v; p.d = d; p.dtype = dtype;
    p.parts = dtype == T_F32 ? 3 : 1;
    p.dp = (int)up(d, 32);
    p.direct = dtype != T_F32 && d % 32 == 0;
    p.n_pad = up(n, 256);
    p.small = n <= 32;
    int64_t most = DZ_BYTES / (p.n_pad * 2 * p.parts);
    if (!p.direct) {
        const int64_t m2 = WPACK_BYTES / ((int64_t)p.dp * 2 * p.parts);
        most = most < m2 ? most : m2;
    }
    most = most / 256 * 256;
    if (most < 256) most = 256;
    p.vc = up(v, 256) < most ? up(v, 256) : most;
    p.bm = d > 128 ? 256 : (d > 64 ? 128 : 64);
    const int bn = p.bm == 64 ? 256 : 128;
    // enough workgroups for two per CU, but at least 8 K steps each
    const int64_t want = 512;
    auto splits = [&](int64_t tiles, int64_t steps) {
        int64_t s = (want + tiles - 1) / tiles;
        s = s < steps / 8 ? s : steps / 8;
        return (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
    };
    const int64_t tm = (p.dp + p.bm - 1) / p.bm;
    const int seg = p.parts == 3 ? 6 : 1;
    p.k_dx = p.vc / BK;
    p.k_dw = up(n, BK) / BK;
    p.split_dx = splits(tm * ((n + bn - 1) / bn), seg * p.k_dx);
    p.split_dw = splits(tm * ((p.vc + bn - 1) / bn), seg * p.k_dw);
    return p;
}

// classes of one forward launch without packed codes: as many as a grid of 2^22 tiles holds
int64_t fwd_piece(const Plan &p)
{
    const int64_t tiles = (1ll << 22) / ((p.n + 31) / 32);
    return (tiles < 1 ? 1 : tiles) * 256;
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
struct BwdSpace { unsigned short *xs, *xp, *wp, *dz; float *dxp, *dwp, *weight, *top; };

FwdSpace fwd_space(const Plan &p, Space &s)
{
    FwdSpace f;
    f.xp = p.direct ? nullptr : (unsigned short *)s.take(p.n_pad * p.dp * 2 * p.parts);
    f.wp = p.direct ? nullptr : (unsigned short *)s.take(p.vc * p.dp * 2 * p.parts);
    f.stats = (float2 *)s.take(up(p.v, 256) / 256 * p.n * 8);
    f.loss = (float *)s.take(p.n * 4);
    return f;
}
BwdSpace bwd_space(const Plan &p, Space &s, bool dx, bool dw)
{
    BwdSpace b;
    b.weight = (float *)s.take(p.n * 4);
    b.top = (float *)s.take(4);
    b.xp = p.direct ? nullptr : (unsigned short *)s.take(p.n_pad * p.dp * 2 * p.parts);
    b.wp = p.direct ? nullptr : (unsigned short *)s.take(p.vc * p.dp * 2 * p.parts);
    b.xs = dw ? (unsigned short *)s.take(p.n_pad * p.dp * 2 * p.parts) : nullptr;
    b.dz = (unsigned short *)s.take(p.n_pad * p.vc * 2 * p.parts);
    b.dxp = dx ? (float *)s.take(p.split_dx * p.n * (int64_t)p.dp * 4) : nullptr;
    b.dwp = dw && p.split_dw > 1 ? (float *)s.take(p.split_dw * p.vc * (int64_t)p.dp * 4) : nullptr;
    return b;
}

unsigned grid1(int64_t items) { const int64_t b = (items + 255) / 256; return (unsigned)(b < 1 ? 1 : (b > 8192 ? 8192 : b)); }

void pack(int dtype, const void *src, int64_t rows, int d, int64_t rows_pad, int dp, const float *weight, unsigned short *dst,
          hipStream_t st)
{
    const unsigned g = grid1(rows_pad * (dp / 8));
    if (dtype == T_F32) pack_kernel<T_F32><<<g, 256, 0, st>>>(src, rows, d, rows_pad, dp, weight, dst);
    else if (dtype == T_BF16) pack_kernel<T_BF16><<<g, 256, 0, st>>>(src, rows, d, rows_pad, dp, weight, dst);
    else pack_kernel<T_F16><<<g, 256, 0, st>>>(src, rows, d, rows_pad, dp, weight, dst);
}

template <class TL, bool DZ, int PARTS>
void launch_head(HeadArgs a, hipStream_t st)
{
    a.tiles_n = (a.n + TL::BN - 1) / TL::BN;
    if (DZ) a.tiles_n = a.n_pad / TL::BN;       // (the padding rows of dz are written too: the products read them)
    a.tiles = (a.vc + TL::BM - 1) / TL::BM * a.tiles_n;
    const unsigned g = (unsigned)(up(a.tiles, 8));
    head_kernel<TL, DZ, PARTS><<<g, THREADS, 0, st>>>(a);
}

template <bool DZ>
void head(const Plan &p, const HeadArgs &a, hipStream_t st)
{
    if (p.dtype == T_F16) {
        if (!DZ && p.small) launch_head<Tile<256, 32, 4, false, false, true>, DZ, 1>(a, st);
        else launch_head<Tile<256, 128, 2, false, false, true>, DZ, 1>(a, st);
    } else if (p.dtype == T_BF16) {
        if (!DZ && p.small) launch_head<Tile<256, 32, 4, false, false, false>, DZ, 1>(a, st);
        else launch_head<Tile<256, 128, 2, false, false, false>, DZ, 1>(a, st);
    } else {
        if (!DZ && p.small) launch_head<Tile<256, 32, 4, false, false, false>, DZ, 3>(a, st);
        else launch_head<Tile<256, 128, 2, false, false, false>, DZ, 3>(a, st);
    }
}

template <class TL>
void launch_product(const Plan &p, ProdArgs a, int splits, hipStream_t st)
{
    a.tiles_m = (p.dp + TL::BM - 1) / TL::BM;
    a.tiles = a.tiles_m * ((a.rows + TL::BN - 1) / TL::BN);
    const dim3 g((unsigned)up(a.tiles, 8), (unsigned)splits);
    if (p.dtype == T_F32) product_kernel<TL, T_F32><<<g, THREADS, 0, st>>>(a);
    else if (TL::F16) product_kernel<TL, T_F16><<<g, THREADS, 0, st>>>(a);
    else product_kernel<TL, T_BF16><<<g, THREADS, 0, st>>>(a);
}
template <bool BCOLS, bool F16>
void product_w(const Plan &p, const ProdArgs &a, int splits, hipStream_t st)
{
    if (p.bm == 64) launch_product<Tile<64, 256, 1, true, BCOLS, F16>>(p, a, splits, st);
    else if (p.bm == 128) launch_product<Tile<128, 128, 2, true, BCOLS, F16>>(p, a, splits, st);
    else launch_product<Tile<256, 128, 2, true, BCOLS, F16>>(p, a, splits, st);
}
template <bool BCOLS>
void product(const Plan &p, const ProdArgs &a, int splits, hipStream_t st)
{
    if (p.dtype == T_F16) product_w<BCOLS, true>(p, a, splits, st);
    else product_w<BCOLS, false>(p, a, splits, st);
}

void join(const Plan &p, const float *part, int64_t stride, int splits, int64_t rows, const float *weight, const float *top,
          float scale, void *out, hipStream_t st)
{
    const unsigned g = grid1(rows * (p.dp / 4));
    if (p.dtype == T_F32) join_kernel<T_F32><<<g, 256, 0, st>>>(part, stride, splits, rows, p.d, p.dp, weight, top, scale, out);
    else if (p.dtype == T_BF16) join_kernel<T_BF16><<<g, 256, 0, st>>>(part, stride, splits, rows, p.d, p.dp, weight, top, scale, out);
    else join_kernel<T_F16><<<g, 256, 0, st>>>(part, stride, splits, rows, p.d, p.dp, weight, top, scale, out);
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

Operand rows_of(const void *p, int64_t plane, int64_t ld) { return Operand{(const unsigned short *)p, plane, ld, 0, 0}; }

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

int rsdf_class_head_fwd(const void *x, const void *w, int64_t n, int64_t v, int d, int dtype, const int64_t *ids,
                        const float *teacher_logits, int k, int64_t ignore_id, float temperature, int reduction, float *loss,
                        float *lse, float *count, float *q, float *listed_z, int32_t *bad_ids, void *workspace,
                        int64_t workspace_bytes, void *stream)
{
    const char *bad = bad_head(n, v, d, dtype, k, x, w);
    RSDF_CHECK_ARG(bad == nullptr, bad);
    RSDF_CHECK_ARG(temperature > 0.0f, "class_head_fwd: temperature must be positive");
    RSDF_CHECK_ARG(teacher_logits != nullptr ? (q != nullptr && listed_z != nullptr) : k == 1,
                   "class_head_fwd: a teacher needs q and listed_z, labels need k = 1");
    RSDF_CHECK_ARG(reduction >= 0 && reduction <= 2, "class_head_fwd: reduction must be 0 (none), 1 (mean) or 2 (sum)");
    const Plan p = make_plan(n, v, d, dtype);
    Space s{(unsigned char *)workspace};
    const FwdSpace f = fwd_space(p, s);
    RSDF_CHECK_ARG(s.at <= workspace_bytes, "class_head_fwd: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    const int64_t xplane = p.n_pad * p.dp, wplane = p.vc * p.dp;
    if (!p.direct) pack(dtype, x, n, d, p.n_pad, p.dp, nullptr, f.xp, st);
    const int64_t piece = p.direct ? fwd_piece(p) : p.vc;       // (nothing is kept of a piece but the packed codes)
    for (int64_t v0 = 0; v0 < v; v0 += piece) {
        const int64_t here = v - v0 < piece ? v - v0 : piece;
        HeadArgs a = {};
        if (!p.direct) pack(dtype, row_ptr(w, v0, d, dtype), here, d, p.vc, p.dp, nullptr, f.wp, st);
        a.x = p.direct ? rows_of(x, 0, d) : rows_of(f.xp, xplane, p.dp);
        a.w = p.direct ? rows_of(row_ptr(w, v0, d, dtype), 0, d) : rows_of(f.wp, wplane, p.dp);
        a.n = n; a.vc = here;
        a.nseg = p.parts == 3 ? 6 : 1;
        a.ksteps = p.dp / BK;
        a.c = LOG2E / temperature;
        a.stats = f.stats;
        a.tile0 = v0 / 256;
        head<false>(p, a, st);
    }
    RowArgs r = {x, w, n, v, d, k, f.stats, up(v, 256) / 256, ids, teacher_logits, ignore_id, temperature,
                 reduction == 0 ? loss : f.loss, lse, q, listed_z, bad_ids};
    const unsigned g = (unsigned)((n + 3) / 4);
    if (dtype == T_F32) rows_kernel<T_F32><<<g, 256, 0, st>>>(r);
    else if (dtype == T_BF16) rows_kernel<T_BF16><<<g, 256, 0, st>>>(r);
    else rows_kernel<T_F16><<<g, 256, 0, st>>>(r);
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
    RSDF_CHECK_ARG((((uintptr_t)dx | (uintptr_t)dw) & 15) == 0, "class_head_bwd: dx and dw must be 16-byte aligned");
    if (dx == nullptr && dw == nullptr) return 0;
    const Plan p = make_plan(n, v, d, dtype);
    Space s{(unsigned char *)workspace};
    const BwdSpace b = bwd_space(p, s, dx != nullptr, dw != nullptr);
    RSDF_CHECK_ARG(s.at <= workspace_bytes, "class_head_bwd: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    const int nseg = p.parts == 3 ? 6 : 1;
    const int64_t xplane = p.n_pad * p.dp, wplane = p.vc * p.dp, zplane = p.n_pad * p.vc;
    const float scale = dtype == T_F16 ? 1.0f / F16_DZ : 1.0f;
    weights_kernel<<<1, 1024, 0, st>>>(lse, grad, grad_per_row, count, temperature, n, b.weight, b.top);
    if (!p.direct) pack(dtype, x, n, d, p.n_pad, p.dp, nullptr, b.xp, st);
    if (dw != nullptr) pack(dtype, x, n, d, p.n_pad, p.dp, b.weight, b.xs, st);
    for (int64_t v0 = 0; v0 < v; v0 += p.vc) {
        const int64_t here = v - v0 < p.vc ? v - v0 : p.vc;
        HeadArgs a = {};
        if (!p.direct) pack(dtype, row_ptr(w, v0, d, dtype), here, d, p.vc, p.dp, nullptr, b.wp, st);
        a.x = p.direct ? rows_of(x, 0, d) : rows_of(b.xp, xplane, p.dp);
        a.w = p.direct ? rows_of(row_ptr(w, v0, d, dtype), 0, d) : rows_of(b.wp, wplane, p.dp);
        a.n = n; a.n_pad = p.n_pad; a.vc = here; a.ldz = p.vc;
        a.nseg = nseg;
        a.ksteps = p.dp / BK;
        a.c = LOG2E / temperature;
        a.lse = lse;
        a.weight = b.weight; a.top = b.top;
        a.label = q == nullptr ? ids : nullptr;
        a.v0 = v0;
        a.dz = b.dz;
        head<true>(p, a, st);
        if (q != nullptr) {
            const unsigned g = (unsigned)((n * k + 255) / 256);
            if (dtype == T_F32) listed_kernel<false, 3><<<g, 256, 0, st>>>(ids, q, listed_z, lse, b.weight, b.top, n, k, a.c, v0, p.vc, p.n_pad, b.dz);
            else if (dtype == T_BF16) listed_kernel<false, 1><<<g, 256, 0, st>>>(ids, q, listed_z, lse, b.weight, b.top, n, k, a.c, v0, p.vc, p.n_pad, b.dz);
            else listed_kernel<true, 1><<<g, 256, 0, st>>>(ids, q, listed_z, lse, b.weight, b.top, n, k, a.c, v0, p.vc, p.n_pad, b.dz);
        }
        if (dx != nullptr) {
            ProdArgs r = {};
            r.a = a.w;
            r.a.k_rows = p.direct ? here : p.vc;
            r.b = rows_of(b.dz, zplane, p.vc);
            r.rows = n; r.d = d; r.nseg = nseg;
            r.ksteps = up(here, BK) / BK;
            r.part = b.dxp; r.ldp = p.dp; r.part_stride = n * p.dp; r.add = v0 > 0;
            product<false>(p, r, p.split_dx, st);
        }
        if (dw != nullptr) {
            ProdArgs r = {};
            r.a = rows_of(b.xs, xplane, p.dp);
            r.a.k_rows = p.n_pad;
            r.b = rows_of(b.dz, zplane, p.vc);
            r.b.k_rows = p.n_pad;
            r.rows = here; r.d = d; r.nseg = nseg;
            r.ksteps = p.k_dw;
            r.part = b.dwp; r.ldp = p.dp; r.part_stride = p.vc * p.dp;
            r.out = (unsigned char *)dw + v0 * d * (dtype == T_F32 ? 4 : 2);
            r.top = b.top;
            r.scale = scale;
            product<true>(p, r, p.split_dw, st);
            if (b.dwp != nullptr) join(p, b.dwp, r.part_stride, p.split_dw, here, nullptr, b.top, scale, r.out, st);
        }
    }
    if (dx != nullptr) join(p, b.dxp, n * p.dp, p.split_dx, n, b.weight, b.top, scale, dx, st);
    RSDF_RETURN_LAUNCH();
}

}  // extern "C"
