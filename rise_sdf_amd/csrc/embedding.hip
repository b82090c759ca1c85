// Code lookup by integer id and its gradient.
//
//   out[n][:] = scale * table[id_n][:]                     (0 where id_n is the padding id, NaN where it is outside [0, V))
//   d table[v][:] = scale * sum over {n : id_n = v} g[n][:]
//
// Both are bound by memory: the lookup reads each row that occurs and writes N rows, the gradient reads N rows and writes V.
// Products and sums are fp32, one rounding to the table's type at the end.
//
// The gradient sorts the positions by id (a stable radix sort of at most 8 bits a pass) and sums the rows of one id in
// order: no float atomics, the same bits every time.  The sorted list is cut into chunks of equal LENGTH, so an id that takes
// half of all positions costs no more than any other: a group of lanes sums its chunk's runs; a run that lies inside one chunk
// is written at once, one that crosses chunks leaves its parts in `part` for the join.  Rows of the table that no position
// names are zeroed by other workgroups of the same launch, which look each row up in the sorted list: every row of the
// result is written exactly once.
#include "common.h"

namespace {

constexpr int T_F32 = 0, T_BF16 = 1, T_F16 = 2;

template <int DT> struct Elem;
template <> struct Elem<T_F32> {
    using type = float;
    __device__ static __forceinline__ float get(float v) { return v; }
    __device__ static __forceinline__ float put(float v) { return v; }
};
template <> struct Elem<T_BF16> {
    using type = unsigned short;
    __device__ static __forceinline__ float get(unsigned short v) { return __builtin_bit_cast(float, (unsigned)v << 16); }
    __device__ static __forceinline__ unsigned short put(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
};
template <> struct Elem<T_F16> {
    using type = unsigned short;
    __device__ static __forceinline__ float get(unsigned short v) { return (float)__builtin_bit_cast(_Float16, v); }
    __device__ static __forceinline__ unsigned short put(float v) { return __builtin_bit_cast(unsigned short, (_Float16)v); }
};
template <class T, int N> struct alignas(sizeof(T) * N) Vec { T v[N]; };

// ---- lookup -------------------------------------------------------------------------------------------------------------------
template <int DT, int VW>
__global__ void __launch_bounds__(256) lookup_kernel(const int64_t *__restrict__ ids, int64_t n, const void *__restrict__ table, int64_t v,
                                                     int per_row, float scale, int64_t padding, int rows_per_block,
                                                     void *__restrict__ out, int *__restrict__ bad_ids)
{
    using E = Elem<DT>;
    using V = Vec<typename E::type, VW>;
    const int64_t r0 = (int64_t)blockIdx.x * rows_per_block;
    const int rows = (int)(n - r0 < rows_per_block ? n - r0 : rows_per_block);
    for (int i = threadIdx.x; i < rows * per_row; i += 256) {
        const int r = i / per_row, c = i - r * per_row;
        const int64_t id = ids[r0 + r];
        V o;
        if (id >= 0 && id < v && id != padding) {
            const V t = ((const V *)table)[id * per_row + c];
#pragma unroll
            for (int e = 0; e < VW; ++e) o.v[e] = E::put(E::get(t.v[e]) * scale);
        } else {
            const float f = id == padding ? 0.0f : __builtin_nanf("");
#pragma unroll
            for (int e = 0; e < VW; ++e) o.v[e] = E::put(f);
            if (c == 0 && id != padding && bad_ids != nullptr) atomicAdd(bad_ids, 1);
        }
        ((V *)out)[(r0 + r) * per_row + c] = o;
    }
}

// ---- stable radix sort of (id, position) ----------------------------------------------------------------------------------------
// One pass = a histogram per workgroup and a scatter; a workgroup's share is contiguous, at most MAX_BLOCKS workgroups.
constexpr int SORT_BINS = 256, MAX_BLOCKS = 256, SORT_ROUND = 256;

__device__ __forceinline__ unsigned sort_key(const int64_t *ids, const unsigned *keys, int64_t i, int64_t v, int64_t padding)
{
    if (ids == nullptr) return keys[i];
    const int64_t id = ids[i];
    return (id >= 0 && id < v && id != padding) ? (unsigned)id : (unsigned)v;      // v: behind every real id
}

// lanes of this wave with the same digit as this lane (among the lanes in `active`)
__device__ __forceinline__ unsigned long long same_digit(unsigned digit, int bits, unsigned long long active)
{
    unsigned long long m = active;
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((digit >> b) & 1);
        m &= (digit >> b) & 1 ? set : ~set;
    }
    return m;
}

__global__ void __launch_bounds__(256) sort_count_kernel(const int64_t *__restrict__ ids, const unsigned *__restrict__ keys, int64_t n, int64_t v,
                                                         int64_t padding, int shift, int bits, int64_t share, unsigned *__restrict__ counts)
{
    __shared__ unsigned c[SORT_BINS];
    c[threadIdx.x] = 0;
    __syncthreads();
    const int64_t b = blockIdx.x * share, e = b + share < n ? b + share : n;
    const unsigned mask = (1u << bits) - 1;
    for (int64_t i = b + threadIdx.x; i < e; i += 256) atomicAdd(&c[(sort_key(ids, keys, i, v, padding) >> shift) & mask], 1u);
    __syncthreads();
    counts[blockIdx.x * SORT_BINS + threadIdx.x] = c[threadIdx.x];
}

__global__ void __launch_bounds__(256) sort_scatter_kernel(const int64_t *__restrict__ ids, const unsigned *__restrict__ keys,
                                                           const unsigned *__restrict__ pos, int64_t n, int64_t v, int64_t padding, int shift,
                                                           int bits, int64_t share, const unsigned *__restrict__ counts,
                                                           unsigned *__restrict__ keys_out, unsigned *__restrict__ pos_out)
{
    __shared__ unsigned base[SORT_BINS];               // where this workgroup's next item of a digit goes
    __shared__ unsigned wave_count[4][SORT_BINS];
    __shared__ unsigned total[4];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    // items of smaller digits anywhere + items of this digit in earlier workgroups
    unsigned before = 0, all = 0;
    for (int b = 0; b < (int)gridDim.x; ++b) {
        const unsigned c = counts[b * SORT_BINS + t];
        before += b < (int)blockIdx.x ? c : 0;
        all += c;
    }
    unsigned incl = (unsigned)wave_incl_sum_i((int)all);
    if (lane == 63) total[w] = incl;
    __syncthreads();
    for (int k = 0; k < w; ++k) incl += total[k];
    base[t] = incl - all + before;
    const int64_t b0 = blockIdx.x * share, e0 = b0 + share < n ? b0 + share : n;
    const unsigned mask = (1u << bits) - 1;
    for (int64_t r = b0; r < e0; r += SORT_ROUND) {
        for (int k = 0; k < 4; ++k) wave_count[k][t] = 0;
        __syncthreads();
        const int64_t i = r + t;
        const bool here = i < e0;
        const unsigned key = here ? sort_key(ids, keys, i, v, padding) : 0;
        const unsigned digit = (key >> shift) & mask;
        const unsigned long long same = same_digit(digit, bits, __ballot(here));
        const unsigned rank = __popcll(same & ((1ull << lane) - 1));
        if (here && rank == 0) wave_count[w][digit] = (unsigned)__popcll(same);
        __syncthreads();
        if (here) {
            unsigned at = base[digit] + rank;
            for (int k = 0; k < w; ++k) at += wave_count[k][digit];
            keys_out[at] = key;
            pos_out[at] = pos == nullptr ? (unsigned)i : pos[i];
        }
        __syncthreads();
        base[t] += wave_count[0][t] + wave_count[1][t] + wave_count[2][t] + wave_count[3][t];
    }
}

// ---- sums over the sorted list --------------------------------------------------------------------------------------------------
struct SumArgs {
    const unsigned *keys, *pos;
    int64_t n, v;
    int d, per_row;              // row length in elements / in vectors
    int chunk;
    int64_t chunks;
    const void *g;
    float scale;
    float *part;                 // [chunk][2][d]: what continues a run of earlier chunks; what begins a run that goes on
    void *out;
    int64_t sum_blocks;          // later workgroups zero rows
    int zero_rows;               // rows per such workgroup
    int groups, lanes;           // groups of lanes per workgroup, lanes per group
};

template <int DT, int VW>
__global__ void __launch_bounds__(256) sum_kernel(SumArgs a)
{
    using E = Elem<DT>;
    using V = Vec<typename E::type, VW>;
    constexpr int U = 4;
    if ((int64_t)blockIdx.x >= a.sum_blocks) {
        // rows without a position
        if (blockIdx.y != 0) return;
        __shared__ unsigned char absent[256];
        const int64_t r0 = ((int64_t)blockIdx.x - a.sum_blocks) * a.zero_rows;
        const int rows = (int)(a.v - r0 < a.zero_rows ? a.v - r0 : a.zero_rows);
        if ((int)threadIdx.x < rows) {
            const unsigned key = (unsigned)(r0 + threadIdx.x);
            int64_t lo = 0, hi = a.n;
            while (lo < hi) {
                const int64_t mid = (lo + hi) >> 1;
                if (a.keys[mid] < key) lo = mid + 1;
                else hi = mid;
            }
            absent[threadIdx.x] = !(lo < a.n && a.keys[lo] == key);
        }
        __syncthreads();
        V z = {};
        for (int i = threadIdx.x; i < rows * a.per_row; i += 256) {
            const int r = i / a.per_row;
            if (absent[r]) ((V *)a.out)[r0 * a.per_row + i] = z;
        }
        return;
    }
    const int group = threadIdx.x / a.lanes, l = threadIdx.x % a.lanes;
    const int64_t c = (int64_t)blockIdx.x * a.groups + group;
    const int col = blockIdx.y * a.lanes + l;
    if (c >= a.chunks || col >= a.per_row) return;
    const int64_t b = c * a.chunk, e = b + a.chunk < a.n ? b + a.chunk : a.n;
    const unsigned none = (unsigned)a.v;
    const unsigned prev = b > 0 ? a.keys[b - 1] : none, next = e < a.n ? a.keys[e] : none;
    unsigned cur = a.keys[b];
    bool first = true;
    float acc[VW];
#pragma unroll
    for (int k = 0; k < VW; ++k) acc[k] = 0.0f;
    auto flush = [&](bool last) {
        if (cur == none) return;
        const bool head = first && prev == cur, tail = last && next == cur;
        if (!head && !tail) {
            V o;
#pragma unroll
            for (int k = 0; k < VW; ++k) o.v[k] = E::put(acc[k] * a.scale);
            ((V *)a.out)[(int64_t)cur * a.per_row + col] = o;
        } else {
            float *p = a.part + (c * 2 + (head ? 0 : 1)) * a.d + col * VW;
#pragma unroll
            for (int k = 0; k < VW; ++k) p[k] = acc[k];
        }
    };
    for (int64_t i = b; i < e; i += U) {
        unsigned key[U];
        V row[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t j = i + u < e ? i + u : e - 1;
            key[u] = a.keys[j];
            row[u] = ((const V *)a.g)[(int64_t)a.pos[j] * a.per_row + col];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u >= e) continue;
            if (key[u] != cur) {
                flush(false);
                first = false;
                cur = key[u];
#pragma unroll
                for (int k = 0; k < VW; ++k) acc[k] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < VW; ++k) acc[k] += E::get(row[u].v[k]);
        }
    }
    flush(true);
}

// a run that begins in chunk c and goes on: its parts in order, 4 waves taking every fourth part
template <int DT>
__global__ void __launch_bounds__(256) join_kernel(SumArgs a)
{
    using E = Elem<DT>;
    __shared__ float sums[4][64];
    const int64_t c = blockIdx.x, b = c * a.chunk, e = b + a.chunk;
    if (e >= a.n) return;
    const unsigned key = a.keys[e - 1];
    if (key == (unsigned)a.v || a.keys[e] != key) return;
    if (b > 0 && a.keys[b] == key && a.keys[b - 1] == key) return;      // began earlier
    int64_t lo = e, hi = a.n;                                           // first position behind the run
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (a.keys[mid] <= key) lo = mid + 1;
        else hi = mid;
    }
    const int64_t last = (lo - 1) / a.chunk;
    const int w = threadIdx.x >> 6, col = blockIdx.y * 64 + (threadIdx.x & 63);
    float s = 0.0f;
    if (col < a.d) {
        if (w == 0) s = a.part[(c * 2 + 1) * a.d + col];
        for (int64_t k = c + 1 + w; k <= last; k += 4) s += a.part[k * 2 * a.d + col];
    }
    sums[w][threadIdx.x & 63] = s;
    __syncthreads();
    if (w == 0 && col < a.d) {
        const int l = threadIdx.x;
        s = (sums[0][l] + sums[1][l]) + (sums[2][l] + sums[3][l]);
        ((typename E::type *)a.out)[(int64_t)key * a.d + col] = E::put(s * a.scale);
    }
}

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

struct Sorting { int passes, bits; int64_t share; unsigned blocks; };
Sorting sorting(int64_t n, int64_t v)
{
    int bits = 1;
    while ((1ll << bits) <= v) ++bits;           // keys 0 .. v
    Sorting s;
    s.passes = (bits + 7) / 8;
    s.bits = (bits + s.passes - 1) / s.passes;
    s.share = up((n + MAX_BLOCKS - 1) / MAX_BLOCKS, SORT_ROUND);
    s.share = s.share < 1024 ? 1024 : s.share;
    s.blocks = (unsigned)((n + s.share - 1) / s.share);
    return s;
}

int chunk_of(int64_t n) { const int64_t c = n / 4096; return (int)(c < 8 ? 8 : (c > 64 ? 64 : c)); }

struct Space { unsigned *keys[2], *pos[2], *counts; float *part; int64_t bytes; };
Space space(void *ws, int64_t n, int64_t v, int d)
{
    Space s;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        void *p = (unsigned char *)ws + at;
        at += up(bytes, 256);
        return p;
    };
    for (int i = 0; i < 2; ++i) { s.keys[i] = (unsigned *)take(n * 4); s.pos[i] = (unsigned *)take(n * 4); }
    s.counts = (unsigned *)take(MAX_BLOCKS * SORT_BINS * 4);
    const int64_t chunk = chunk_of(n);
    s.part = (float *)take((n + chunk - 1) / chunk * 2 * d * 4);
    s.bytes = at;
    return s;
}

const char *bad_shape(int64_t n, int64_t v, int d, int dtype)
{
    if (dtype < T_F32 || dtype > T_F16) return "embedding: dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)";
    if (n < 0 || n > (1ll << 30) || v < 1 || v > (1ll << 30)) return "embedding: positions must be in [0, 2^30], rows in [1, 2^30]";
    if (d < 1 || d > (1 << 16)) return "embedding: row length must be in [1, 2^16]";
    return nullptr;
}

// bytes of a vector that divides a row of d elements and the addresses
int vector_bytes(int d, int dtype, const void *p, const void *q)
{
    const uintptr_t row = (uintptr_t)d * (dtype == T_F32 ? 4 : 2);
    const uintptr_t all = row | (uintptr_t)p | (uintptr_t)q | 16;
    return (int)(all & (~all + 1));
}

}  // namespace

// dispatch over the type and the vector width: F<dtype, elements per vector>
#define RSDF_EMBEDDING_DISPATCH(dtype, bytes, CALL)                                   \
    do {                                                                              \
        if (dtype == T_F32) {                                                         \
            if (bytes == 16) CALL(T_F32, 4);                                          \
            else if (bytes == 8) CALL(T_F32, 2);                                      \
            else CALL(T_F32, 1);                                                      \
        } else if (dtype == T_BF16) {                                                 \
            if (bytes == 16) CALL(T_BF16, 8);                                         \
            else if (bytes == 8) CALL(T_BF16, 4);                                     \
            else if (bytes == 4) CALL(T_BF16, 2);                                     \
            else CALL(T_BF16, 1);                                                     \
        } else {                                                                      \
            if (bytes == 16) CALL(T_F16, 8);                                          \
            else if (bytes == 8) CALL(T_F16, 4);                                      \
            else if (bytes == 4) CALL(T_F16, 2);                                      \
            else CALL(T_F16, 1);                                                      \
        }                                                                             \
    } while (0)

extern "C" {

int rsdf_embedding_fwd(const int64_t *ids, int64_t n, const void *table, int64_t v, int d, int dtype, float scale, int64_t padding_id,
                       void *out, int32_t *bad_ids, void *stream)
{
    const char *bad = bad_shape(n, v, d, dtype);
    RSDF_CHECK_ARG(bad == nullptr, bad);
    if (n == 0) return 0;
    const int bytes = vector_bytes(d, dtype, table, out);
    const int per_row = d * (dtype == T_F32 ? 4 : 2) / bytes;
    int rows = 1024 / per_row;                          // about four vectors a thread
    rows = rows < 1 ? 1 : rows;
    const unsigned grid = (unsigned)((n + rows - 1) / rows);
#define CALL(DT, VW) lookup_kernel<DT, VW><<<grid, 256, 0, (hipStream_t)stream>>>(ids, n, table, v, per_row, scale, padding_id, rows, out, bad_ids)
    RSDF_EMBEDDING_DISPATCH(dtype, bytes, CALL);
#undef CALL
    RSDF_RETURN_LAUNCH();
}

int64_t rsdf_embedding_bwd_workspace_bytes(int64_t n, int64_t v, int d)
{
    const char *bad = bad_shape(n, v, d, T_F32);
    if (bad != nullptr) { rsdf_set_error(bad); return -1; }
    return space(nullptr, n, v, d).bytes;
}

int rsdf_embedding_bwd(const int64_t *ids, int64_t n, const void *grad, int64_t v, int d, int dtype, float scale, int64_t padding_id,
                       void *d_table, void *workspace, int64_t workspace_bytes, void *stream)
{
    const char *bad = bad_shape(n, v, d, dtype);
    RSDF_CHECK_ARG(bad == nullptr, bad);
    const Space s = space(workspace, n, v, d);
    RSDF_CHECK_ARG(s.bytes <= workspace_bytes, "embedding_bwd: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    const Sorting so = sorting(n, v);
    int from = 1;
    if (n > 0)
        for (int p = 0; p < so.passes; ++p) {
            const int64_t *first = p == 0 ? ids : nullptr;
            const int to = 1 - from;
            sort_count_kernel<<<so.blocks, 256, 0, st>>>(first, s.keys[from], n, v, padding_id, p * so.bits, so.bits, so.share, s.counts);
            sort_scatter_kernel<<<so.blocks, 256, 0, st>>>(first, s.keys[from], p == 0 ? nullptr : s.pos[from], n, v, padding_id,
                                                           p * so.bits, so.bits, so.share, s.counts, s.keys[to], s.pos[to]);
            from = to;
        }
    const int bytes = vector_bytes(d, dtype, grad, d_table);
    const int per_row = d * (dtype == T_F32 ? 4 : 2) / bytes;
    SumArgs a;
    a.keys = s.keys[from]; a.pos = s.pos[from];
    a.n = n; a.v = v; a.d = d; a.per_row = per_row;
    a.chunk = chunk_of(n);
    a.chunks = (n + a.chunk - 1) / a.chunk;
    a.g = grad; a.scale = scale; a.part = s.part; a.out = d_table;
    a.lanes = 1;
    while (a.lanes < per_row && a.lanes < 64) a.lanes *= 2;
    a.groups = 256 / a.lanes;
    a.sum_blocks = (a.chunks + a.groups - 1) / a.groups;
    a.zero_rows = 4096 / per_row;
    a.zero_rows = a.zero_rows < 1 ? 1 : (a.zero_rows > 256 ? 256 : a.zero_rows);
    const int64_t blocks = a.sum_blocks + (v + a.zero_rows - 1) / a.zero_rows;
    const dim3 grid((unsigned)blocks, (unsigned)((per_row + a.lanes - 1) / a.lanes));
#define CALL(DT, VW) sum_kernel<DT, VW><<<grid, 256, 0, st>>>(a)
    RSDF_EMBEDDING_DISPATCH(dtype, bytes, CALL);
#undef CALL
    if (a.chunks > 1) {
        const dim3 g((unsigned)(a.chunks - 1), (unsigned)((d + 63) / 64));
        if (dtype == T_F32) join_kernel<T_F32><<<g, 256, 0, st>>>(a);
        else if (dtype == T_BF16) join_kernel<T_BF16><<<g, 256, 0, st>>>(a);
        else join_kernel<T_F16><<<g, 256, 0, st>>>(a);
    }
    RSDF_RETURN_LAUNCH();
}

}  // extern "C"
