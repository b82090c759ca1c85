// Code lookup by integer id and its gradient.
//
//   out[n][:] = scale * table[id_n][:]                     (0 where id_n is the padding id, NaN where it is outside [0, V))
//   d table[v][:] = scale * sum over {n : id_n = v} g[n][:]
//
// Both are bound by memory: the lookup reads each row that occurs and writes N rows, the gradient reads N rows and writes V.
// Products and sums are fp32, one rounding to the table's type at the end.  262144 rows of 65536 x 256 bf16: lookup 28 us (6 TB/s:
// the popular rows come from the caches), gradient 76 (sort 33, sums 33, joins 10).
//
// The gradient sorts the positions by id (a stable radix sort) and sums the rows of one id in
// order: no float atomics, the same bits every time.  The sorted list is cut into chunks of equal LENGTH, so an id that takes
// half of all positions costs no more than any other: a group of lanes sums its chunk's runs; a run that lies inside one chunk
// is written at once, one that crosses chunks leaves its parts in `part` for the join.  Rows of the table that no position
// names are zeroed by other workgroups of the same launch, which look each row up in the sorted list: every row of the
// result is written exactly once.
#include "common.h"

namespace {

constexpr int T_F32 = 0, T_BF16 = 1, T_F16 = 2;
constexpr int64_t L2_BYTES = 32ll << 20;          // of the eight XCDs

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
// N elements at any address of an element: rows of an odd length start anywhere, and the last vector of a row begins where it
// ends with the row (what it shares with the one before is handled twice, alike)
template <class T, int N> struct Vec { T v[N]; };
template <int BYTES> struct Bits { using type = __attribute__((ext_vector_type(BYTES / 4))) unsigned; };
template <> struct Bits<4> { using type = unsigned; };
template <> struct Bits<2> { using type = unsigned short; };
template <class V> __device__ __forceinline__ int element_of(int c, int d)
{
    constexpr int N = sizeof(V) / sizeof(V::v[0]);
    return c * N + N <= d ? c * N : d - N;
}
template <class V, class T> __device__ __forceinline__ V load_at(const T *p, int64_t i)
{
    typedef typename Bits<sizeof(V)>::type B __attribute__((aligned(sizeof(T))));
    return __builtin_bit_cast(V, *(const B *)(p + i));
}
// NT: a store that does not stay in the caches: written once, read by someone else
template <bool NT, class V, class T> __device__ __forceinline__ void store_at(T *p, int64_t i, const V &v)
{
    typedef typename Bits<sizeof(V)>::type B __attribute__((aligned(sizeof(T))));
    if (NT && sizeof(V) >= 8) __builtin_nontemporal_store(__builtin_bit_cast(typename Bits<sizeof(V)>::type, v), (B *)(p + i));
    else *(B *)(p + i) = __builtin_bit_cast(typename Bits<sizeof(V)>::type, v);
}

// ---- lookup -------------------------------------------------------------------------------------------------------------------
// NT: the output passes the caches by, the table stays in them (262144 x 256 bf16: 28 instead of 42 us where few ids are frequent, 39 and 40
// where all are alike; 10000 x 100 fp16 3.5 and 3.4; with a reader right behind it 4 to 128 MB differ by less than 5 % either way)
template <int DT, int VW, bool NT>
__global__ void __launch_bounds__(256) lookup_kernel(const int64_t *__restrict__ ids, int64_t n, const void *__restrict__ table, int64_t v,
                                                     int d, int per_row, float scale, int64_t padding, int rows_per_block,
                                                     void *__restrict__ out, int *__restrict__ bad_ids)
{
    using E = Elem<DT>;
    using T = typename E::type;
    using V = Vec<T, VW>;
    constexpr int U = 4;
    const int64_t r0 = (int64_t)blockIdx.x * rows_per_block;
    const int rows = (int)(n - r0 < rows_per_block ? n - r0 : rows_per_block), items = rows * per_row;
    for (int i0 = threadIdx.x; i0 < items; i0 += 256 * U) {
        int64_t id[U];
        int c[U], to[U];
        V o[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * 256 < items ? i0 + u * 256 : i0;
            const int r = i / per_row;
            c[u] = element_of<V>(i - r * per_row, d);
            to[u] = r * d + c[u];
            id[u] = ids[r0 + r];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = id[u] >= 0 && id[u] < v;
            o[u] = load_at<V>((const T *)table, (in ? id[u] : 0) * d + c[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u * 256 >= items) continue;
            const bool in = id[u] >= 0 && id[u] < v;
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                const float f = in ? E::get(o[u].v[e]) * scale : __builtin_nanf("");
                o[u].v[e] = E::put(id[u] == padding ? 0.0f : f);
            }
            if (!in && id[u] != padding && c[u] == 0 && bad_ids != nullptr) atomicAdd(bad_ids, 1);
            store_at<NT>((T *)out + r0 * d, to[u], o[u]);
        }
    }
}

// ---- stable radix sort of (id, position) ----------------------------------------------------------------------------------------
// A pass: a histogram per workgroup (left out where there is one workgroup) and a scatter.  A workgroup's share of the list is
// contiguous and so is a wave's part of it: a wave ranks its 64 x ITEMS items among themselves with ballots, one table of counts per
// wave in LDS, and the waves' tables are summed once.  Up to 9 bits a pass: two passes for 2^18 ids.
constexpr int SORT_THREADS = 512, SORT_WAVES = 8, ITEMS = 4, ROUND = SORT_THREADS * ITEMS, SORT_BITS = 9, BINS = 1 << SORT_BITS, MAX_BLOCKS = 128;

__device__ __forceinline__ unsigned sort_key(const int64_t *ids, const unsigned *keys, int64_t i, int64_t v, int64_t padding)
{
    if (ids == nullptr) return keys[i];
    const int64_t id = ids[i];
    return (id >= 0 && id < v && id != padding) ? (unsigned)id : (unsigned)v;      // v: behind every real id
}

// lanes of this wave in `active` with the same digit as this lane
__device__ __forceinline__ unsigned long long same_digit(unsigned digit, int bits, unsigned long long active)
{
    unsigned long long m = active;
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((digit >> b) & 1);
        m &= (digit >> b) & 1 ? set : ~set;
    }
    return m;
}

__global__ void __launch_bounds__(SORT_THREADS) sort_count_kernel(const int64_t *__restrict__ ids, const unsigned *__restrict__ keys, int64_t n,
                                                                  int64_t v, int64_t padding, int shift, int bits, int64_t share,
                                                                  unsigned *__restrict__ counts)
{
    __shared__ unsigned c[BINS];
    c[threadIdx.x] = 0;
    __syncthreads();
    const int64_t b = blockIdx.x * share, e = b + share < n ? b + share : n;
    const unsigned mask = (1u << bits) - 1;
#pragma unroll 4
    for (int64_t i = b + threadIdx.x; i < e; i += SORT_THREADS) atomicAdd(&c[(sort_key(ids, keys, i, v, padding) >> shift) & mask], 1u);
    __syncthreads();
    counts[blockIdx.x * BINS + threadIdx.x] = c[threadIdx.x];
}

__global__ void __launch_bounds__(SORT_THREADS) sort_scatter_kernel(const int64_t *__restrict__ ids, const unsigned *__restrict__ keys,
                                                                    const unsigned *__restrict__ pos, int64_t n, int64_t v, int64_t padding,
                                                                    int shift, int bits, int64_t share, const unsigned *__restrict__ counts,
                                                                    unsigned *__restrict__ keys_out, unsigned *__restrict__ pos_out)
{
    __shared__ unsigned count[SORT_WAVES][BINS];       // items of a digit in a wave's part, then where its next one goes
    __shared__ unsigned total[SORT_WAVES];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const unsigned mask = (1u << bits) - 1;
    // sum over the digits before digit t of their items
    auto before_digit = [&](unsigned all) {
        unsigned incl = (unsigned)wave_incl_sum_i((int)all);
        if (lane == 63) total[w] = incl;
        __syncthreads();
        for (int k = 0; k < w; ++k) incl += total[k];
        return incl - all;
    };
    unsigned base = 0;                                 // where the next item of digit t goes
    if (gridDim.x > 1) {
        unsigned before = 0, all = 0;
#pragma unroll 16
        for (int b = 0; b < (int)gridDim.x; ++b) {
            const unsigned c = counts[b * BINS + t];
            before += b < (int)blockIdx.x ? c : 0;
            all += c;
        }
        base = before_digit(all) + before;
    }
    const int64_t b0 = blockIdx.x * share, e0 = b0 + share < n ? b0 + share : n;
    for (int64_t r = b0; r < e0; r += ROUND) {
        const int64_t first = r + w * (64 * ITEMS) + lane;
        unsigned key[ITEMS], rank[ITEMS];
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) key[j] = first + j * 64 < e0 ? sort_key(ids, keys, first + j * 64, v, padding) : 0;
        for (int k = lane; k < BINS; k += 64) count[w][k] = 0;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const bool here = first + j * 64 < e0;
            const unsigned digit = (key[j] >> shift) & mask;
            const unsigned long long same = same_digit(digit, bits, __ballot(here));
            const unsigned mine = __popcll(same & ((1ull << lane) - 1));
            volatile unsigned *c = &count[w][digit];
            const unsigned seen = *c;
            rank[j] = seen + mine;
            if (here && mine == 0) *c = seen + (unsigned)__popcll(same);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        unsigned all = 0;
        for (int k = 0; k < SORT_WAVES; ++k) {
            const unsigned c = count[k][t];
            count[k][t] = all;
            all += c;
        }
        if (gridDim.x == 1 && r == b0 && e0 - b0 <= ROUND) base = before_digit(all);       // the whole list is here
        for (int k = 0; k < SORT_WAVES; ++k) count[k][t] += base;
        base += all;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const int64_t i = first + j * 64;
            if (i >= e0) continue;
            const unsigned at = count[w][(key[j] >> shift) & mask] + rank[j];
            keys_out[at] = key[j];
            pos_out[at] = pos == nullptr ? (unsigned)i : pos[i];
        }
        __syncthreads();
    }
}

// ---- few positions: no sort -----------------------------------------------------------------------------------------------------
// One launch, no workspace: a wave per row of the table looks through all ids, 64 at a time, and lists the first LIGHT positions of its
// row.  Groups of lanes (as many as a row of vectors needs) take every so-manieth position, and their sums are added in order.  A row
// with more positions, the one id of a whole batch for instance, is listed again and added up by all four waves.
// Against sorting (four or five launches; both in us of kernels): 256 positions of 100 x 48 fp32 4.1 and 13.1, 1024 of 4000 x 48 7.1 and 19,
// 512 of 16000 x 64 10.6 and 20, one id for 512 rows of 512 fp32 15.2 and 15.2; but one id for 2048 such rows 73 and 22, 100 of 60000
// x 48 30 and 19: so up to FEW positions of FEW_ROWS rows.
constexpr int LIGHT = 64, FEW = 1024;
constexpr int64_t FEW_ROWS = 16384;
template <int DT, int VW>
__global__ void __launch_bounds__(256) few_kernel(const int64_t *__restrict__ ids, int n, const void *__restrict__ g, int64_t v, int d, int per_row,
                                                  int lanes, float scale, int64_t padding, void *__restrict__ out)
{
    using E = Elem<DT>;
    using T = typename E::type;
    using V = Vec<T, VW>;
    constexpr int U = 8;                                 // rows on their way at once
    __shared__ unsigned short list[FEW];                 // LIGHT of each wave; all of one row
    __shared__ int counts[4];
    __shared__ float sums[256 * VW];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t first = (int64_t)blockIdx.x * 4;
    const unsigned long long below = (1ull << lane) - 1;

    // positions of a row into a list of at most `most`; their number
    auto look = [&](int64_t row, unsigned short *to, int most) {
        int count = 0;
        for (int i0 = 0; i0 < n; i0 += 64 * U) {
            bool mine[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * 64 + lane;
                mine[u] = ids[i < n ? i : 0] == row && i < n;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const unsigned long long m = __ballot(mine[u]);
                const int at = count + __popcll(m & below);
                if (mine[u] && at < most) to[at] = (unsigned short)(i0 + u * 64 + lane);
                count += __popcll(m);
            }
        }
        return count;
    };
    // vector c of the positions k, k + step, ... of a list
    auto add = [&](float (&acc)[VW], const unsigned short *from, int count, int k, int step, int c) {
        const int col = element_of<V>(c, d);
#pragma unroll
        for (int e = 0; e < VW; ++e) acc[e] = 0.0f;
        for (; k < count; k += step * U) {
            V x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = load_at<V>((const T *)g, (int64_t)from[k + u * step < count ? k + u * step : k] * d + col);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < VW; ++e) acc[e] += k + u * step < count ? E::get(x[u].v[e]) : 0.0f;
        }
    };
    auto put = [&](const float (&acc)[VW], int64_t row, int c) {
        V o;
#pragma unroll
        for (int e = 0; e < VW; ++e) o.v[e] = E::put(acc[e] * scale);
        store_at<false>((T *)out, row * d + element_of<V>(c, d), o);
    };

    const int64_t row = first + w;
    const int count = row < v && row != padding ? look(row, list + w * LIGHT, LIGHT) : 0;
    if (lane == 0) counts[w] = count;
    __builtin_amdgcn_wave_barrier();
    if (row < v && count <= LIGHT) {
        const int in_wave = lanes < 64 ? lanes : 64, groups = 64 / in_wave, k = lane / in_wave;
        for (int c0 = 0; c0 < per_row; c0 += in_wave) {
            const int c = c0 + lane % in_wave;
            float acc[VW];
            add(acc, list + w * LIGHT, c < per_row ? count : 0, k, groups, c < per_row ? c : 0);
            for (int o = 32; o >= in_wave; o >>= 1)
#pragma unroll
                for (int e = 0; e < VW; ++e) acc[e] += __shfl_xor(acc[e], o, 64);
            if (k == 0 && c < per_row) put(acc, row, c);
        }
    }
    __syncthreads();
    for (int heavy = 0; heavy < 4; ++heavy) {
        if (counts[heavy] <= LIGHT) continue;
        if (w == heavy) look(row, list, FEW);
        __syncthreads();
        const int groups = 256 / lanes, k = threadIdx.x / lanes;
        for (int c0 = 0; c0 < per_row; c0 += lanes) {
            const int c = c0 + threadIdx.x % lanes;
            float acc[VW];
            add(acc, list, c < per_row ? counts[heavy] : 0, k, groups, c < per_row ? c : 0);
#pragma unroll
            for (int e = 0; e < VW; ++e) sums[e * 256 + threadIdx.x] = acc[e];
            __syncthreads();
            if (k == 0 && c < per_row) {
                for (int j = 1; j < groups; ++j)
#pragma unroll
                    for (int e = 0; e < VW; ++e) acc[e] += sums[e * 256 + j * lanes + threadIdx.x];
                put(acc, first + heavy, c);
            }
            __syncthreads();
        }
    }
}

// ---- sums over the sorted list --------------------------------------------------------------------------------------------------
constexpr int LONG = 16;         // a run over more chunks than this is joined by a whole workgroup
struct SumArgs {
    const unsigned *keys, *pos;
    int64_t n, v;
    int d, per_row;              // row length in elements / in vectors (the last one may overlap)
    int chunk;
    int64_t chunks;
    const void *g;
    float scale;
    float *part;                 // [chunk][2][d]: what continues a run of earlier chunks; what begins a run that goes on
    unsigned char *goes_on;      // [chunk]: a run begins there that goes on (1; 2 over more than LONG chunks)
    void *out;
    int64_t sum_blocks;          // later workgroups zero rows
    int zero_rows;               // rows per such workgroup
    int groups, lanes;           // groups of lanes per workgroup, lanes per group
};

template <int DT, int VW>
__global__ void __launch_bounds__(256) sum_kernel(SumArgs a)
{
    using E = Elem<DT>;
    using T = typename E::type;
    using V = Vec<T, VW>;
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
            if (absent[r]) store_at<false>((T *)a.out + r0 * a.d, r * a.d + element_of<V>(i - r * a.per_row, a.d), z);
        }
        return;
    }
    const int group = threadIdx.x / a.lanes, l = threadIdx.x % a.lanes;
    const int64_t c = (int64_t)blockIdx.x * a.groups + group;
    const int vec = blockIdx.y * a.lanes + l, col = element_of<V>(vec, a.d);
    if (c >= a.chunks || vec >= a.per_row) return;
    const int64_t b = c * a.chunk, e = b + a.chunk < a.n ? b + a.chunk : a.n;
    const unsigned none = (unsigned)a.v;
    const unsigned prev = b > 0 ? a.keys[b - 1] : none, next = e < a.n ? a.keys[e] : none;
    unsigned cur = a.keys[b];
    bool first = true, marked = false;
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
            store_at<false>((T *)a.out, (int64_t)cur * a.d + col, o);
        } else {
            float *p = a.part + (c * 2 + (head ? 0 : 1)) * a.d + col;
#pragma unroll
            for (int k = 0; k < VW; ++k) p[k] = acc[k];
            if (!head && vec == 0) {
                const int64_t far = b + (int64_t)a.chunk * (LONG + 1);
                a.goes_on[c] = far < a.n && a.keys[far] == cur ? 2 : 1;
                marked = true;
            }
        }
    };
    for (int64_t i = b; i < e; i += U) {
        unsigned key[U];
        V row[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t j = i + u < e ? i + u : e - 1;
            key[u] = a.keys[j];
            row[u] = load_at<V>((const T *)a.g, (int64_t)a.pos[j] * a.d + col);
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
    if (!marked && vec == 0) a.goes_on[c] = 0;
}

// The runs that cross chunks: one wave per chunk and 64 columns looks whether one begins there.  A short run it joins by itself, a
// long one with the other 15 waves of the workgroup (each every sixteenth part).
constexpr int JOIN_WAVES = 16;
template <int DT>
__global__ void __launch_bounds__(64 * JOIN_WAVES) join_kernel(SumArgs a)
{
    using E = Elem<DT>;
    using T = typename E::type;
    __shared__ float sums[JOIN_WAVES][64];
    __shared__ unsigned char is_long[JOIN_WAVES];
    const int segs = (a.d + 63) / 64, l = threadIdx.x & 63, w = threadIdx.x >> 6;
    // (chunks run fastest: the columns of one long run go to different workgroups)
    const int64_t job0 = (int64_t)blockIdx.x * JOIN_WAVES, each = a.chunks - 1, jobs = each * segs;
    const int kind = job0 + w < jobs ? a.goes_on[(job0 + w) % each] : 0;
    if (l == 0) is_long[w] = kind == 2;
    if (kind == 1) {
        const int64_t c = (job0 + w) % each, e = (c + 1) * a.chunk;
        const unsigned key = a.keys[e];
        // chunks behind c that begin with this id (at most LONG)
        const int64_t at = e + (int64_t)l * a.chunk;
        const unsigned long long other = ~__ballot(at < a.n && a.keys[at] == key);
        const int parts = __ffsll((long long)other) - 1;
        const int col = (int)((job0 + w) / each) * 64 + l;
        if (col < a.d) {
            float s = a.part[(c * 2 + 1) * a.d + col];
#pragma unroll 4
            for (int k = 1; k <= parts; ++k) s += a.part[(c + k) * 2 * a.d + col];
            ((T *)a.out)[(int64_t)key * a.d + col] = E::put(s * a.scale);
        }
    }
    __syncthreads();
    for (int i = 0; i < JOIN_WAVES; ++i) {
        if (!is_long[i]) continue;
        const int64_t c = (job0 + i) % each, e = (c + 1) * a.chunk;
        const unsigned key = a.keys[e];
        int64_t last = c;                                               // the last chunk that begins with this id
        for (int here = JOIN_WAVES * 64; here == JOIN_WAVES * 64;) {
            const int64_t at = (last + 1 + threadIdx.x) * a.chunk;
            here = __syncthreads_count(at < a.n && a.keys[at] == key);
            last += here;
        }
        const int col = (int)((job0 + i) / each) * 64 + l;
        float s = 0.0f;
        if (col < a.d) {
            if (w == 0) s = a.part[(c * 2 + 1) * a.d + col];
#pragma unroll 4
            for (int64_t k = c + 1 + w; k <= last; k += JOIN_WAVES) s += a.part[k * 2 * a.d + col];
        }
        sums[w][l] = s;
        __syncthreads();
        if (w == 0 && col < a.d) {
            s = 0.0f;
#pragma unroll
            for (int k = 0; k < JOIN_WAVES; ++k) s += sums[k][l];
            ((T *)a.out)[(int64_t)key * a.d + col] = E::put(s * a.scale);
        }
        __syncthreads();
    }
}

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

struct Sorting { int passes, bits; int64_t share; unsigned blocks; };
Sorting sorting(int64_t n, int64_t v)
{
    int bits = 1;
    while ((1ll << bits) <= v) ++bits;           // keys 0 .. v
    Sorting s;
    s.passes = (bits + SORT_BITS - 1) / SORT_BITS;
    s.bits = (bits + s.passes - 1) / s.passes;
    s.share = up((n + MAX_BLOCKS - 1) / MAX_BLOCKS, ROUND);
    s.blocks = (unsigned)((n + s.share - 1) / s.share);
    return s;
}

// (sums and joins of 262144 x 256 bf16: chunks of 8 83 us, of 32 46, of 64 43; of 10000 x 250 fp32: 15, 18, 28; of 100000 x 64: 20, 21, 31)
int chunk_of(int64_t n) { const int64_t c = n / 4096; return (int)(c < 8 ? 8 : (c > 64 ? 64 : c)); }

bool use_few(int64_t n, int64_t v) { return n > 0 && n <= FEW && v <= FEW_ROWS; }

struct Space { unsigned *keys[2], *pos[2], *counts; unsigned char *goes_on; float *part; int64_t bytes; };
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
    s.counts = (unsigned *)take(MAX_BLOCKS * BINS * 4);
    const int64_t chunk = chunk_of(n);
    s.goes_on = (unsigned char *)take((n + chunk - 1) / chunk);
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

// bytes of a vector: 16, less only where a row is shorter
int vector_bytes(int d, int dtype)
{
    const int size = dtype == T_F32 ? 4 : 2;
    int bytes = 16;
    while (bytes > d * size) bytes /= 2;
    return bytes;
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
    RSDF_CHECK_ARG(ids != nullptr && table != nullptr && out != nullptr, "embedding_fwd: ids, table and out must not be NULL");
    const int bytes = vector_bytes(d, dtype), size = dtype == T_F32 ? 4 : 2;
    const int per_row = (d * size + bytes - 1) / bytes;
    int rows = 1024 / per_row;                          // about four vectors a thread
    rows = rows < 1 ? 1 : rows;
    const unsigned grid = (unsigned)((n + rows - 1) / rows);
    const bool past = n * d * size >= L2_BYTES;
#define CALL(DT, VW)                                                                                                                   \
    past ? lookup_kernel<DT, VW, true><<<grid, 256, 0, (hipStream_t)stream>>>(ids, n, table, v, d, per_row, scale, padding_id, rows, out, bad_ids) \
         : lookup_kernel<DT, VW, false><<<grid, 256, 0, (hipStream_t)stream>>>(ids, n, table, v, d, per_row, scale, padding_id, rows, out, bad_ids)
    RSDF_EMBEDDING_DISPATCH(dtype, bytes, CALL);
#undef CALL
    RSDF_RETURN_LAUNCH();
}

int64_t rsdf_embedding_bwd_workspace_bytes(int64_t n, int64_t v, int d)
{
    const char *bad = bad_shape(n, v, d, T_F32);
    if (bad != nullptr) { rsdf_set_error(bad); return -1; }
    return use_few(n, v) ? 0 : space(nullptr, n, v, d).bytes;
}

int rsdf_embedding_bwd(const int64_t *ids, int64_t n, const void *grad, int64_t v, int d, int dtype, float scale, int64_t padding_id,
                       void *d_table, void *workspace, int64_t workspace_bytes, void *stream)
{
    const char *bad = bad_shape(n, v, d, dtype);
    RSDF_CHECK_ARG(bad == nullptr, bad);
    RSDF_CHECK_ARG(d_table != nullptr && (n == 0 || (ids != nullptr && grad != nullptr)),
                   "embedding_bwd: d_table, and with positions ids and grad, must not be NULL");
    hipStream_t st = (hipStream_t)stream;
    const int bytes = vector_bytes(d, dtype), size = dtype == T_F32 ? 4 : 2;
    const int per_row = (d * size + bytes - 1) / bytes;
    if (use_few(n, v)) {
        int lanes = 1;
        while (lanes < per_row && lanes < 256) lanes *= 2;
#define CALL(DT, VW) \
    few_kernel<DT, VW><<<(unsigned)((v + 3) / 4), 256, 0, st>>>(ids, (int)n, grad, v, d, per_row, lanes, scale, padding_id, d_table)
        RSDF_EMBEDDING_DISPATCH(dtype, bytes, CALL);
#undef CALL
        RSDF_RETURN_LAUNCH();
    }
    const Space s = space(workspace, n, v, d);
    RSDF_CHECK_ARG(workspace != nullptr && s.bytes <= workspace_bytes, "embedding_bwd: workspace too small");
    const Sorting so = sorting(n, v);
    int from = 1;
    if (n > 0)
        for (int p = 0; p < so.passes; ++p) {
            const int64_t *first = p == 0 ? ids : nullptr;
            const int to = 1 - from;
            if (so.blocks > 1)
                sort_count_kernel<<<so.blocks, SORT_THREADS, 0, st>>>(first, s.keys[from], n, v, padding_id, p * so.bits, so.bits, so.share,
                                                                      s.counts);
            sort_scatter_kernel<<<so.blocks, SORT_THREADS, 0, st>>>(first, s.keys[from], p == 0 ? nullptr : s.pos[from], n, v, padding_id,
                                                                    p * so.bits, so.bits, so.share, s.counts, s.keys[to], s.pos[to]);
            from = to;
        }
    SumArgs a;
    a.keys = s.keys[from]; a.pos = s.pos[from];
    a.n = n; a.v = v; a.d = d; a.per_row = per_row;
    a.chunk = chunk_of(n);
    a.chunks = (n + a.chunk - 1) / a.chunk;
    a.g = grad; a.scale = scale; a.part = s.part; a.goes_on = s.goes_on; a.out = d_table;
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
        const int64_t jobs = (a.chunks - 1) * ((d + 63) / 64);
        const unsigned g = (unsigned)((jobs + JOIN_WAVES - 1) / JOIN_WAVES);
        if (dtype == T_F32) join_kernel<T_F32><<<g, 64 * JOIN_WAVES, 0, st>>>(a);
        else if (dtype == T_BF16) join_kernel<T_BF16><<<g, 64 * JOIN_WAVES, 0, st>>>(a);
        else join_kernel<T_F16><<<g, 64 * JOIN_WAVES, 0, st>>>(a);
    }
    RSDF_RETURN_LAUNCH();
}

}  // extern "C"
