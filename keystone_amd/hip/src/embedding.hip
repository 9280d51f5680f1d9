// Token embeddings: rows of a table by id, their weighted sums over bags,
// and the table's gradient.
//
//   lookup   Y[i]  = s T[id_i]
//   bag      Y[b]  = s sum_{j in bag b} w_j T[id_j]
//   grad     dT[v] = s sum_{j : id_j = v} w_j dY[row_j]
//
// An id outside [0, V) reads nothing and adds nothing.  The last two are one
// operation, a segmented sum of gathered rows: a bag's segment is its own
// stretch of ids, a token's is its stretch of the sorted tokens, so that
// every sum has one order and no atomics, and two runs agree bit for bit.
// Sums are held in 32 bits and rounded once, to the output's type.
//
// All of it is memory.  Measured on one MI355X (a large copy: 4.75 TB/s):
//   lookup of 262144 x 512 bf16 rows of 100000: 54 us, 5 TB/s written
//   sums of 3.3 M f16 rows of 256 over 32768 bags: 127 us, 13 TB/s gathered, 61 %
//     of it from the L2s, which all hold the same hottest rows
//   gradient of 1048576 bf16 rows of 256 onto 100000: 136 us, 4.7 TB/s
//   gradient of 7.8 M weighted entries onto 100000 x 2 f32: 142 us; each
//     weight, gathered in the sorted order, costs a cache line
#include "common.h"

#include <cstdint>

namespace {

template <typename T, int N>
using Vec = T __attribute__((ext_vector_type(N)));

template <typename T, int N, bool PAST = false>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
    using M = typename InMemory<T, N>::type;
    if constexpr (PAST)
        return __builtin_nontemporal_load(reinterpret_cast<const M*>(p));
    else
        return *reinterpret_cast<const M*>(p);
}

template <typename T, int N>
__device__ __forceinline__ void load_row(const T* p, float (&v)[N]) {
    const Vec<T, N> x = load_vec<T, N>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)x[i];
}

// PAST: past the caches, for what is too large to be found there later.
template <typename T, int N, bool PAST = false>
__device__ __forceinline__ void store_row(T* p, const float (&v)[N]) {
    using M = typename InMemory<T, N>::type;
    Vec<T, N> x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (T)v[i];
    if constexpr (PAST)
        __builtin_nontemporal_store(x, reinterpret_cast<M*>(p));
    else
        *reinterpret_cast<M*>(p) = x;
}

template <typename T, int N, bool PAST>
__device__ __forceinline__ Vec<T, N> load_buffer(__amdgpu_buffer_rsrc_t b,
                                                 unsigned at) {
    static_assert(N * sizeof(T) == 16);
    return __builtin_bit_cast(
        Vec<T, N>, __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, PAST ? 2 : 0));
}

// Where lane c of a row begins: at c VEC, the last one early enough to end with
// the row.  What it then shares with its neighbour both compute alike, and
// write alike.
template <int VEC>
__device__ __forceinline__ int column_of(int c, int D) {
    return min(c * VEC, D - VEC);
}

// Token ids as they come: 32 or 64 bits; -1 for one outside the table.
struct Ids {
    const void* p;
    int wide;
    long long rows;   // V
};

__device__ __forceinline__ int row_of(const Ids& t, long long i) {
    const long long v = t.wide ? ((const long long*)t.p)[i]
                               : (long long)((const int*)t.p)[i];
    return (v >= 0 && v < t.rows) ? (int)v : -1;
}

// Segments of n entries: stretches of one fixed length, or bounds in 32 or
// 64 bits.  Whatever the bounds hold, what is read stays inside [0, n].
struct Segs {
    const void* p;
    int kind;         // 0: fixed length, 1: int32 bounds, 2: int64 bounds
    int fixed;
    int count;
    int n;
};

__device__ __forceinline__ int bound_at(const Segs& s, int i) {
    const long long v = s.kind == 1 ? (long long)((const int*)s.p)[i]
                                    : ((const long long*)s.p)[i];
    return v < 0 ? 0 : v > s.n ? s.n : (int)v;
}

__device__ __forceinline__ void bounds_of(const Segs& s, int i, int& b, int& e) {
    if (s.kind == 0) {
        b = i * s.fixed;
        e = b + s.fixed;
    } else {
        b = bound_at(s, i);
        e = bound_at(s, i + 1);
        e = e < b ? b : e;
    }
}

// The last segment that begins at or before entry i, found by a whole wave:
// each round splits what is left in 64.
__device__ __forceinline__ int segment_of(const Segs& s, int i) {
    if (s.kind == 0) return i / s.fixed;
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = s.count;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64;
        const long long at = (long long)lo + (long long)(lane + 1) * step;
        const bool below = at < hi && bound_at(s, (int)at) <= i;
        lo += __popcll(__ballot(below)) * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// What a segmented sum adds up: for entry i the row ids(i) of src, times the
// weight of entry order(i).
struct Entries {
    Ids ids;
    const int* order;     // null: entry i itself
    const float* weights; // null: ones
    const int* keys;      // entry's segment, where it is known; else null
};

// Rows in flight a lane, and as many of the next entries' indices: an index
// is on its way while the rows before it are.
constexpr int U = 4;

__device__ __forceinline__ void load_entries(const Entries& t, int i, int step,
                                             int e, int (&row)[U],
                                             float (&w)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int j = i + u * step;
        row[u] = -1;
        w[u] = 1.0f;
        if (j < e) {
            row[u] = row_of(t.ids, j);
            if (t.weights) w[u] = t.weights[t.order ? t.order[j] : j];
        }
    }
}

// Sums src's rows of entries [b, e): lane (el, g) of a team takes every
// `el_n`-th entry and the columns at `col`.
template <typename TS, int VEC>
__device__ __forceinline__ void add_entries(
        const Entries& t, const TS* src, long long ld, int col, bool live,
        int b, int e, int el, int el_n, float (&acc)[VEC]) {
    using V = Vec<TS, VEC>;
    int row[U];
    float w[U];
    int i = b + el;
    if (i >= e) return;
    load_entries(t, i, el_n, e, row, w);
    do {
        V v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u] = V{};
            if (live && row[u] >= 0)
                v[u] = load_vec<TS, VEC>(src + (long long)row[u] * ld + col);
            else
                w[u] = 0.0f;
        }
        int next[U];
        float wn[U];
        i += U * el_n;
        load_entries(t, i, el_n, e, next, wn);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                acc[k] = fmaf(w[u], (float)v[u][k], acc[k]);
            row[u] = next[u];
            w[u] = wn[u];
        }
    } while (i < e);
}

// The same with rows of eight lanes or more: each lane of a team finds one
// entry's place and weight, and hands it to the others, so that an entry's
// index work is done once and not by each lane of its row.  ONCE: no row is
// read twice, so none is to push others out of the caches.  Places are counted
// in 2^unit elements, in 32 bits.  The team is a part of a wave; `waves` of them
// take turns.
template <typename TS, int VEC, bool ONCE>
__device__ __forceinline__ void add_batches(
        const Entries& t, const TS* src, unsigned pitch, int unit, int col,
        bool live, int b, int e, int g_log, int el_log, int wave, int waves,
        float (&acc)[VEC]) {
    using V = Vec<TS, VEC>;
    constexpr unsigned ABSENT = ~0u;
    constexpr int R = 4;
    const int t_n = 1 << (g_log + el_log), lane = threadIdx.x & 63;
    const int own = lane & (t_n - 1), base = lane - own;
    const int el = own >> g_log, el_n = 1 << el_log;
    const TS* const at = src + col;
    const auto find = [&](int j, unsigned& place, float& w) {
        place = ABSENT;
        w = 1.0f;
        if (j < e) {
            const int row = row_of(t.ids, j);
            if (row >= 0) place = (unsigned)row * pitch;
            if (t.weights) w = t.weights[t.order ? t.order[j] : j];
        }
    };
    int i = b + wave * t_n;
    unsigned place;
    float w;
    find(i + own, place, w);
    for (; i < e; i += waves * t_n) {
        unsigned next;
        float wn;
        find(i + waves * t_n + own, next, wn);
        const int m = min(t_n, e - i);
        for (int j = el; j - el < m; j += R * el_n) {
            V v[R];
            float f[R];
#pragma unroll
            for (int u = 0; u < R; ++u) {
                const int k = j + u * el_n;
                const unsigned p = __shfl((int)place, base + (k & (t_n - 1)), 64);
                f[u] = __shfl(w, base + (k & (t_n - 1)), 64);
                v[u] = V{};
                if (live && k < m && p != ABSENT)
                    v[u] = load_vec<TS, VEC, ONCE>(
                        at + ((unsigned long long)p << unit));
                else
                    f[u] = 0.0f;
            }
#pragma unroll
            for (int u = 0; u < R; ++u)
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    acc[k] = fmaf(f[u], (float)v[u][k], acc[k]);
        }
        place = next;
        w = wn;
    }
}

// The same through a buffer of up to 2 GB: an entry outside the table has a
// place outside the buffer, which reads as zeros without a branch, and places
// are bytes.  Sums of 3.3 M f16 rows of 256 over 32768 bags: 127 us, against
// 193 us by add_batches, whose 34 vector instructions a load fill half the
// cycles.
template <typename TS, int VEC, bool ONCE>
__device__ __forceinline__ void add_buffered(
        const Entries& t, const TS* src, unsigned bytes, unsigned pitch, int col,
        int b, int e, int g_log, int el_log, int wave, int waves,
        float (&acc)[VEC]) {
    constexpr unsigned OUTSIDE = 0x80000000u;
    constexpr int R = 8;          // divides the lanes of a row, eight or more
    const int t_n = 1 << (g_log + el_log), lane = threadIdx.x & 63;
    const int own = lane & (t_n - 1), base = lane - own;
    const int el = own >> g_log, el_n = 1 << el_log;
    const __amdgpu_buffer_rsrc_t rows =
        __builtin_amdgcn_make_buffer_rsrc((void*)src, 0, bytes, 0x00020000);
    const unsigned at = (unsigned)col * sizeof(TS);
    const auto find = [&](int j, unsigned& place, float& w) {
        place = OUTSIDE;
        w = 0.0f;
        if (j < e) {
            const int row = row_of(t.ids, j);
            if (row >= 0) {
                place = (unsigned)row * pitch;
                w = t.weights ? t.weights[t.order ? t.order[j] : j] : 1.0f;
            }
        }
    };
    int i = b + wave * t_n;
    unsigned place;
    float w;
    find(i + own, place, w);
    for (; i < e; i += waves * t_n) {
        unsigned next;
        float wn;
        find(i + waves * t_n + own, next, wn);
        const int m = min(t_n, e - i);
        for (int j = el; j - el < m; j += R * el_n) {
            Vec<TS, VEC> v[R];
            float f[R];
#pragma unroll
            for (int u = 0; u < R; ++u) {
                const int from = base + j + u * el_n;
                const unsigned p = (unsigned)__shfl((int)place, from, 64) + at;
                f[u] = __shfl(w, from, 64);
                v[u] = load_buffer<TS, VEC, ONCE>(rows, p);
            }
#pragma unroll
            for (int u = 0; u < R; ++u)
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    acc[k] = fmaf(f[u], (float)v[u][k], acc[k]);
        }
        place = next;
        w = wn;
    }
}

// skip: how many of the columns are the neighbour's, for sums that are added.
template <typename TO, int VEC>
__device__ __forceinline__ void put_row(TO* out, const float (&acc)[VEC],
                                        float scale, int accumulate, int skip,
                                        int past) {
    float v[VEC];
    if (accumulate && skip) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (k >= skip) out[k] = (TO)fmaf(scale, acc[k], (float)out[k]);
        return;
    }
    if (accumulate) {
        load_row<TO, VEC>(out, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = fmaf(scale, acc[k], v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = scale * acc[k];
    }
    if (past)
        store_row<TO, VEC, true>(out, v);
    else
        store_row<TO, VEC>(out, v);
}

template <int VEC>
__device__ __forceinline__ void add_lanes(float (&acc)[VEC], int from, int to) {
    for (int m = from; m < to; m <<= 1)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += __shfl_xor(acc[k], m, 64);
}

// The sums of a block's four waves, each over its own lanes first, to its
// first g_n threads.
template <int VEC>
__device__ __forceinline__ void add_block(float (&acc)[VEC], int g_n,
                                          float (*red)[64 * VEC]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    add_lanes<VEC>(acc, g_n, 64);
    __syncthreads();      // the sums before these have been read
    if (wave && lane < g_n)
#pragma unroll
        for (int k = 0; k < VEC; ++k) red[wave - 1][k * 64 + lane] = acc[k];
    __syncthreads();
    if (threadIdx.x < g_n)
#pragma unroll
        for (int w = 0; w < 3; ++w)
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] += red[w][k * 64 + lane];
}

// How a call's work is cut.  A row's columns lie on g_n lanes, el_n such
// groups are a team and sum one segment; a block takes `strip` segments, in runs
// of neighbours from all over: tokens by frequency have the long ones side by
// side.  A segment over `cut` entries is summed by the whole block; one
// over `chunk` is cut into chunks, each summed by a block of its own, and
// joined by a second launch.
struct Cut {
    int g_log, el_log, strip, run_log;
    int cut, chunk, chunks;
    unsigned bytes;        // src's, where it is read through a buffer; else 0
    unsigned pitch;        // src's row pitch in bytes or in 2^unit elements; 0:
    int unit;              // by add_entries
    int by_entry;          // segments are looked for at entries, not by number
    int dp;                // pitch of part
    float* part;           // [chunks][2][dp]
    int* begins;           // [chunks]: the long segment that begins there
};

template <typename TS, typename TO>
struct Sum {
    Segs segs;
    Entries t;
    const TS* src;
    long long ld;
    TO* out;
    long long ldo;
    int D;
    float scale;
    int accumulate;
    int past;              // out is written past the caches
    Cut c;
};

// Rows of eight lanes or more have 16 bytes a lane; shorter reads are for rows of
// one lane or two.
template <typename TS, int VEC>
constexpr bool WHOLE = VEC * sizeof(TS) == 16;

// Sums entries [b, e) by teams of 2^el_log groups of lanes: by one of them, or by
// `waves` of a wave each.  el: the lane's group among the el_n of all of them.
template <typename TS, typename TO, int VEC, bool ONCE>
__device__ __forceinline__ void add_rows(const Sum<TS, TO>& a, int col, bool live,
                                         int b, int e, int el_log, int wave,
                                         int waves, int el, int el_n,
                                         float (&acc)[VEC]) {
    if constexpr (WHOLE<TS, VEC>) {
        if (a.c.bytes) {
            add_buffered<TS, VEC, ONCE>(a.t, a.src, a.c.bytes, a.c.pitch, col, b, e,
                                        a.c.g_log, el_log, wave, waves, acc);
            return;
        }
        if (a.c.pitch) {
            add_batches<TS, VEC, ONCE>(a.t, a.src, a.c.pitch, a.c.unit, col, live,
                                       b, e, a.c.g_log, el_log, wave, waves, acc);
            return;
        }
    }
    add_entries<TS, VEC>(a.t, a.src, a.ld, col, live, b, e, el, el_n, acc);
}

// Sums entries [b, e) by the whole block.
template <typename TS, typename TO, int VEC, bool ONCE>
__device__ __forceinline__ void add_by_block(const Sum<TS, TO>& a, int col,
                                             bool live, int b, int e,
                                             float (&acc)[VEC]) {
    add_rows<TS, TO, VEC, ONCE>(a, col, live, b, e, 6 - a.c.g_log,
                                threadIdx.x >> 6, 4, threadIdx.x >> a.c.g_log,
                                256 >> a.c.g_log, acc);
}

// The long segment that entry i lies in, else -1; a whole wave's work.
__device__ __forceinline__ int long_segment(const Segs& segs, const int* keys,
                                            int i, int chunk, int& b, int& e) {
    const int s = keys ? keys[i] : segment_of(segs, i);
    if (s >= segs.count) return -1;   // sorted tokens outside the table
    bounds_of(segs, s, b, e);
    return (e - b > chunk && b <= i && i < e) ? s : -1;
}

// Chunk c holds entries [c chunk, (c + 1) chunk).  Of the segments over
// `chunk` at most one comes in from the left and at most one begins in it
// (and then reaches its right end): two parts.
template <typename TS, typename TO, int VEC, bool ONCE>
__device__ void sum_chunk(const Sum<TS, TO>& a, int c, float (*red)[64 * VEC]) {
    __shared__ int found[2][3];
    const int g_n = 1 << a.c.g_log, wave = threadIdx.x >> 6;
    const int place = blockIdx.y * g_n + (threadIdx.x & (g_n - 1));
    const int col = column_of<VEC>(place, a.D);
    const bool live = place * VEC < a.D;
    const int i0 = c * a.c.chunk;
    const int i1 = (int)min((long long)a.segs.n, (long long)i0 + a.c.chunk);
    if (wave < 2) {
        int b = 0, e = 0;
        int s = long_segment(a.segs, a.t.keys, wave ? i1 - 1 : i0, a.c.chunk, b, e);
        if ((b >= i0) != (wave == 1)) s = -1;
        found[wave][0] = s;
        found[wave][1] = max(b, i0);
        found[wave][2] = min(e, i1);
    }
    __syncthreads();
    if (threadIdx.x == 0 && blockIdx.y == 0) a.c.begins[c] = found[1][0];
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
        if (found[side][0] < 0) continue;
        float acc[VEC] = {};
        add_by_block<TS, TO, VEC, ONCE>(a, col, live, found[side][1],
                                        found[side][2], acc);
        add_block<VEC>(acc, g_n, red);
        if (threadIdx.x < g_n && live)
            store_row<float, VEC>(
                a.c.part + ((long long)c * 2 + side) * a.c.dp + col, acc);
    }
}

template <typename TS, typename TO, int VEC, bool ONCE>
__global__ __launch_bounds__(256, 5)
void segment_sum_kernel(Sum<TS, TO> a) {
    __shared__ float red[3][64 * VEC];
    // the strip's segments: number, first and last entry; those for a team
    // from the front, those for the block from the back
    __shared__ int seg[64], from[64], to[64], teams_share, blocks_share;
    __shared__ unsigned long long empty;
    if ((int)blockIdx.x < a.c.chunks) {
        sum_chunk<TS, TO, VEC, ONCE>(a, blockIdx.x, red);
        return;
    }
    const int block = blockIdx.x - a.c.chunks, blocks = gridDim.x - a.c.chunks;
    const int run = a.c.run_log;
    const auto place = [=](int r) {
        return (((long long)block + (long long)(r >> run) * blocks) << run) +
               (r & ((1 << run) - 1));
    };
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        long long s = place(lane);
        bool mine = lane < a.c.strip;
        if (a.c.by_entry) {
            // the first entry of a token stands for it
            const long long i = s;
            mine = mine && i < a.segs.n &&
                   (i == 0 || a.t.keys[i] != a.t.keys[i - 1]);
            s = mine ? a.t.keys[i] : 0;
        }
        mine = mine && s < a.segs.count;
        int b = 0, e = 0;
        if (mine) bounds_of(a.segs, (int)s, b, e);
        const bool some = mine && e > b && e - b <= a.c.chunk;
        const bool one = some && e - b <= a.c.cut, all = some && !one;
        const unsigned long long ones = __ballot(one), alls = __ballot(all);
        const unsigned long long below = (1ull << lane) - 1;
        if (some) {
            const int at = one ? __popcll(ones & below)
                               : 63 - __popcll(alls & below);
            seg[at] = (int)s;
            from[at] = b;
            to[at] = e;
        }
        const unsigned long long none = __ballot(mine && e == b);
        if (lane == 0) {
            teams_share = __popcll(ones);
            blocks_share = __popcll(alls);
            empty = a.accumulate ? 0 : none;
        }
    }
    __syncthreads();

    const int g_n = 1 << a.c.g_log, el_n = 1 << a.c.el_log;
    const int team_log = a.c.g_log + a.c.el_log;
    const int place_in_row = blockIdx.y * g_n + (threadIdx.x & (g_n - 1));
    const int block_el = threadIdx.x >> a.c.g_log, block_el_n = 256 >> a.c.g_log;
    const int el = block_el & (el_n - 1);
    const int col = column_of<VEC>(place_in_row, a.D);
    const bool live = place_in_row * VEC < a.D;
    const int skip = place_in_row * VEC - col;
    if (empty && live) {
        const float zero[VEC] = {};
        for (int r = block_el; r < a.c.strip; r += block_el_n)
            if (empty >> r & 1)
                put_row<TO, VEC>(a.out + place(r) * a.ldo + col, zero, 0.0f, 0, 0,
                                 a.past);
    }
    for (int k = threadIdx.x >> team_log; k < teams_share; k += 256 >> team_log) {
        float acc[VEC] = {};
        add_rows<TS, TO, VEC, ONCE>(a, col, live, from[k], to[k], a.c.el_log, 0, 1,
                                    el, el_n, acc);
        add_lanes<VEC>(acc, g_n, g_n * el_n);
        if (live && el == 0)
            put_row<TO, VEC>(a.out + (long long)seg[k] * a.ldo + col, acc,
                             a.scale, a.accumulate, skip, a.past);
    }
#pragma unroll 1
    for (int k = 63; k > 63 - blocks_share; --k) {
        float acc[VEC] = {};
        add_by_block<TS, TO, VEC, ONCE>(a, col, live, from[k], to[k], acc);
        add_block<VEC>(acc, g_n, red);
        if (live && threadIdx.x < g_n)
            put_row<TO, VEC>(a.out + (long long)seg[k] * a.ldo + col, acc,
                             a.scale, a.accumulate, skip, a.past);
    }
}

// Joins a long segment's parts: the block of the chunk that it begins in.
template <typename TO, int VEC>
__global__ __launch_bounds__(256)
void segment_join_kernel(Segs segs, Cut c, TO* __restrict__ out, long long ldo,
                         int D, float scale, int accumulate) {
    __shared__ float red[3][64 * VEC];
    const int s = c.begins[blockIdx.x];
    if (s < 0) return;
    int b, e;
    bounds_of(segs, s, b, e);
    const int last = (e - 1) / c.chunk;
    const int g_n = 1 << c.g_log, el_n = 256 >> c.g_log;
    const int place = blockIdx.y * g_n + (threadIdx.x & (g_n - 1));
    const int el = threadIdx.x >> c.g_log, col = column_of<VEC>(place, D);
    const bool live = place * VEC < D;
    float acc[VEC] = {};
    if (live) {
        const float* first = c.part + (long long)blockIdx.x * 2 * c.dp + col;
        if (el == 0) load_row<float, VEC>(first + c.dp, acc);
#pragma unroll 4
        for (int k = 1 + el; k <= last - (int)blockIdx.x; k += el_n) {
            float v[VEC];
            load_row<float, VEC>(first + (long long)k * 2 * c.dp, v);
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] += v[q];
        }
    }
    add_block<VEC>(acc, g_n, red);
    if (live && threadIdx.x < g_n)
        put_row<TO, VEC>(out + (long long)s * ldo + col, acc, scale, accumulate,
                         place * VEC - col, 0);
}

// The output's vectors in one line, 1024 a block, whatever a row's length:
// rows that end inside a cache line are written along with the next.
template <typename T, int VEC, bool PAST>
__global__ __launch_bounds__(256)
void lookup_kernel(Ids ids, long long vectors, const T* __restrict__ src,
                   long long ld, T* __restrict__ out, int D, unsigned cols,
                   unsigned magic, float scale) {
    using V = Vec<T, VEC>;
    constexpr int N = 4;
    const long long first = (long long)blockIdx.x * (256 * N);
    const long long row0 = first / cols;
    const unsigned rest = (unsigned)(first - row0 * cols);
    V v[N];
    long long to[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const unsigned at = rest + u * 256 + threadIdx.x;
        // magic: 2^32 / cols, rounded up; exact as long as at cols < 2^32
        const unsigned r = magic ? __umulhi(at, magic) : at / cols;
        const int col = column_of<VEC>(at - r * cols, D);
        to[u] = (row0 + r) * D + col;
        v[u] = V{};
        if (first + u * 256 + threadIdx.x < vectors) {
            const int row = row_of(ids, row0 + r);
            if (row >= 0)
                v[u] = load_vec<T, VEC>(src + (long long)row * ld + col);
        }
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const long long i = first + u * 256 + threadIdx.x;
        if (i < vectors) {
            float f[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) f[k] = (float)v[u][k] * scale;
            store_row<T, VEC, PAST>(out + to[u], f);
        }
    }
}

// Bytes that no longer lie in the card's L2s (32 MB) when they are wanted.
constexpr long long LARGE = 32 << 20;

int log2_up(int x, int most) {
    int l = 0;
    while (l < most && (1 << l) < x) ++l;
    return l;
}

enum { F32 = 0, BF16 = 1, F16 = 2 };

struct SumCall {
    Segs segs;
    Entries t;
    const void* src;
    long long ld;
    void* out;
    long long ldo;
    void* work;
    int D;
    float scale;
    int accumulate;
    bool once;
    hipStream_t stream;
};

// Lanes a row; entries a chunk: 32 a lane of the block, at most 512.
// A row of 75 lanes is three times 32 of them rather than twice 64.
int lanes_log(int D, int vec) {
    const int cols = (D + vec - 1) / vec;
    if (cols > 64 && (cols + 31) / 32 * 5 <= (cols + 63) / 64 * 8) return 5;
    return log2_up(cols, 6);
}
// A gradient of up to 1024 tokens has none: 777 of 100 f32 take 11.1 us, sort
// included, without the join's launch and 12.4 us with it, and the host's part
// of a launch goes too.  Where all 1024 are one token, of 512 f32, its block
// takes 25 us alone, against 14 us.
int chunk_of(int D, int vec, int n, bool sorted) {
    if (sorted && n <= 1024) return 1024;
    const int c = 8192 >> lanes_log(D, vec);
    return c < 512 ? c : 512;
}

template <typename TS, typename TO, int VEC>
int segment_sum(const SumCall& a) {
    const int cols = (a.D + VEC - 1) / VEC;
    Cut c;
    c.g_log = lanes_log(a.D, VEC);
    const int slices = (cols + (1 << c.g_log) - 1) >> c.g_log;
    c.chunk = chunk_of(a.D, VEC, a.segs.n, a.t.keys);
    c.unit = 0;
    while (c.unit < 6 && a.ld && !(a.ld >> c.unit & 1)) ++c.unit;
    const long long pitch = a.ld >> c.unit;
    c.pitch = WHOLE<TS, VEC> && c.g_log >= 3 &&
                      pitch * a.t.ids.rows < 0xffffffffll
                  ? (unsigned)pitch : 0;
    // through a buffer: up to 2 GB, at whole words
    const long long bytes =
        ((a.t.ids.rows - 1) * a.ld + a.D) * (long long)sizeof(TS);
    c.bytes = 0;
    if (c.pitch && bytes <= 0x7fffffffll &&
        ((uintptr_t)a.src | a.ld * sizeof(TS) | a.D * sizeof(TS)) % 4 == 0) {
        c.bytes = (unsigned)bytes;
        c.pitch = (unsigned)(a.ld * sizeof(TS));
    }
    const bool some_long = a.segs.n > c.chunk &&
                           !(a.segs.kind == 0 && a.segs.fixed <= c.chunk);
    c.chunks = some_long ? (int)(((long long)a.segs.n + c.chunk - 1) / c.chunk) : 0;
    c.dp = (a.D + 7) & ~7;
    c.part = (float*)a.work;
    c.begins = (int*)(c.part + (long long)c.chunks * 2 * c.dp);
    c.by_entry = a.accumulate && a.t.keys && a.segs.n < a.segs.count;
    const long long places = c.by_entry ? a.segs.n : a.segs.count;

    // Lanes that are left over share a segment's entries, up to one for each
    // four that a segment has on average.  Where waves of such teams do not
    // fill the card, the whole block is a team.
    const long long mean = a.segs.n / a.segs.count;
    const int share = (int)(mean / 4 < 64 ? mean / 4 : 64);
    c.el_log = log2_up(share, 6 - c.g_log);
    const long long waves = (places << (c.g_log + c.el_log)) / 64;
    const bool block_team = (share >> c.el_log) > 1 && waves < 8192;
    // A block's segments: four times as many blocks as the card holds, to even
    // out their lengths; where most segments are empty, one time.
    long long strip = places / (mean ? 4096 : 1024) / 8 * 8;
    strip = strip < 8 ? 8 : strip > 64 ? 64 : strip;
    c.strip = block_team ? 1 : (int)strip;
    // a run's rows are 64 bytes or more, to be written whole
    c.run_log = 0;
    while ((long long)a.D * sizeof(TO) << c.run_log < 64 &&
           2 << c.run_log <= c.strip) ++c.run_log;
    c.strip &= -1 << c.run_log;
    // A segment stays with its team up to twice what a team sums on average
    // on a full card (some 20 waves a compute unit), or four times the mean
    // segment; a longer one would be the call's tail.
    const long long full = 256 * 20 * 64 >> (c.g_log + c.el_log);
    long long cut = 2 * (a.segs.n / full);
    if (cut < 4 * mean) cut = 4 * mean;
    if (cut < (2 * U) << c.el_log) cut = (2 * U) << c.el_log;
    c.cut = (int)(cut < c.chunk ? cut : c.chunk);
    if (block_team) c.cut = 0;

    const long long blocks = c.chunks + (places + c.strip - 1) / c.strip;
    // Past the caches: a gradient of many rows, and rows of which each is read
    // once.  1048576 x 256 bf16 onto 100000 rows take 161 us through the caches,
    // 149 us with the writes past them, 137 us with the reads too.
    const int past = !a.accumulate &&
                     (long long)a.segs.count * a.D * sizeof(TO) >= LARGE;
    const bool once = c.pitch && a.once &&
                      (long long)a.segs.n * a.D * sizeof(TS) >= LARGE;
    const Sum<TS, TO> s{a.segs, a.t, (const TS*)a.src, a.ld, (TO*)a.out, a.ldo,
                        a.D, a.scale, a.accumulate, past, c};
    auto* kernel = segment_sum_kernel<TS, TO, VEC, false>;
    if constexpr (WHOLE<TS, VEC>)
        if (once) kernel = segment_sum_kernel<TS, TO, VEC, true>;
    kernel<<<dim3((unsigned)blocks, slices), 256, 0, a.stream>>>(s);
    if (c.chunks)
        segment_join_kernel<TO, VEC><<<dim3(c.chunks, slices), 256, 0,
            a.stream>>>(a.segs, c, (TO*)a.out, a.ldo, a.D, a.scale,
                        a.accumulate);
    return (int)hipGetLastError();
}

template <typename TS, typename TO>
int sum_by_width(const SumCall& c, int vec) {
    switch (vec) {
        case 1: return segment_sum<TS, TO, 1>(c);
        case 2: return segment_sum<TS, TO, 2>(c);
        case 4: return segment_sum<TS, TO, 4>(c);
        default:
            if constexpr (sizeof(TS) == 2) return segment_sum<TS, TO, 8>(c);
            return (int)hipErrorInvalidValue;
    }
}

template <typename TS>
int sum_by_out(const SumCall& c, int out_type, int vec) {
    switch (out_type) {
        case F32: return sum_by_width<TS, float>(c, vec);
        case BF16: return sum_by_width<TS, __bf16>(c, vec);
        default: return sum_by_width<TS, _Float16>(c, vec);
    }
}

template <typename T, int VEC>
int lookup(const Ids& ids, long long n, const void* src, long long ld,
           void* out, int D, float scale, hipStream_t stream) {
    const unsigned cols = (D + VEC - 1) / VEC;
    const unsigned magic = cols == 1 || cols > 32768
                               ? 0 : (unsigned)((1ull << 32) / cols) + 1;
    // 268 MB of rows past the caches leave the table there: 55 us against 88;
    // what fits the caches is left there for its reader
    auto* kernel = n * D * (long long)sizeof(T) >= LARGE
                       ? lookup_kernel<T, VEC, true> : lookup_kernel<T, VEC, false>;
    // a launch has fewer than 2^32 threads, a quarter of its vectors
    const long long most = (1ll << 33) / cols;
    for (long long at = 0; at < n; at += most) {
        const long long vectors = (n - at < most ? n - at : most) * cols;
        const Ids some{(const char*)ids.p + at * (ids.wide ? 8 : 4), ids.wide,
                       ids.rows};
        kernel<<<(unsigned)((vectors + 1023) / 1024), 256, 0, stream>>>(
            some, vectors, (const T*)src, ld, (T*)out + at * D, D, cols, magic,
            scale);
    }
    return (int)hipGetLastError();
}

template <typename T>
int lookup_by_width(const Ids& ids, long long n, const void* src, long long ld,
                    void* out, int D, float scale, int vec, hipStream_t st) {
    switch (vec) {
        case 1: return lookup<T, 1>(ids, n, src, ld, out, D, scale, st);
        case 2: return lookup<T, 2>(ids, n, src, ld, out, D, scale, st);
        case 4: return lookup<T, 4>(ids, n, src, ld, out, D, scale, st);
        default:
            if constexpr (sizeof(T) == 2)
                return lookup<T, 8>(ids, n, src, ld, out, D, scale, st);
            return (int)hipErrorInvalidValue;
    }
}

}  // namespace

// Y[n, D] = scale * T[ids], T [V, D] with row pitch ld.  vec: elements a lane,
// a power of two, at most D and 16 bytes.
KS_EXPORT int ks_embedding_lookup(const void* ids, int ids_wide, long long n,
                                  const void* table, int type, long long V,
                                  long long ld, void* out, int D, float scale,
                                  int vec, hipStream_t stream) {
    if (n == 0 || D == 0) return 0;
    if (!ids || !out || (V && !table)) return (int)hipErrorInvalidValue;
    const Ids t{ids, ids_wide, V};
    switch (type) {
        case F32: return lookup_by_width<float>(t, n, table, ld, out, D, scale, vec, stream);
        case BF16: return lookup_by_width<__bf16>(t, n, table, ld, out, D, scale, vec, stream);
        default: return lookup_by_width<_Float16>(t, n, table, ld, out, D, scale, vec, stream);
    }
}

// How many floats of workspace a segmented sum of n entries needs.
// sorted: entries come with keys.
KS_EXPORT long long ks_segment_work(int n, int D, int vec, int sorted) {
    const int chunk = chunk_of(D, vec, n, sorted);
    if (n <= chunk) return 0;
    return ((long long)n + chunk - 1) / chunk * (2 * ((D + 7) & ~7) + 1);
}

// out[count, D] (pitch ldo) = scale * sums of src's rows over segments.
// kind/bounds/fixed: the segments; ids: each entry's row of src [V, D] (pitch
// ld); order, weights, keys may be null.  work: ks_segment_work() floats.
KS_EXPORT int ks_segment_sum(int kind, const void* bounds, int fixed,
                             int count, int n, const void* ids, int ids_wide,
                             long long V, const int* order,
                             const float* weights, const int* keys,
                             const void* src, int type, long long ld,
                             void* out, int out_type, long long ldo,
                             void* work, int D, float scale, int accumulate,
                             int vec, hipStream_t stream) {
    if (count == 0 || D == 0) return 0;
    if (!out || (n && !ids) || (V && !src) || (kind && !bounds) ||
        (!work && ks_segment_work(n, D, vec, keys != nullptr)))
        return (int)hipErrorInvalidValue;
    const SumCall c{{bounds, kind, fixed, count, n},
                    {{ids, ids_wide, V}, order, weights, keys},
                    src, ld, out, ldo, work, D, scale, accumulate,
                    order && ids == (const void*)order, stream};
    switch (type) {
        case F32: return sum_by_out<float>(c, out_type, vec);
        case BF16: return sum_by_out<__bf16>(c, out_type, vec);
        default: return sum_by_out<_Float16>(c, out_type, vec);
    }
}
