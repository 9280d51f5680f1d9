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
#include "common.h"

#include <cstdint>

namespace {

template <typename T, int N>
using Vec = T __attribute__((ext_vector_type(N)));

template <typename T, int N>
__device__ __forceinline__ void load_row(const T* p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = (float)p[0];
    } else {
        const Vec<T, N> x = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)x[i];
    }
}

template <typename T, int N>
__device__ __forceinline__ void store_row(T* p, const float (&v)[N]) {
    if constexpr (N == 1) {
        p[0] = (T)v[0];
    } else {
        Vec<T, N> x;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (T)v[i];
        *reinterpret_cast<Vec<T, N>*>(p) = x;
    }
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

// The last segment that begins at or before entry i.
__device__ __forceinline__ int segment_of(const Segs& s, int i) {
    if (s.kind == 0) return i / s.fixed;
    int lo = 0, hi = s.count;
    while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        if (bound_at(s, mid) <= i) lo = mid; else hi = mid;
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

// Sums src's rows of entries [b, e): lane (el, g) of a team takes every
// `el_n`-th entry and the columns at `col`.  Four rows are in flight a lane.
template <typename TS, int VEC>
__device__ __forceinline__ void add_entries(
        const Entries& t, const TS* src, long long ld, int col, bool live,
        int b, int e, int el, int el_n, float (&acc)[VEC]) {
    constexpr int U = 4;
    for (int i = b + el; i < e; i += U * el_n) {
        int row[U];
        float w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = i + u * el_n;
            row[u] = -1;
            w[u] = 1.0f;
            if (j < e) {
                row[u] = row_of(t.ids, j);
                if (t.weights) w[u] = t.weights[t.order ? t.order[j] : j];
            }
        }
        float v[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (live && row[u] >= 0) {
                load_row<TS, VEC>(src + (long long)row[u] * ld + col, v[u]);
            } else {
                w[u] = 0.0f;
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[u][k] = 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] = fmaf(w[u], v[u][k], acc[k]);
    }
}

template <typename TO, int VEC>
__device__ __forceinline__ void put_row(TO* out, const float (&acc)[VEC],
                                        float scale, int accumulate) {
    float v[VEC];
    if (accumulate) {
        load_row<TO, VEC>(out, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = fmaf(scale, acc[k], v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = scale * acc[k];
    }
    store_row<TO, VEC>(out, v);
}

// A segment over LONG entries is cut into chunks of LONG, each summed by a
// wave of its own, and joined afterwards.
constexpr int LONG = 128;

// One team of g_n * el_n lanes a segment.
template <typename TS, typename TO, int VEC>
__global__ __launch_bounds__(256)
void segment_sum_kernel(Segs segs, Entries t, const TS* __restrict__ src,
                        long long ld, TO* __restrict__ out, long long ldo,
                        int D, int g_log, int el_log, float scale,
                        int accumulate) {
    const int g_n = 1 << g_log, el_n = 1 << el_log;
    const int lane = threadIdx.x;
    const int g = lane & (g_n - 1), el = (lane >> g_log) & (el_n - 1);
    const int team = lane >> (g_log + el_log), teams = 256 >> (g_log + el_log);
    const int col = (blockIdx.y * g_n + g) * VEC;
    const bool live = col < D;
    for (long long s = (long long)blockIdx.x * teams + team; s < segs.count;
         s += (long long)gridDim.x * teams) {
        int b, e;
        bounds_of(segs, (int)s, b, e);
        if (e - b > LONG || (accumulate && e == b)) continue;
        float acc[VEC] = {};
        add_entries<TS, VEC>(t, src, ld, col, live, b, e, el, el_n, acc);
        for (int m = g_n; m < g_n * el_n; m <<= 1)
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] += __shfl_xor(acc[k], m, 64);
        if (live && el == 0)
            put_row<TO, VEC>(out + s * ldo + col, acc, scale, accumulate);
    }
}

// The segment that entry i lies in, if it is longer than LONG; else -1.
__device__ __forceinline__ int long_segment(const Segs& segs, const int* keys,
                                            int i, int& b, int& e) {
    const int s = keys ? keys[i] : segment_of(segs, i);
    if (s >= segs.count) return -1;   // sorted tokens outside the table
    bounds_of(segs, s, b, e);
    return (e - b > LONG && b <= i && i < e) ? s : -1;
}

// Chunk c holds entries [c LONG, (c + 1) LONG).  Of the segments over LONG
// at most one comes in from the left and at most one begins in it (and then
// reaches its right end): two parts of part[c][2][dp].
template <typename TS, int VEC>
__global__ __launch_bounds__(256)
void long_part_kernel(Segs segs, Entries t, const TS* __restrict__ src,
                      long long ld, float* __restrict__ part, int dp, int D,
                      int g_log, int chunks) {
    const int c = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (c >= chunks) return;
    const int g_n = 1 << g_log, el_n = 64 >> g_log;
    const int g = lane & (g_n - 1), el = lane >> g_log;
    const int col = (blockIdx.y * g_n + g) * VEC;
    const bool live = col < D;
    const int i0 = c * LONG, i1 = min(segs.n, i0 + LONG);
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
        int b, e;
        const int s = long_segment(segs, t.keys, side ? i1 - 1 : i0, b, e);
        if (s < 0 || (b >= i0) != (side == 1)) continue;
        float acc[VEC] = {};
        add_entries<TS, VEC>(t, src, ld, col, live, max(b, i0), min(e, i1),
                             el, el_n, acc);
        for (int m = g_n; m < 64; m <<= 1)
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] += __shfl_xor(acc[k], m, 64);
        if (live && el == 0)
            store_row<float, VEC>(part + ((long long)c * 2 + side) * dp + col,
                                  acc);
    }
}

// Joins a long segment's parts: the block of the chunk that it begins in
// adds them, every el_n-th by one row of threads, then the rows in LDS.
template <typename TO, int VEC>
__global__ __launch_bounds__(256)
void long_join_kernel(Segs segs, const int* keys,
                      const float* __restrict__ part, int dp,
                      TO* __restrict__ out, long long ldo, int D, int g_log,
                      float scale, int accumulate) {
    __shared__ float red[256 * VEC];
    const int c = blockIdx.x, i0 = c * LONG, i1 = min(segs.n, i0 + LONG);
    int b, e;
    const int s = long_segment(segs, keys, i1 - 1, b, e);
    if (s < 0 || b < i0) return;
    const int last = (e - 1) / LONG;
    const int g_n = 1 << g_log, el_n = 256 >> g_log;
    const int g = threadIdx.x & (g_n - 1), el = threadIdx.x >> g_log;
    const int col = (blockIdx.y * g_n + g) * VEC;
    const bool live = col < D;
    float acc[VEC] = {};
    if (live) {
        if (el == 0)
            load_row<float, VEC>(part + ((long long)c * 2 + 1) * dp + col, acc);
#pragma unroll 4
        for (int k = c + 1 + el; k <= last; k += el_n) {
            float v[VEC];
            load_row<float, VEC>(part + (long long)k * 2 * dp + col, v);
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] += v[q];
        }
    }
#pragma unroll
    for (int q = 0; q < VEC; ++q) red[q * 256 + threadIdx.x] = acc[q];
    for (int half = el_n >> 1; half; half >>= 1) {
        __syncthreads();
        if (el < half)
#pragma unroll
            for (int q = 0; q < VEC; ++q)
                red[q * 256 + threadIdx.x] +=
                    red[q * 256 + threadIdx.x + half * g_n];
    }
    if (live && el == 0) {
#pragma unroll
        for (int q = 0; q < VEC; ++q) acc[q] = red[q * 256 + threadIdx.x];
        put_row<TO, VEC>(out + (long long)s * ldo + col, acc, scale, accumulate);
    }
}

// One team of g_n lanes a row, four rows in flight.
template <typename T, int VEC>
__global__ __launch_bounds__(256)
void lookup_kernel(Ids ids, long long n, const T* __restrict__ src,
                   long long ld, T* __restrict__ out, int D, int g_log,
                   float scale) {
    constexpr int U = 4;
    const int g_n = 1 << g_log, g = threadIdx.x & (g_n - 1);
    const int col = (blockIdx.y * g_n + g) * VEC;
    if (col >= D) return;
    const long long teams = 256 >> g_log;
    const long long first = (long long)blockIdx.x * teams * U +
                            (threadIdx.x >> g_log);
    int row[U];
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = first + u * teams;
        row[u] = i < n ? row_of(ids, i) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[u][k] = 0.0f;
        if (row[u] >= 0)
            load_row<T, VEC>(src + (long long)row[u] * ld + col, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = first + u * teams;
        if (i < n) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[u][k] *= scale;
            store_row<T, VEC>(out + i * D + col, v[u]);
        }
    }
}

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
    float* part;
    int D;
    float scale;
    int accumulate;
    hipStream_t stream;
};

template <typename TS, typename TO, int VEC>
int segment_sum(const SumCall& c) {
    const int cols = (c.D + VEC - 1) / VEC;
    const int g_log = log2_up(cols, 6), slices = (cols + (1 << g_log) - 1) >> g_log;
    // lanes that are left over share a segment's entries, up to one for each
    // four that a segment has on average
    const long long mean = c.segs.n / c.segs.count;
    const int el_log = log2_up((int)(mean / 4 < 64 ? mean / 4 : 64), 6 - g_log);
    const long long teams = 256 >> (g_log + el_log);
    long long blocks = (c.segs.count + teams - 1) / teams;
    if (blocks > (1 << 20)) blocks = 1 << 20;
    const TS* src = (const TS*)c.src;
    TO* out = (TO*)c.out;
    segment_sum_kernel<TS, TO, VEC><<<dim3((unsigned)blocks, slices), 256, 0,
        c.stream>>>(c.segs, c.t, src, c.ld, out, c.ldo, c.D, g_log, el_log,
                    c.scale, c.accumulate);
    if (c.segs.n > LONG && !(c.segs.kind == 0 && c.segs.fixed <= LONG)) {
        const int chunks = (c.segs.n + LONG - 1) / LONG;
        const int dp = (c.D + 3) & ~3;
        long_part_kernel<TS, VEC><<<dim3((chunks + 3) / 4, slices), 256, 0,
            c.stream>>>(c.segs, c.t, src, c.ld, c.part, dp, c.D, g_log, chunks);
        long_join_kernel<TO, VEC><<<dim3(chunks, slices), 256, 0, c.stream>>>(
            c.segs, c.t.keys, c.part, dp, out, c.ldo, c.D, g_log, c.scale,
            c.accumulate);
    }
    return (int)hipGetLastError();
}

template <typename TS, typename TO>
int sum_by_width(const SumCall& c, int vec) {
    switch (vec) {
        case 1: return segment_sum<TS, TO, 1>(c);
        case 2: return segment_sum<TS, TO, 2>(c);
        default: return segment_sum<TS, TO, 4>(c);
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
    const int cols = (D + VEC - 1) / VEC;
    const int g_log = log2_up(cols, 6), slices = (cols + (1 << g_log) - 1) >> g_log;
    const long long rows = (256 >> g_log) * 4;
    lookup_kernel<T, VEC><<<dim3((unsigned)((n + rows - 1) / rows), slices),
        256, 0, stream>>>(ids, n, (const T*)src, ld, (T*)out, D, g_log, scale);
    return (int)hipGetLastError();
}

template <typename T>
int lookup_by_width(const Ids& ids, long long n, const void* src, long long ld,
                    void* out, int D, float scale, int vec, hipStream_t st) {
    switch (vec) {
        case 1: return lookup<T, 1>(ids, n, src, ld, out, D, scale, st);
        case 2: return lookup<T, 2>(ids, n, src, ld, out, D, scale, st);
        default: return lookup<T, 4>(ids, n, src, ld, out, D, scale, st);
    }
}

}  // namespace

// Y[n, D] = scale * T[ids], T [V, D] with row pitch ld.  vec: how many
// elements every row of T and Y can be read by at once.
KS_EXPORT int ks_embedding_lookup(const void* ids, int ids_wide, long long n,
                                  const void* table, int type, long long V,
                                  long long ld, void* out, int D, float scale,
                                  int vec, hipStream_t stream) {
    if (n == 0 || D == 0) return 0;
    const Ids t{ids, ids_wide, V};
    switch (type) {
        case F32: return lookup_by_width<float>(t, n, table, ld, out, D, scale, vec, stream);
        case BF16: return lookup_by_width<__bf16>(t, n, table, ld, out, D, scale, vec, stream);
        default: return lookup_by_width<_Float16>(t, n, table, ld, out, D, scale, vec, stream);
    }
}

KS_EXPORT int ks_segment_long() { return LONG; }

// out[count, D] (pitch ldo) = scale * sums of src's rows over segments.
// kind/bounds/fixed: the segments; ids: each entry's row of src [V, D] (pitch
// ld); order, weights, keys may be null.  part: two rows of ceil4(D) floats
// for every ks_segment_long() entries; may be null for at most that many.
KS_EXPORT int ks_segment_sum(int kind, const void* bounds, int fixed,
                             int count, int n, const void* ids, int ids_wide,
                             long long V, const int* order,
                             const float* weights, const int* keys,
                             const void* src, int type, long long ld,
                             void* out, int out_type, long long ldo,
                             float* part, int D, float scale, int accumulate,
                             int vec, hipStream_t stream) {
    if (count == 0 || D == 0) return 0;
    const SumCall c{{bounds, kind, fixed, count, n},
                    {{ids, ids_wide, V}, order, weights, keys},
                    src, ld, out, ldo, part, D, scale, accumulate, stream};
    switch (type) {
        case F32: return sum_by_out<float>(c, out_type, vec);
        case BF16: return sum_by_out<__bf16>(c, out_type, vec);
        default: return sum_by_out<_Float16>(c, out_type, vec);
    }
}
