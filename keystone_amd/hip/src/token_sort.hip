// A stable sort of token positions by token id, for the embedding gradient:
// sums over a token's occurrences then run over one stretch, in ascending
// order of their positions.
//
// Radix sort from the lowest digit, at most nine bits a digit.  A digit's
// pass counts the digits of every tile of 2048 tokens, scans the counts over
// the tiles, and moves each token to its digit's place.  Inside a wave the
// tokens of one digit are found by a ballot over each of its bits, so that
// equal digits keep their order without atomics.  A tile is put in order in
// LDS first, so that what it writes of one digit is one run.
//
// Bound by latency and launches: 1048576 tokens of 100000 take 57 us in eight
// launches (78 us with scattered writes of 4 bytes), 8388608 take 198 us, 777
// take 12 us in two.
#include "common.h"

#include <cstdint>

namespace {

constexpr int TILE = 2048, WAVES = 4, ROUNDS = TILE / (WAVES * 64);
constexpr int MAX_BITS = 9, MAX_BINS = 1 << MAX_BITS;

// The bag of position i: -1 where the bounds leave it out.  lo, hi: a bag that
// begins at or before i, and one after it or `bags`.
__device__ __forceinline__ int bag_of(const void* bounds, int kind, int fixed,
                                      int bags, int i, int lo, int hi) {
    if (kind == 0) return i / fixed;
    if (bags == 0) return -1;
    auto at = [&](int k) -> long long {
        return kind == 1 ? (long long)((const int*)bounds)[k]
                         : ((const long long*)bounds)[k];
    };
    while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        if (at(mid) <= i) lo = mid; else hi = mid;
    }
    return (at(lo) <= i && i < at(lo + 1)) ? lo : -1;
}

// What a pass reads: the token ids themselves, or (key, position) pairs.  A
// key is the id, or V for one outside the table or outside every bag.
struct Source {
    const int2* pairs;
    const void* ids;
    int wide, n, V;
    const int* bag;    // the positions' bags, where there are bags
};

__device__ __forceinline__ int2 pair_at(const Source& s, int i) {
    if (s.pairs) return s.pairs[i];
    const long long v = s.wide ? ((const long long*)s.ids)[i]
                               : (long long)((const int*)s.ids)[i];
    int key = (v >= 0 && v < s.V) ? (int)v : s.V;
    if (s.bag && s.bag[i] < 0) key = s.V;
    return make_int2(key, i);
}

__global__ __launch_bounds__(256)
void position_bags_kernel(const void* __restrict__ bounds, int kind, int fixed,
                          int bags, int n, int* __restrict__ bag) {
    // the bags of the block's ends, then each position's between them
    __shared__ int ends[2];
    const long long first = (long long)blockIdx.x * TILE;
    if (kind && bags && (threadIdx.x & 63) == 0 && threadIdx.x < 128) {
        const bool last = threadIdx.x;
        const long long i = last ? min(first + TILE, (long long)n) - 1 : first;
        int lo = 0, hi = bags;
        while (hi - lo > 1) {
            const int mid = lo + (hi - lo) / 2;
            const long long v = kind == 1 ? (long long)((const int*)bounds)[mid]
                                          : ((const long long*)bounds)[mid];
            if (v <= i) lo = mid; else hi = mid;
        }
        ends[last] = lo + last;
    }
    __syncthreads();
    for (int r = 0; r < TILE / 256; ++r) {
        const long long i = first + r * 256 + threadIdx.x;
        if (i < n)
            bag[i] = bag_of(bounds, kind, fixed, bags, (int)i, ends[0], ends[1]);
    }
}

__global__ __launch_bounds__(256)
void digit_count_kernel(Source src, int shift, int bits,
                        int* __restrict__ counts, int tiles) {
    __shared__ int bin[MAX_BINS];
    const int bins = 1 << bits;
    for (int i = threadIdx.x; i < bins; i += 256) bin[i] = 0;
    __syncthreads();
    const int first = blockIdx.x * TILE;
    for (int r = 0; r < TILE / 256; ++r) {
        const int i = first + r * 256 + threadIdx.x;
        if (i < src.n) atomicAdd(&bin[(pair_at(src, i).x >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += 256)
        counts[(long long)i * tiles + blockIdx.x] = bin[i];
}

// Exclusive sums over the tiles of one digit, in place, and its total.
__global__ __launch_bounds__(256)
void digit_scan_kernel(int* __restrict__ counts, int tiles,
                       int* __restrict__ totals) {
    __shared__ int wave_sum[4];
    int* row = counts + (long long)blockIdx.x * tiles;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int carry = 0;
    for (int first = 0; first < tiles; first += 256) {
        const int i = first + threadIdx.x;
        const int x = i < tiles ? row[i] : 0;
        int s = x;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(s, d, 64);
            if (lane >= d) s += y;
        }
        if (lane == 63) wave_sum[wave] = s;
        __syncthreads();
        int before = carry, all = 0;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) before += wave_sum[w];
            all += wave_sum[w];
        }
        if (i < tiles) row[i] = before + s - x;
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// The lanes of this wave whose digit equals this lane's.
__device__ __forceinline__ unsigned long long same_digit(int digit, int bits,
                                                         bool live) {
    unsigned long long m = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long s = __ballot((digit >> b) & 1);
        m &= ((digit >> b) & 1) ? s : ~s;
    }
    return m;
}

// A wave's tokens in 64s: each one's rank among its digit's in this wave so
// far, counted in `count`.  The wave's LDS accesses run in order; the fences
// keep the compiler from moving them.
__device__ __forceinline__ int rank_digit(int digit, int bits, bool live,
                                          int* count) {
    const int lane = threadIdx.x & 63;
    const unsigned long long m = same_digit(digit, bits, live);
    const int before = __popcll(m & ((1ull << lane) - 1));
    int rank = 0;
    if (live) rank = count[digit] + before;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (live && before == 0) count[digit] += __popcll(m);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return rank;
}

// Exclusive sums over the block's 256 threads.
__device__ __forceinline__ int scan_block(int x, int* wave_sum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(s, d, 64);
        if (lane >= d) s += y;
    }
    if (lane == 63) wave_sum[wave] = s;
    __syncthreads();
    s -= x;
    for (int w = 0; w < wave; ++w) s += wave_sum[w];
    __syncthreads();
    return s;
}

// The last pass (pairs_out null) writes keys, order and rows.
__global__ __launch_bounds__(256)
void digit_move_kernel(Source src, int shift, int bits,
                       const int* __restrict__ counts, int tiles,
                       const int* __restrict__ totals,
                       int2* __restrict__ pairs_out, int* __restrict__ keys,
                       int* __restrict__ order, int* __restrict__ rows) {
    __shared__ int count[WAVES][MAX_BINS];
    __shared__ int there[MAX_BINS];   // global less local place of a digit
    __shared__ int2 sorted[TILE];
    __shared__ int wave_sum[WAVES];
    const int bins = 1 << bits;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int begin = blockIdx.x * TILE, mine = min(TILE, src.n - begin);
    const int first = wave * (ROUNDS * 64) + lane;
    int2 pair[ROUNDS];
    int rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int i = first + r * 64;
        pair[r] = i < mine ? pair_at(src, begin + i) : make_int2(0, 0);
    }
    for (int i = threadIdx.x; i < bins; i += 256)
        for (int w = 0; w < WAVES; ++w) count[w][i] = 0;
    // two digits a thread
    const int d0 = threadIdx.x * 2, d1 = d0 + 1;
    const int t0 = d0 < bins ? totals[d0] : 0, t1 = d1 < bins ? totals[d1] : 0;
    const int c0 = d0 < bins ? counts[(long long)d0 * tiles + blockIdx.x] : 0;
    const int c1 = d1 < bins ? counts[(long long)d1 * tiles + blockIdx.x] : 0;
    const int global = scan_block(t0 + t1, wave_sum);
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        rank[r] = rank_digit((pair[r].x >> shift) & (bins - 1), bits,
                             first + r * 64 < mine, count[wave]);
    __syncthreads();
    int n0 = 0, n1 = 0;
    if (d0 < bins)
        for (int w = 0; w < WAVES; ++w) n0 += count[w][d0];
    if (d1 < bins)
        for (int w = 0; w < WAVES; ++w) n1 += count[w][d1];
    const int local = scan_block(n0 + n1, wave_sum);
    if (d0 < bins) {
        there[d0] = global + c0 - local;
        int at = local;
        for (int w = 0; w < WAVES; ++w) {
            const int c = count[w][d0];
            count[w][d0] = at;
            at += c;
        }
    }
    if (d1 < bins) {
        there[d1] = global + t0 + c1 - (local + n0);
        int at = local + n0;
        for (int w = 0; w < WAVES; ++w) {
            const int c = count[w][d1];
            count[w][d1] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (first + r * 64 < mine)
            sorted[count[wave][(pair[r].x >> shift) & (bins - 1)] + rank[r]] =
                pair[r];
    __syncthreads();
    for (int i = threadIdx.x; i < mine; i += 256) {
        const int2 p = sorted[i];
        const int to = there[(p.x >> shift) & (bins - 1)] + i;
        if (pairs_out) {
            pairs_out[to] = p;
        } else {
            keys[to] = p.x;
            order[to] = p.y;
            // a token outside every bag sorts last and is never read
            if (rows) rows[to] = max(src.bag[p.y], 0);
        }
    }
}

// Up to SMALL tokens: one block sorts them in LDS, all digits in one launch.
// Each of its waves has four rounds of 64 tokens.
constexpr int SMALL = 4096, SMALL_ROUNDS = 4;

template <int SMALL_WAVES>
__global__ __launch_bounds__(64 * SMALL_WAVES)
void small_sort_kernel(const void* __restrict__ ids, int wide, int n, int V,
                       const void* __restrict__ bounds, int kind, int fixed,
                       int bags, int bits, int passes, int* __restrict__ keys,
                       int* __restrict__ order, int* __restrict__ rows) {
    constexpr int THREADS = 64 * SMALL_WAVES, MOST = THREADS * SMALL_ROUNDS;
    __shared__ int key_at[MOST], from_at[MOST];
    __shared__ int count[SMALL_WAVES][MAX_BINS];
    __shared__ int wave_sum[SMALL_WAVES];
    // digits a thread
    constexpr int EACH = THREADS < MAX_BINS ? MAX_BINS / THREADS : 1;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bins = 1 << bits;
    const int first = wave * (SMALL_ROUNDS * 64) + lane;
    int key[SMALL_ROUNDS], from[SMALL_ROUNDS], rank[SMALL_ROUNDS];
#pragma unroll
    for (int r = 0; r < SMALL_ROUNDS; ++r) {
        const int i = first + r * 64;
        from[r] = i;
        key[r] = V;
        if (i < n) {
            const long long v = wide ? ((const long long*)ids)[i]
                                     : (long long)((const int*)ids)[i];
            if (v >= 0 && v < V) key[r] = (int)v;
            if (rows && bag_of(bounds, kind, fixed, bags, i, 0, bags) < 0) key[r] = V;
        }
    }
    for (int p = 0; p < passes; ++p) {
        const int shift = p * bits;
        for (int i = tid; i < SMALL_WAVES * MAX_BINS; i += THREADS)
            (&count[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SMALL_ROUNDS; ++r)
            rank[r] = rank_digit((key[r] >> shift) & (bins - 1), bits,
                                 first + r * 64 < n, count[wave]);
        __syncthreads();
        // where each wave's tokens of each digit go
        int total[EACH], all = 0, s = 0;
        if (tid < MAX_BINS / EACH) {
#pragma unroll
            for (int q = 0; q < EACH; ++q) {
                total[q] = 0;
                for (int w = 0; w < SMALL_WAVES; ++w)
                    total[q] += count[w][tid * EACH + q];
                all += total[q];
            }
            s = all;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int y = __shfl_up(s, d, 64);
                if (lane >= d) s += y;
            }
            if (lane == 63) wave_sum[wave] = s;
        }
        __syncthreads();
        if (tid < MAX_BINS / EACH) {
            int at = s - all;
            for (int w = 0; w < wave; ++w) at += wave_sum[w];
#pragma unroll
            for (int q = 0; q < EACH; ++q)
                for (int w = 0; w < SMALL_WAVES; ++w) {
                    const int c = count[w][tid * EACH + q];
                    count[w][tid * EACH + q] = at;
                    at += c;
                }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SMALL_ROUNDS; ++r) {
            if (first + r * 64 < n) {
                const int to = count[wave][(key[r] >> shift) & (bins - 1)] + rank[r];
                key_at[to] = key[r];
                from_at[to] = from[r];
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SMALL_ROUNDS; ++r) {
            const int i = first + r * 64;
            if (i < n) {
                key[r] = key_at[i];
                from[r] = from_at[i];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < SMALL_ROUNDS; ++r) {
        const int i = first + r * 64;
        if (i < n) {
            keys[i] = key[r];
            order[i] = from[r];
            if (rows)
                rows[i] = max(bag_of(bounds, kind, fixed, bags, from[r], 0, bags), 0);
        }
    }
}

// starts[v]: how many sorted keys are below v.
__global__ __launch_bounds__(256)
void token_starts_kernel(const int* __restrict__ keys, int n, int V,
                         int* __restrict__ starts) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v > V) return;
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (keys[mid] < v) lo = mid + 1; else hi = mid;
    }
    starts[v] = lo;
}

int digit_passes(int V, int& bits) {
    int all = 1;
    while (all < 31 && (1 << all) <= V) ++all;   // keys go up to V
    const int passes = (all + MAX_BITS - 1) / MAX_BITS;
    bits = (all + passes - 1) / passes;
    return passes;
}

}  // namespace

// How many ints of workspace ks_token_sort needs.
KS_EXPORT long long ks_token_sort_work(int n, int V) {
    if (n <= SMALL) return 0;
    int bits;
    digit_passes(V, bits);
    const long long tiles = ks_ceil_div(n, TILE);
    return 5ll * n + (tiles + 1) * (1 << bits);
}

// Sorts n tokens: keys [n], order [n], rows [n] (null without bags: order
// serves as rows), starts [V + 1].
KS_EXPORT int ks_token_sort(const void* ids, int ids_wide, int n, int V,
                            int kind, const void* bounds, int fixed, int bags,
                            int* keys, int* order, int* rows, int* starts,
                            int* work, hipStream_t stream) {
    int bits;
    const int passes = digit_passes(V, bits);
    if (n > 0 && n <= SMALL) {
        // four waves have less to count and scan than sixteen: 777 tokens
        // take 12.2 us against 14.1 us, starts included
        auto* kernel = n <= SMALL / 4 ? small_sort_kernel<4> : small_sort_kernel<16>;
        kernel<<<1, n <= SMALL / 4 ? 256 : 1024, 0, stream>>>(
            ids, ids_wide, n, V, bounds, kind, fixed, bags, bits, passes, keys,
            order, rows);
    } else if (n > 0) {
        const int tiles = ks_ceil_div(n, TILE);
        int2* pairs[2] = {(int2*)work, (int2*)(work + 2ll * n)};
        int* totals = work + 4ll * n;
        int* counts = totals + (1 << bits);
        int* bag = rows ? counts + (long long)tiles * (1 << bits) : nullptr;
        if (bag)
            position_bags_kernel<<<tiles, 256, 0, stream>>>(
                bounds, kind, fixed, bags, n, bag);
        Source src{nullptr, ids, ids_wide, n, V, bag};
        for (int p = 0; p < passes; ++p) {
            int2* to = p == passes - 1 ? nullptr : pairs[p & 1];
            digit_count_kernel<<<tiles, 256, 0, stream>>>(src, p * bits, bits,
                                                          counts, tiles);
            digit_scan_kernel<<<1 << bits, 256, 0, stream>>>(counts, tiles, totals);
            digit_move_kernel<<<tiles, 256, 0, stream>>>(
                src, p * bits, bits, counts, tiles, totals, to, keys, order, rows);
            src.pairs = to;
        }
    }
    token_starts_kernel<<<V / 256 + 1, 256, 0, stream>>>(keys, n, V, starts);
    return (int)hipGetLastError();
}
