// A stable sort of token positions by token id, for the embedding gradient:
// sums over a token's occurrences then run over one stretch, in ascending
// order of their positions.
//
// Radix sort from the lowest digit, at most nine bits a digit.  A digit's
// pass counts the digits of every tile of 4096 tokens, scans the counts over
// the tiles, and moves each token to its digit's place.  Inside a wave the
// tokens of one digit are found by a ballot over each of its bits, so that
// equal digits keep their order without atomics.
#include "common.h"

#include <cstdint>

namespace {

constexpr int TILE = 4096, WAVES = 4, ROUNDS = TILE / (WAVES * 64);
constexpr int MAX_BITS = 9, MAX_BINS = 1 << MAX_BITS;

// The bag of position i: -1 where the bounds leave it out.
__device__ __forceinline__ int bag_of(const void* bounds, int kind, int fixed,
                                      int bags, int n, int i) {
    if (kind == 0) return i / fixed;
    if (bags == 0) return -1;
    auto at = [&](int k) -> long long {
        return kind == 1 ? (long long)((const int*)bounds)[k]
                         : ((const long long*)bounds)[k];
    };
    int lo = 0, hi = bags;
    while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        if (at(mid) <= i) lo = mid; else hi = mid;
    }
    return (at(lo) <= i && i < at(lo + 1)) ? lo : -1;
}

// Sort keys (V for a token outside the table or outside every bag), and the
// bags of the positions where there are bags.
__global__ __launch_bounds__(256)
void token_keys_kernel(const void* __restrict__ ids, int wide, int n, int V,
                       const void* __restrict__ bounds, int kind, int fixed,
                       int bags, int* __restrict__ keys,
                       int* __restrict__ bag) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long long v = wide ? ((const long long*)ids)[i]
                             : (long long)((const int*)ids)[i];
    int key = (v >= 0 && v < V) ? (int)v : V;
    if (bag) {
        const int b = bag_of(bounds, kind, fixed, bags, n, i);
        bag[i] = b;
        if (b < 0) key = V;
    }
    keys[i] = key;
}

__global__ __launch_bounds__(256)
void digit_count_kernel(const int* __restrict__ keys, int n, int shift,
                        int bits, int* __restrict__ counts, int tiles) {
    __shared__ int bin[MAX_BINS];
    const int bins = 1 << bits;
    for (int i = threadIdx.x; i < bins; i += 256) bin[i] = 0;
    __syncthreads();
    const int first = blockIdx.x * TILE;
    for (int r = 0; r < TILE / 256; ++r) {
        const int i = first + r * 256 + threadIdx.x;
        if (i < n) atomicAdd(&bin[(keys[i] >> shift) & (bins - 1)], 1);
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

__global__ __launch_bounds__(256)
void digit_move_kernel(const int* __restrict__ keys_in,
                       const int* __restrict__ order_in, int n, int shift,
                       int bits, const int* __restrict__ counts, int tiles,
                       const int* __restrict__ totals,
                       int* __restrict__ keys_out, int* __restrict__ order_out,
                       const int* __restrict__ bag, int* __restrict__ rows) {
    __shared__ int count[WAVES][MAX_BINS];
    __shared__ int base[MAX_BINS];
    __shared__ int wave_sum[WAVES];
    const int bins = 1 << bits;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < bins; i += 256)
        for (int w = 0; w < WAVES; ++w) count[w][i] = 0;
    // where each digit begins: totals summed, two digits a thread
    const int d0 = threadIdx.x * 2;
    const int t0 = d0 < bins ? totals[d0] : 0;
    const int t1 = d0 + 1 < bins ? totals[d0 + 1] : 0;
    int s = t0 + t1;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(s, d, 64);
        if (lane >= d) s += y;
    }
    if (lane == 63) wave_sum[wave] = s;
    __syncthreads();
    s -= t0 + t1;
    for (int w = 0; w < wave; ++w) s += wave_sum[w];
    if (d0 < bins) base[d0] = s + counts[(long long)d0 * tiles + blockIdx.x];
    if (d0 + 1 < bins)
        base[d0 + 1] = s + t0 +
                       counts[(long long)(d0 + 1) * tiles + blockIdx.x];
    __syncthreads();

    const int first = blockIdx.x * TILE + wave * (ROUNDS * 64) + lane;
    int key[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int i = first + r * 64;
        key[r] = i < n ? keys_in[i] : 0;
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        rank[r] = rank_digit((key[r] >> shift) & (bins - 1), bits,
                             first + r * 64 < n, count[wave]);
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += 256) {
        int at = base[i];
        for (int w = 0; w < WAVES; ++w) {
            const int c = count[w][i];
            count[w][i] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int i = first + r * 64;
        if (i < n) {
            const int to = count[wave][(key[r] >> shift) & (bins - 1)] + rank[r];
            const int from = order_in ? order_in[i] : i;
            keys_out[to] = key[r];
            order_out[to] = from;
            // a token outside every bag sorts last and is never read
            if (rows) rows[to] = max(bag[from], 0);
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
    int bits;
    digit_passes(V, bits);
    const long long tiles = ks_ceil_div(n, TILE);
    return 3ll * n + (tiles + 1) * (1 << bits);
}

// Sorts n tokens: keys [n], order [n], rows [n] (null without bags: order
// serves as rows), starts [V + 1].
KS_EXPORT int ks_token_sort(const void* ids, int ids_wide, int n, int V,
                            int kind, const void* bounds, int fixed, int bags,
                            int* keys, int* order, int* rows, int* starts,
                            int* work, hipStream_t stream) {
    if (n > 0) {
        int bits;
        const int passes = digit_passes(V, bits);
        const int tiles = ks_ceil_div(n, TILE);
        int* bag = rows ? work : nullptr;
        int* other_keys = work + n;
        int* other_order = work + 2ll * n;
        int* totals = work + 3ll * n;
        int* counts = totals + (1 << bits);
        // passes alternate between the two buffers and end in the caller's
        int* to_keys = passes % 2 ? keys : other_keys;
        int* to_order = passes % 2 ? order : other_order;
        int* from_keys = passes % 2 ? other_keys : keys;
        const int* from_order = nullptr;
        token_keys_kernel<<<ks_ceil_div(n, 256), 256, 0, stream>>>(
            ids, ids_wide, n, V, bounds, kind, fixed, bags, from_keys, bag);
        for (int p = 0; p < passes; ++p) {
            const bool last = p == passes - 1;
            digit_count_kernel<<<tiles, 256, 0, stream>>>(
                from_keys, n, p * bits, bits, counts, tiles);
            digit_scan_kernel<<<1 << bits, 256, 0, stream>>>(counts, tiles, totals);
            digit_move_kernel<<<tiles, 256, 0, stream>>>(
                from_keys, from_order, n, p * bits, bits, counts, tiles, totals,
                to_keys, to_order, bag, last ? rows : nullptr);
            from_keys = to_keys;
            from_order = to_order;
            to_keys = to_keys == keys ? other_keys : keys;
            to_order = to_order == order ? other_order : order;
        }
    }
    token_starts_kernel<<<V / 256 + 1, 256, 0, stream>>>(keys, n, V, starts);
    return (int)hipGetLastError();
}
