// A stable sort of token positions by token id, for the embedding gradient:
// sums over a token's occurrences then run over one stretch, in ascending
// order of their positions.
//
// Radix sort from the lowest digit, at most nine bits a digit.  A digit's
// pass counts the digits of every tile of tokens, scans the counts over the
// tiles, and moves each token to its digit's place.  Inside a wave the tokens
// of one digit are found by a ballot over each of its bits, so that equal
// digits keep their order without atomics.  A tile is put in order in LDS
// first, so that what it writes of one digit is one run.  Up to 8192 tokens
// each one's place is counted instead, in one launch.
//
// Bound by latency and launches, tokens of 100000: 777 take 4.7 us, 4096 take
// 8.2 us, 16384 take 22 us in five launches, 1048576 take 52 us (78 us with
// scattered writes of 4 bytes), 8388608 take 181 us.  Ids in bags take longer,
// 7.86 M of them 329 us: the last pass reads a bag's number for each token, and a
// cache line for it.
#include "common.h"

#include <cstdint>

namespace {

constexpr int WAVES = 4;
// A tile's tokens are so many for each of its block's threads.  Few of them
// fill the card with few tokens: 65536 take 30 us with two a thread, 50 us
// with eight, 262144 take 32 and 39 us, 524288 take 42 and 41 us.
constexpr int FEW = 2, MANY = 8;
constexpr int ROUNDS_LIMIT = 524288;

// Up to so many tiles each sums all tiles' counts itself, without the scan's
// launch: 12000 tokens in bags take 24.2 us, 26.5 us with it, and a launch less on
// the host; 32768 take 25.1 and 23.6 us, but 39 and 40 us with the host's part and
// the gradient's; 65536, of 128 tiles, 36.7 and 29.5 us.
constexpr int UNSCANNED = 64;

int rounds_of(int n) { return n <= ROUNDS_LIMIT ? FEW : MANY; }

constexpr int MAX_BITS = 9, MAX_BINS = 1 << MAX_BITS;

// Bounds of bags, and which positions are in some bag.
struct Bags {
    const void* bounds;
    int kind, fixed, count;  // kind 0: fixed length, 1: int32, 2: int64 bounds
    __device__ __forceinline__ long long at(int k) const {
        return kind == 1 ? (long long)((const int*)bounds)[k]
                         : ((const long long*)bounds)[k];
    }
    __device__ __forceinline__ void inside(int n, long long& from,
                                           long long& to) const {
        from = kind ? (count ? at(0) : n) : 0;
        to = kind && count ? at(count) : n;
    }
};

// What a pass reads: the token ids themselves, or (key, position) pairs.  A
// key is the id, or V for one outside the table or outside every bag.
struct Source {
    const int2* pairs;
    const void* ids;
    int wide, n, V;
    int* bag;          // the positions' bags, where there are bags
};

__device__ __forceinline__ int2 pair_at(const Source& s, int i) {
    if (s.pairs) return s.pairs[i];
    const long long v = s.wide ? ((const long long*)s.ids)[i]
                               : (long long)((const int*)s.ids)[i];
    int key = (v >= 0 && v < s.V) ? (int)v : s.V;
    if (s.bag && s.bag[i] < 0) key = s.V;
    return make_int2(key, i);
}

// Inclusive maxima over the block's 256 threads.
__device__ __forceinline__ int max_block(int x, int* wave_max) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d, 64);
        if (lane >= d) x = max(x, y);
    }
    if (lane == 63) wave_max[wave] = x;
    __syncthreads();
    for (int w = 0; w < wave; ++w) x = max(x, wave_max[w]);
    return x;
}

// The bags of a tile's positions, -1 outside: every bag that begins in the tile
// marks its first position, and a position's bag is the last mark so far.
// 524288 tokens in bags of ten were sorted in 59 us with them, in 69 us where
// each position searched the bounds; now 53 us.
template <int ROUNDS>
__device__ __forceinline__ void bags_of_tile(const Bags& bags, int n,
                                             long long first,
                                             int* __restrict__ bag) {
    constexpr int TILE = ROUNDS * 256;
    __shared__ int mark[TILE], ends[2], wave_max[4];
    const int tid = threadIdx.x;
    if (bags.kind == 0) {
        for (int r = 0; r < ROUNDS; ++r) {
            const long long i = first + r * 256 + tid;
            if (i < n) bag[i] = (int)i / bags.fixed;
        }
        return;
    }
    for (int r = 0; r < ROUNDS; ++r) mark[r * 256 + tid] = 0;
    // the last bags that begin at or before the tile's ends
    if (bags.count && (tid & 63) == 0 && tid < 128) {
        const long long i = tid ? first + TILE - 1 : first;
        int lo = 0, hi = bags.count;
        while (hi - lo > 1) {
            const int mid = lo + (hi - lo) / 2;
            if (bags.at(mid) <= i) lo = mid; else hi = mid;
        }
        ends[tid >> 6] = lo;
    }
    __syncthreads();
    if (bags.count)
        for (int b = ends[0] + tid; b <= ends[1]; b += 256) {
            const long long i = max(bags.at(b), first) - first;
            if (i < TILE) atomicMax(&mark[i], b);
        }
    __syncthreads();
    int last[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        last[r] = mark[tid * ROUNDS + r];
        if (r) last[r] = max(last[r], last[r - 1]);
    }
    const int here = max_block(last[ROUNDS - 1], wave_max);
    int before = __shfl_up(here, 1, 64);
    if ((tid & 63) == 0) {
        before = 0;
        for (int w = 0; w < tid >> 6; ++w) before = max(before, wave_max[w]);
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        mark[tid * ROUNDS + r] = max(before, last[r]);
    __syncthreads();
    long long from, to;
    bags.inside(n, from, to);
    for (int r = 0; r < ROUNDS; ++r) {
        const long long i = first + r * 256 + tid;
        if (i < n) bag[i] = i >= from && i < to ? mark[r * 256 + tid] : -1;
    }
}

// The first pass finds the positions' bags too.
template <int ROUNDS>
__global__ __launch_bounds__(256)
void digit_count_kernel(Source src, int shift, int bits,
                        int* __restrict__ counts, Bags bags) {
    __shared__ int bin[MAX_BINS];
    const int bins = 1 << bits;
    const long long first = (long long)blockIdx.x * (ROUNDS * 256);
    for (int i = threadIdx.x; i < bins; i += 256) bin[i] = 0;
    // a thread reads the bags that it has written itself
    if (src.bag && !src.pairs) bags_of_tile<ROUNDS>(bags, src.n, first, src.bag);
    __syncthreads();
    int digit[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        // past the end the last token is read again, and not counted
        const long long i = first + r * 256 + threadIdx.x;
        const int2 p = pair_at(src, (int)min(i, (long long)src.n - 1));
        digit[r] = (p.x >> shift) & (bins - 1);
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (first + r * 256 + threadIdx.x < src.n) atomicAdd(&bin[digit[r]], 1);
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += 256)
        counts[(long long)blockIdx.x * bins + i] = bin[i];
}

// Exclusive sums over the tiles, in place, and each digit's total.  counts are
// [tile][digit], so that a tile writes and reads its own in whole lines (8388608
// tokens take 175 us, 200 us with [digit][tile]); a block has 16 digits, and 64
// groups of lanes a stretch of the tiles each.
__global__ __launch_bounds__(1024)
void digit_scan_kernel(int* __restrict__ counts, int tiles, int bins,
                       int* __restrict__ totals) {
    __shared__ int part[64][17];
    const int digit = blockIdx.x * 16 + (threadIdx.x & 15), group = threadIdx.x >> 4;
    const int each = (tiles + 63) / 64;
    const int t0 = min(tiles, group * each), t1 = min(tiles, t0 + each);
    int* const at = counts + digit;
    int sum = 0;
    if (digit < bins)
#pragma unroll 4
        for (int t = t0; t < t1; ++t) sum += at[(long long)t * bins];
    part[group][threadIdx.x & 15] = sum;
    __syncthreads();
    // a wave scans one digit's 64 groups
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int x = part[lane][wave];
    int s = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(s, d, 64);
        if (lane >= d) s += y;
    }
    part[lane][wave] = s - x;
    if (lane == 63 && blockIdx.x * 16 + wave < bins)
        totals[blockIdx.x * 16 + wave] = s;
    __syncthreads();
    int before = part[group][threadIdx.x & 15];
    if (digit < bins)
#pragma unroll 4
        for (int t = t0; t < t1; ++t) {
            const int c = at[(long long)t * bins];
            at[(long long)t * bins] = before;
            before += c;
        }
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
template <int ROUNDS>
__global__ __launch_bounds__(256)
void digit_move_kernel(Source src, int shift, int bits,
                       const int* __restrict__ counts,
                       const int* __restrict__ totals,
                       int2* __restrict__ pairs_out, int* __restrict__ keys,
                       int* __restrict__ order, int* __restrict__ rows) {
    constexpr int TILE = ROUNDS * 256;
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
    int t0 = 0, t1 = 0, c0 = 0, c1 = 0;
    if (d0 < bins) {
        const int2* const at = (const int2*)(counts + d0);
        if (totals) {
            const int2 t = *(const int2*)(totals + d0);
            const int2 c = at[(long long)blockIdx.x * (bins / 2)];
            t0 = t.x, t1 = t.y, c0 = c.x, c1 = c.y;
        } else {
            // not scanned: all tiles' counts are summed here
#pragma unroll 8
            for (int k = 0; k < (int)gridDim.x; ++k) {
                const int2 c = at[k * (bins / 2)];
                t0 += c.x;
                t1 += c.y;
                c0 += k < (int)blockIdx.x ? c.x : 0;
                c1 += k < (int)blockIdx.x ? c.y : 0;
            }
        }
    }
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

// Up to SMALL tokens, in one launch: a token's place is how many tokens sort
// before it, counted against all of them in LDS by 16 lanes.  n^2 comparisons
// are less than the passes' barriers: two instructions each, over the whole
// card.  Further blocks count the tokens below each of STARTS ids.  8192
// tokens take 15 us, 20 us by digits; 16384 take 77 and 25 us.
constexpr int SMALL = 8192, PLACED = 16, STARTS = 2048;

__global__ __launch_bounds__(256)
void small_sort_kernel(const void* __restrict__ ids, int wide, int n, int V,
                       Bags bags, int* __restrict__ keys,
                       int* __restrict__ order, int* __restrict__ rows,
                       int* __restrict__ starts, int placing) {
    __shared__ __attribute__((aligned(16))) int key_at[SMALL];
    __shared__ int wave_sum[4];
    const int tid = threadIdx.x;
    long long from, to;
    bags.inside(n, from, to);
    auto key_of = [&](int i) -> int {
        const long long v = wide ? ((const long long*)ids)[i]
                                 : (long long)((const int*)ids)[i];
        return v >= 0 && v < V && i >= from && i < to ? (int)v : V;
    };

    if ((int)blockIdx.x >= placing) {
        int* const bin = key_at;
        const long long v0 = (long long)(blockIdx.x - placing) * STARTS;
        for (int i = tid; i < STARTS; i += 256) bin[i] = 0;
        __syncthreads();
        int below = 0;
#pragma unroll 4
        for (int i = tid; i < n; i += 256) {
            const long long at = key_of(i) - v0;
            if (at < 0) ++below;
            else if (at < STARTS) atomicAdd(&bin[at], 1);
        }
        __syncthreads();
        // eight ids a thread, then what lies below them
        constexpr int EACH = STARTS / 256;
        int x[EACH], all = 0;
#pragma unroll
        for (int q = 0; q < EACH; ++q) {
            x[q] = all;
            all += bin[tid * EACH + q];
        }
        const int mine = scan_block(all, wave_sum);
#pragma unroll
        for (int d = 32; d; d >>= 1) below += __shfl_xor(below, d, 64);
        if ((tid & 63) == 0) wave_sum[tid >> 6] = below;
        __syncthreads();
        below = wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
#pragma unroll
        for (int q = 0; q < EACH; ++q) bin[tid * EACH + q] = below + mine + x[q];
        __syncthreads();
        for (int i = tid; i < STARTS; i += 256)
            if (v0 + i <= V) starts[v0 + i] = bin[i];
        return;
    }

    const int part = tid & 15, i = blockIdx.x * PLACED + (tid >> 4);
    const int groups = (n + 3) / 4;
#pragma unroll 4
    for (int j = tid; j < groups * 4; j += 256)
        key_at[j] = j < n ? key_of(j) : 0x7fffffff;
    // the token's bag, the last that begins at or before it: 16 bounds a step
    int row = 0;
    if (rows) {
        if (bags.kind == 0) {
            row = min(i, n - 1) / bags.fixed;
        } else if (bags.count) {
            int lo = 0, hi = bags.count;
            while (hi - lo > 1) {
                const int step = (hi - lo + 15) / 16;
                const int k = lo + part * step;
                const unsigned long long at =
                    __ballot(k < hi && bags.at(k) <= i);
                const int c = __popcll(at >> (tid & 48) & 0xffff);
                if (c) lo += (c - 1) * step;
                hi = min(hi, lo + step);
            }
            row = lo;
        }
    }
    __syncthreads();
    if (i >= n) return;
    const int key = key_at[i], own = i >> 2;
    int place = 0;
#pragma unroll 4
    for (int g = part; g < groups; g += 16) {
        const int4 k = *(const int4*)(key_at + g * 4);
        const int most = g < own ? key + 1 : key;
        place += (k.x < most) + (k.y < most) + (k.z < most) + (k.w < most);
    }
    if (part < (i & 3)) place += key_at[own * 4 + part] == key;
#pragma unroll
    for (int d = 8; d; d >>= 1) place += __shfl_xor(place, d, 16);
    if (part == 0) {
        keys[place] = key;
        order[place] = i;
        if (rows) rows[place] = row;
    }
}

// starts[v]: how many sorted keys are below v.  Three keys a step, loaded without
// a branch so that they overlap: the plan of 131072 tokens takes 1 us less than
// with a binary search.
__global__ __launch_bounds__(256)
void token_starts_kernel(const int* __restrict__ keys, int n, int V,
                         int* __restrict__ starts) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v > V) return;
    // the number is in [lo, lo + left]
    int lo = 0, left = n;
    while (left > 0) {
        const int step = left / 4 + 1;
        int below = 0;
#pragma unroll
        for (int k = 1; k < 4; ++k) {
            const int key = keys[lo + min(k * step, left) - 1];
            below += (k * step <= left) & (key < v);
        }
        lo += below * step;
        left = min(step - 1, left - below * step);
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

template <int ROUNDS>
void sort_by_digits(Source src, const Bags& bags, int* keys, int* order,
                    int* rows, int* work, hipStream_t stream) {
    int bits;
    const int passes = digit_passes(src.V, bits);
    const int n = src.n, tiles = ks_ceil_div(n, ROUNDS * 256);
    int2* pairs[2] = {(int2*)work, (int2*)(work + 2ll * n)};
    int* totals = work + 4ll * n;
    int* counts = totals + (1 << bits);
    src.bag = rows ? counts + (long long)tiles * (1 << bits) : nullptr;
    for (int p = 0; p < passes; ++p) {
        int2* to = p == passes - 1 ? nullptr : pairs[p & 1];
        digit_count_kernel<ROUNDS><<<tiles, 256, 0, stream>>>(
            src, p * bits, bits, counts, bags);
        if (tiles > UNSCANNED)
            digit_scan_kernel<<<ks_ceil_div(1 << bits, 16), 1024, 0, stream>>>(
                counts, tiles, 1 << bits, totals);
        digit_move_kernel<ROUNDS><<<tiles, 256, 0, stream>>>(
            src, p * bits, bits, counts, tiles > UNSCANNED ? totals : nullptr, to,
            keys, order, rows);
        src.pairs = to;
    }
}

}  // namespace

// How many ints of workspace ks_token_sort needs.
KS_EXPORT long long ks_token_sort_work(int n, int V) {
    if (n <= SMALL) return 0;
    int bits;
    digit_passes(V, bits);
    const long long tiles = ks_ceil_div(n, rounds_of(n) * 256);
    return 5ll * n + (tiles + 1) * (1 << bits);
}

// Sorts n tokens: keys [n], order [n], rows [n] (null without bags: order
// serves as rows), starts [V + 1].
KS_EXPORT int ks_token_sort(const void* ids, int ids_wide, int n, int V,
                            int kind, const void* bounds, int fixed, int bags,
                            int* keys, int* order, int* rows, int* starts,
                            int* work, hipStream_t stream) {
    if (!starts || (n && (!ids || !keys || !order)) || (kind && !bounds) ||
        (!work && ks_token_sort_work(n, V)))
        return (int)hipErrorInvalidValue;
    const Bags segments{bounds, kind, fixed, bags};
    if (n > 0 && n <= SMALL) {
        const int placing = ks_ceil_div(n, PLACED);
        small_sort_kernel<<<placing + V / STARTS + 1, 256, 0, stream>>>(
            ids, ids_wide, n, V, segments, keys, order, rows, starts, placing);
        return (int)hipGetLastError();
    }
    if (n > 0) {
        auto* sort = rounds_of(n) == FEW ? sort_by_digits<FEW> : sort_by_digits<MANY>;
        sort(Source{nullptr, ids, ids_wide, n, V, nullptr}, segments, keys,
             order, rows, work, stream);
    }
    token_starts_kernel<<<V / 256 + 1, 256, 0, stream>>>(keys, n, V, starts);
    return (int)hipGetLastError();
}
