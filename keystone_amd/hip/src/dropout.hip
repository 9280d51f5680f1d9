// Dropout from a counter: whether element i of a call is kept is a function
// of (seed, step, i) alone, so no mask is stored and the gradient's pass is
// the forward pass on the gradient.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", 2011) with key = seed and counter = (i div 8, step): its
// four 32-bit words are eight 16-bit numbers, one for each of eight
// neighbours.  An element is kept where its number is at least
// t = round(65536 p), so that the chance is exact to 2^-16, and a kept one is
// scaled by 65536 / (65536 - t), the inverse of the chance that is meant by
// t: the mean stays exact.  One rounding, to the output's type.
//
// Bound by HBM: 2^28 bf16 take 180 us, 6 TB/s read and written (twenty 32 x 32
// products for eight elements stay under that).
#include "common.h"

#include <cstdint>

namespace {

__device__ __forceinline__ void philox(uint32_t (&c)[4], uint32_t k0,
                                       uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c[0] * 0xD2511F53u;
        const uint64_t b = (uint64_t)c[2] * 0xCD9E8D57u;
        c[0] = (uint32_t)(b >> 32) ^ c[1] ^ k0;
        c[1] = (uint32_t)b;
        c[2] = (uint32_t)(a >> 32) ^ c[3] ^ k1;
        c[3] = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

template <typename T>
__global__ __launch_bounds__(256)
void dropout_kernel(const T* x, T* y, long long n,   // y may be x
                    uint32_t threshold, float scale, uint64_t seed,
                    uint64_t step, const long long* __restrict__ step_at,
                    long long first) {
    // at any element: views need not begin on 16 bytes
    typedef T V8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    if (step_at) step = (uint64_t)*step_at;
    const long long blocks = (n + 7) / 8;
    const long long b = first + (long long)blockIdx.x * 256 + threadIdx.x;
    if (b < blocks) {
        uint32_t c[4] = {(uint32_t)b, (uint32_t)((uint64_t)b >> 32),
                         (uint32_t)step, (uint32_t)(step >> 32)};
        philox(c, (uint32_t)seed, (uint32_t)(seed >> 32));
        const long long i = b * 8;
        if (i + 8 <= n) {
            V8 v = *reinterpret_cast<const V8*>(x + i);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t r = k & 1 ? c[k >> 1] >> 16 : c[k >> 1] & 0xffffu;
                v[k] = r >= threshold ? (T)((float)v[k] * scale) : (T)0.0f;
            }
            *reinterpret_cast<V8*>(y + i) = v;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t r = k & 1 ? c[k >> 1] >> 16 : c[k >> 1] & 0xffffu;
                if (i + k < n)
                    y[i + k] = r >= threshold ? (T)((float)x[i + k] * scale)
                                              : (T)0.0f;
            }
        }
    }
}

template <typename T>
int dropout(const void* x, void* y, long long n, uint32_t threshold,
            float scale, uint64_t seed, uint64_t step, const long long* step_at,
            hipStream_t stream) {
    // one block of eight elements a thread: 180 us for 2^28 bf16, against 220
    // where a grid of 16 blocks a compute unit walks on
    const long long blocks = ((n + 7) / 8 + 255) / 256;
    const long long most = 1 << 23;   // 2^31 threads a launch
    for (long long at = 0; at < blocks; at += most)
        dropout_kernel<T><<<(unsigned)(blocks - at < most ? blocks - at : most),
                            256, 0, stream>>>(
            (const T*)x, (T*)y, n, threshold, scale, seed, step, step_at,
            at * 256);
    return (int)hipGetLastError();
}

}  // namespace

// y = dropout(x) over n elements; type 0: float32, 1: bfloat16, 2: float16.
// step_at: the step in device memory; null: `step`.
KS_EXPORT int ks_dropout(const void* x, void* y, long long n, int type,
                         unsigned threshold, float scale,
                         unsigned long long seed, unsigned long long step,
                         const long long* step_at, hipStream_t stream) {
    if (n == 0) return 0;
    if (!x || !y) return (int)hipErrorInvalidValue;
    switch (type) {
        case 0: return dropout<float>(x, y, n, threshold, scale, seed, step, step_at, stream);
        case 1: return dropout<__bf16>(x, y, n, threshold, scale, seed, step, step_at, stream);
        default: return dropout<_Float16>(x, y, n, threshold, scale, seed, step, step_at, stream);
    }
}
