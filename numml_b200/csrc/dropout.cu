// Dropout from a counter-based generator:  y[i] = (u[i] >= T ? x[i] / (1 - p) : 0) + residual[i].
//
// u[i] is a 32-bit number that depends on (seed, offset, i) alone, so the mask is recomputed wherever
// it is needed and never stored: the backward pass is the same kernel applied to the gradient, and the
// bytes of a pass are its input and its output.
//
// Generator: Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011), key = seed, counter = (i / 8 as 64 bits, offset as 63 bits, one stream bit).
// Of u[i] the high 16 bits are half-word i % 8 of the four output words of stream 0 and the low 16 bits
// the same half-word of stream 1.  Which side of T a number falls on is settled by its high half unless
// that equals T's high half, which happens once in 65536 elements; only then is stream 1 evaluated.  So
// one generator call serves eight elements (with a word per element the ten rounds would cost as much
// issue time as the bytes of a 16-bit type take to arrive) while p keeps a resolution of 2^-32.
#include <cmath>

#include "dense_common.cuh"

namespace nb200 {
namespace {

struct Words { uint32_t w[4]; };

__device__ __forceinline__ Words philox(uint64_t block, uint64_t offset, uint32_t stream_bit, uint64_t seed) {
    uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32);
    uint32_t c2 = static_cast<uint32_t>(offset), c3 = (static_cast<uint32_t>(offset >> 32) & 0x7FFFFFFFu) | (stream_bit << 31);
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u, p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
        c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
        c1 = static_cast<uint32_t>(p1);
        c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
        c3 = static_cast<uint32_t>(p0);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

// Bit q set: element q of the block of eight is kept.
__device__ __forceinline__ uint32_t keep_bits(uint64_t block, uint64_t offset, uint64_t seed, uint32_t t_high, uint32_t t_low) {
    const Words a = philox(block, offset, 0, seed);
    uint32_t keep = 0, tie = 0;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const uint32_t h = (q & 1) ? a.w[q / 2] >> 16 : a.w[q / 2] & 0xFFFFu;
        keep |= (h > t_high ? 1u : 0u) << q;
        tie |= (h == t_high ? 1u : 0u) << q;
    }
    if (tie) {
        const Words b = philox(block, offset, 1, seed);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const uint32_t l = (q & 1) ? b.w[q / 2] >> 16 : b.w[q / 2] & 0xFFFFu;
            if ((tie >> q & 1u) && l >= t_low) keep |= 1u << q;
        }
    }
    return keep;
}

// A thread owns blocks of eight consecutive elements; `state` (device int64[2]: seed, offset) overrides
// the arguments when given, so that a captured graph can be replayed with new numbers.
template <typename T, bool RESIDUAL>
__global__ void __launch_bounds__(256) dropout_kernel(int64_t n, const T* __restrict__ x, const T* __restrict__ residual,
                                                      T* __restrict__ y, uint64_t threshold, acc_t<T> scale, uint64_t seed,
                                                      uint64_t offset, const int64_t* __restrict__ state) {
    using A = acc_t<T>;
    constexpr int V = 16 / sizeof(T) < 8 ? 16 / sizeof(T) : 8;
    if (state) {
        seed = static_cast<uint64_t>(state[0]);
        offset = static_cast<uint64_t>(state[1]);
    }
    // T = 2^32 (p = 1) keeps nothing: no half-word exceeds 0x10000
    const uint32_t t_high = static_cast<uint32_t>(threshold >> 16), t_low = static_cast<uint32_t>(threshold & 0xFFFFu);
    const int64_t blocks = (n + 7) / 8;
    for (int64_t b = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; b < blocks; b += int64_t(gridDim.x) * blockDim.x) {
        const int64_t base = b * 8;
        if (base + 8 <= n) {
            A xv[8], rv[8];
#pragma unroll
            for (int q = 0; q < 8; q += V) {
                load_acc<T, V>(x + base + q, *reinterpret_cast<A(*)[V]>(xv + q));
                if (RESIDUAL) load_acc<T, V>(residual + base + q, *reinterpret_cast<A(*)[V]>(rv + q));
            }
            const uint32_t keep = keep_bits(b, offset, seed, t_high, t_low);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                xv[q] = (keep >> q & 1u) ? xv[q] * scale : A(0);
                if (RESIDUAL) xv[q] += rv[q];
            }
#pragma unroll
            for (int q = 0; q < 8; q += V) store_acc<T, V>(y + base + q, *reinterpret_cast<A(*)[V]>(xv + q));
        } else {
            const uint32_t keep = keep_bits(b, offset, seed, t_high, t_low);
            for (int64_t i = base; i < n; ++i) {
                A v = (keep >> (i - base) & 1u) ? to_acc(x[i]) * scale : A(0);
                if (RESIDUAL) v += to_acc(residual[i]);
                y[i] = from_acc<T>(v);
            }
        }
    }
}

template <typename T>
int launch_dropout(int64_t n, const void* x, const void* residual, void* y, double p, uint64_t seed, uint64_t offset,
                   const int64_t* state, cudaStream_t stream) {
    const uint64_t threshold = static_cast<uint64_t>(std::nearbyint(p * 4294967296.0));
    const acc_t<T> scale = p < 1.0 ? static_cast<acc_t<T>>(1.0 / (1.0 - p)) : acc_t<T>(0);
    const int64_t blocks = ceil_div(n, 8);
    const int grid = static_cast<int>(ceil_div(blocks, 256) < kSMs * 8 ? ceil_div(blocks, 256) : kSMs * 8);
    const T* xt = static_cast<const T*>(x);
    if (residual)
        dropout_kernel<T, true><<<grid, 256, 0, stream>>>(n, xt, static_cast<const T*>(residual), static_cast<T*>(y), threshold,
                                                          scale, seed, offset, state);
    else
        dropout_kernel<T, false><<<grid, 256, 0, stream>>>(n, xt, nullptr, static_cast<T*>(y), threshold, scale, seed, offset, state);
    return launch_status();
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" int nb200_dropout(int64_t n, const void* x, const void* residual, void* y, double p, uint64_t seed, uint64_t offset,
                             const int64_t* state, int dtype, nb200_stream stream) {
    if (n < 0 || !(p >= 0.0 && p <= 1.0) || !known_dense_dtype(dtype)) return NB200_ERR_BAD_ARG;
    if (n == 0) return NB200_OK;
    if (!x || !y) return NB200_ERR_BAD_ARG;
    if (!aligned16(x) || !aligned16(y) || (residual && !aligned16(residual))) return NB200_ERR_ALIGN;
    return NB200_DISPATCH_DENSE(dtype, launch_dropout<T>(n, x, residual, y, p, seed, offset, state, as_stream(stream)));
}
