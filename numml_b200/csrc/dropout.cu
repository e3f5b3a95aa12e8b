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

// Which of a block's eight elements are kept.  `high` holds the threshold's high half in its upper 16 bits (zeros
// below): a word's upper half is above it where the word is above high | 0xFFFF, its lower half where the word
// shifted up is above high, so no half is taken out.  A half that equals the threshold's makes a zero half in
// word ^ pattern; one test finds it in all four words.
struct Threshold {
    uint32_t high, pattern, low;
};
__device__ __forceinline__ void keep_flags(uint64_t block, uint64_t offset, uint64_t seed, const Threshold& t, bool (&keep)[8]) {
    const Words a = philox(block, offset, 0, seed);
    uint32_t zero = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        keep[2 * q] = (a.w[q] << 16) > t.high;
        keep[2 * q + 1] = a.w[q] > (t.high | 0xFFFFu);
        const uint32_t z = a.w[q] ^ t.pattern;
        zero |= (z - 0x00010001u) & ~z;
    }
    if (zero & 0x80008000u) {                        // at most a few in 65536: a carry may report a half that is none
        const Words b = philox(block, offset, 1, seed);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const uint32_t h = (q & 1) ? a.w[q / 2] >> 16 : a.w[q / 2] & 0xFFFFu, l = (q & 1) ? b.w[q / 2] >> 16 : b.w[q / 2] & 0xFFFFu;
            if (h == t.high >> 16) keep[q] = l >= t.low;
        }
    }
}

template <typename T>
constexpr int batch() { return sizeof(T) == 8 ? 1 : sizeof(T) == 4 ? 2 : 4; }

template <typename T>
__device__ __forceinline__ void load8(const T* p, acc_t<T> (&v)[8]) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int q = 0; q < 8; q += V) load_acc<T, V>(p + q, *reinterpret_cast<acc_t<T>(*)[V]>(v + q));
}

// A thread has kBatch blocks of eight consecutive elements, all of whose loads are under way before the first is used;
// `state` (device int64[2]: seed, offset) overrides the arguments when given, so that a captured graph can be
// replayed with new numbers.
template <typename T, bool RESIDUAL>
__global__ void __launch_bounds__(256) dropout_kernel(int64_t n, const T* __restrict__ x, const T* __restrict__ residual,
                                                      T* __restrict__ y, Threshold threshold, acc_t<T> scale, uint64_t seed,
                                                      uint64_t offset, const int64_t* __restrict__ state) {
    using A = acc_t<T>;
    constexpr int V = 16 / sizeof(T), kBatch = batch<T>();
    if (state) {
        seed = static_cast<uint64_t>(state[0]);
        offset = static_cast<uint64_t>(state[1]);
    }
    const int64_t whole = n / 8;
    constexpr int64_t stride = 256;
    int64_t b = blockIdx.x * (kBatch * stride) + threadIdx.x;
    const int64_t limit = min(whole, (blockIdx.x + int64_t(1)) * (kBatch * stride));
    auto finish = [&](int64_t block, A (&xv)[8], const A (&rv)[8]) {
        bool keep[8];
        keep_flags(block, offset, seed, threshold, keep);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            xv[q] = keep[q] ? xv[q] * scale : A(0);
            if (RESIDUAL) xv[q] += rv[q];
        }
#pragma unroll
        for (int q = 0; q < 8; q += V) store_acc<T, V>(y + block * 8 + q, *reinterpret_cast<A(*)[V]>(xv + q));
    };
    if (b + (kBatch - 1) * stride < whole) {
        Pack<T, V> xr[kBatch][8 / V], rr[kBatch][8 / V];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int q = 0; q < 8 / V; ++q) {
                xr[u][q] = *reinterpret_cast<const Pack<T, V>*>(x + (b + u * stride) * 8 + q * V);
                if (RESIDUAL) rr[u][q] = *reinterpret_cast<const Pack<T, V>*>(residual + (b + u * stride) * 8 + q * V);
            }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            A xv[8], rv[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                xv[q] = to_acc(xr[u][q / V].v[q % V]);
                rv[q] = RESIDUAL ? to_acc(rr[u][q / V].v[q % V]) : A(0);
            }
            finish(b + u * stride, xv, rv);
        }
        return;
    }
    for (; b < limit; b += stride) {
        A xv[8], rv[8] = {};
        load8(x + b * 8, xv);
        if (RESIDUAL) load8(residual + b * 8, rv);
        finish(b, xv, rv);
    }
    if (b == whole && n % 8 != 0 && b < (blockIdx.x + int64_t(1)) * (kBatch * stride)) {          // the last, partial block
        bool keep[8];
        keep_flags(whole, offset, seed, threshold, keep);
#pragma unroll
        for (int q = 0; q < 7; ++q) {
            const int64_t i = whole * 8 + q;
            if (i >= n) break;
            A v = keep[q] ? to_acc(x[i]) * scale : A(0);
            if (RESIDUAL) v += to_acc(residual[i]);
            y[i] = from_acc<T>(v);
        }
    }
}

template <typename T>
int launch_dropout(int64_t n, const void* x, const void* residual, void* y, double p, uint64_t seed, uint64_t offset,
                   const int64_t* state, cudaStream_t stream) {
    const uint64_t bar = static_cast<uint64_t>(std::nearbyint(p * 4294967296.0));
    // 2^32 (p = 1) keeps nothing: no half is above 0xFFFF and no lower half reaches 0x10000
    const uint32_t half = bar >> 32 ? 0xFFFFu : static_cast<uint32_t>(bar >> 16);
    const Threshold threshold{half << 16, half << 16 | half, bar >> 32 ? 0x10000u : static_cast<uint32_t>(bar & 0xFFFFu)};
    const acc_t<T> scale = p < 1.0 ? static_cast<acc_t<T>>(1.0 / (1.0 - p)) : acc_t<T>(0);
    constexpr int kBatch = batch<T>();
    const int64_t blocks = ceil_div(ceil_div(n, 8), 256 * kBatch);
    if (blocks > INT32_MAX) return NB200_ERR_TOO_LARGE;
    const unsigned grid = static_cast<unsigned>(blocks);
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
