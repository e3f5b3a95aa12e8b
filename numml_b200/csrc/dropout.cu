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
//
// Measured (a pass; copy 6548 GB/s): 14.6 M doubles 37 us = 6.3 TB/s (0.96); 67 M bfloat16 with a residual 69 us = 5.8 TB/s
// (0.89), without 64 us = 4.2 TB/s: for two bytes each way the generator's instructions are the bound (61 % of the issue
// slots, the rest waits for the multiplier).
#include <cmath>
#include <type_traits>

#include "dense_common.cuh"

namespace nb200 {
namespace {

struct Words { uint32_t w[4]; };

// The key of each round.  Formed on the host, they are operands from constant memory.
struct Keys {
    uint32_t k[10][2];
    __host__ __device__ __forceinline__ explicit Keys(uint64_t seed) {
        uint32_t a = static_cast<uint32_t>(seed), b = static_cast<uint32_t>(seed >> 32);
#pragma unroll
        for (int r = 0; r < 10; ++r, a += 0x9E3779B9u, b += 0xBB67AE85u) {
            k[r][0] = a;
            k[r][1] = b;
        }
    }
};

__device__ __forceinline__ Words philox(uint64_t block, uint64_t offset, uint32_t stream_bit, const Keys& keys) {
    uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32);
    uint32_t c2 = static_cast<uint32_t>(offset), c3 = (static_cast<uint32_t>(offset >> 32) & 0x7FFFFFFFu) | (stream_bit << 31);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u, p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
        c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ keys.k[r][0];
        c1 = static_cast<uint32_t>(p1);
        c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ keys.k[r][1];
        c3 = static_cast<uint32_t>(p0);
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
__device__ __forceinline__ void keep_flags(uint64_t block, uint64_t offset, const Keys& keys, const Threshold& t, bool (&keep)[8]) {
    const Words a = philox(block, offset, 0, keys);
    uint32_t zero = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        keep[2 * q] = (a.w[q] << 16) > t.high;
        keep[2 * q + 1] = a.w[q] > (t.high | 0xFFFFu);
        const uint32_t z = a.w[q] ^ t.pattern;
        zero |= (z - 0x00010001u) & ~z;
    }
    if (zero & 0x80008000u) {                        // at most a few in 65536: a carry may report a half that is none
        const Words b = philox(block, offset, 1, keys);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const uint32_t h = (q & 1) ? a.w[q / 2] >> 16 : a.w[q / 2] & 0xFFFFu, l = (q & 1) ? b.w[q / 2] >> 16 : b.w[q / 2] & 0xFFFFu;
            if (h == t.high >> 16) keep[q] = l >= t.low;
        }
    }
}

// Eight values as they lie in memory, and in arithmetic.
template <typename T> struct Eight {                                  // 16-bit types: four words of two
    uint32_t w[4];
    __device__ __forceinline__ void load(const T* p) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    }
    __device__ __forceinline__ float get(int q) const {
        if constexpr (std::is_same<T, __half>::value) {
            const __half2 h = *reinterpret_cast<const __half2*>(&w[q / 2]);
            return q & 1 ? __high2float(h) : __low2float(h);
        } else {
            return __uint_as_float(q & 1 ? w[q / 2] & 0xFFFF0000u : w[q / 2] << 16);
        }
    }
    static __device__ __forceinline__ void store(T* p, const float (&v)[8]) {
        uint32_t r[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(v[2 * q], v[2 * q + 1]);
                r[q] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * q], v[2 * q + 1]);
                r[q] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]);
    }
};
template <typename T> struct EightWide {
    T v[8];
    __device__ __forceinline__ void load(const T* p) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int q = 0; q < 8; q += V) load_acc<T, V>(p + q, *reinterpret_cast<T(*)[V]>(v + q));
    }
    __device__ __forceinline__ T get(int q) const { return v[q]; }
    static __device__ __forceinline__ void store(T* p, const T (&v)[8]) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int q = 0; q < 8; q += V) store_acc<T, V>(p + q, *reinterpret_cast<const T(*)[V]>(v + q));
    }
};
template <> struct Eight<float> : EightWide<float> {};
template <> struct Eight<double> : EightWide<double> {};

template <typename T>
constexpr int batch() { return sizeof(T) == 2 ? 2 : 1; }

// A thread has batch<T>() blocks of eight consecutive elements, all of whose loads are under way before the first is
// used.  STATE: `state` (device int64[2]: seed, offset) takes the place of the keys and the offset, so that a captured
// graph can be replayed with new numbers.
template <typename T, bool RESIDUAL, bool STATE>
__global__ void __launch_bounds__(256, sizeof(T) == 8 ? 4 : 5) dropout_kernel(int64_t n, const T* __restrict__ x, const T* __restrict__ residual,
                                                                              T* __restrict__ y, const __grid_constant__ Threshold threshold,
                                                                              acc_t<T> scale, const __grid_constant__ Keys given,
                                                                              uint64_t offset, const int64_t* __restrict__ state) {
    using A = acc_t<T>;
    constexpr int kBatch = batch<T>();
    constexpr int64_t stride = 256;
    const int64_t whole = n / 8, first = blockIdx.x * (kBatch * stride) + threadIdx.x;
    auto run = [&](const Keys& keys, uint64_t off) {
        Eight<T> xr[kBatch], rr[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int64_t b = first + u * stride;
            if (b < whole) {
                xr[u].load(x + b * 8);
                if (RESIDUAL) rr[u].load(residual + b * 8);
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int64_t b = first + u * stride;
            if (b > whole || (b == whole && n % 8 == 0)) return;
            bool keep[8];
            keep_flags(b, off, keys, threshold, keep);
            if (b < whole) {
                A v[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    v[q] = keep[q] ? xr[u].get(q) * scale : A(0);
                    if (RESIDUAL) v[q] += rr[u].get(q);
                }
                Eight<T>::store(y + b * 8, v);
            } else {                                 // the last, partial block
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
    };
    if constexpr (STATE)
        run(Keys(static_cast<uint64_t>(state[0])), static_cast<uint64_t>(state[1]));
    else
        run(given, offset);
}

template <typename T>
int launch_dropout(int64_t n, const void* x, const void* residual, void* y, double p, uint64_t seed, uint64_t offset,
                   const int64_t* state, cudaStream_t stream) {
    const uint64_t bar = static_cast<uint64_t>(std::nearbyint(p * 4294967296.0));
    // 2^32 (p = 1) keeps nothing: no half is above 0xFFFF and no lower half reaches 0x10000
    const uint32_t half = bar >> 32 ? 0xFFFFu : static_cast<uint32_t>(bar >> 16);
    const Threshold threshold{half << 16, half << 16 | half, bar >> 32 ? 0x10000u : static_cast<uint32_t>(bar & 0xFFFFu)};
    const acc_t<T> scale = p < 1.0 ? static_cast<acc_t<T>>(1.0 / (1.0 - p)) : acc_t<T>(0);
    const int64_t blocks = ceil_div(ceil_div(n, 8), 256 * batch<T>());
    if (blocks > INT32_MAX) return NB200_ERR_TOO_LARGE;
    const unsigned grid = static_cast<unsigned>(blocks);
    const Keys keys(seed);
    const T *xt = static_cast<const T*>(x), *rt = static_cast<const T*>(residual);
    T* yt = static_cast<T*>(y);
    if (state) {
        if (residual) dropout_kernel<T, true, true><<<grid, 256, 0, stream>>>(n, xt, rt, yt, threshold, scale, keys, offset, state);
        else dropout_kernel<T, false, true><<<grid, 256, 0, stream>>>(n, xt, rt, yt, threshold, scale, keys, offset, state);
    } else {
        if (residual) dropout_kernel<T, true, false><<<grid, 256, 0, stream>>>(n, xt, rt, yt, threshold, scale, keys, offset, state);
        else dropout_kernel<T, false, false><<<grid, 256, 0, stream>>>(n, xt, rt, yt, threshold, scale, keys, offset, state);
    }
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
