// Shared pieces of the dense operators of the graph layers (linear, group norm, dropout): the four
// value types, 16-byte vectors of them, and the activations with their derivatives.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace nb200 {

// Arithmetic type of a value type: 32 bits for everything narrower, 64 for double.
template <typename T> struct Acc { using type = float; };
template <> struct Acc<double> { using type = double; };
template <typename T> using acc_t = typename Acc<T>::type;

__device__ __forceinline__ float to_acc(float v) { return v; }
__device__ __forceinline__ double to_acc(double v) { return v; }
__device__ __forceinline__ float to_acc(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_acc(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_acc(acc_t<T> v) { return static_cast<T>(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_acc<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_acc<__half>(float v) { return __float2half_rn(v); }

// V consecutive values moved as 16-byte (or narrower) accesses; V * sizeof(T) is a power of two.
template <typename T, int V>
struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Pack {
    T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_acc(const T* p, acc_t<T> (&out)[V]) {
    const Pack<T, V> t = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int q = 0; q < V; ++q) out[q] = to_acc(t.v[q]);
}

template <typename T, int V>
__device__ __forceinline__ void store_acc(T* p, const acc_t<T> (&in)[V]) {
    Pack<T, V> t;
#pragma unroll
    for (int q = 0; q < V; ++q) t.v[q] = from_acc<T>(in[q]);
    *reinterpret_cast<Pack<T, V>*>(p) = t;
}

// ---- activations ---------------------------------------------------------------------------------
__device__ __forceinline__ float tanh_acc(float v) { return tanhf(v); }
__device__ __forceinline__ double tanh_acc(double v) { return tanh(v); }

__device__ __forceinline__ float abs_acc(float v) { return fabsf(v); }
__device__ __forceinline__ double abs_acc(double v) { return fabs(v); }
// In 32 bits the short forms, good to a few units in the last place (the exponential to 2 + 1.2 |v|).
__device__ __forceinline__ float exp_acc(float v) { return __expf(v); }
__device__ __forceinline__ double exp_acc(double v) { return exp(v); }
__device__ __forceinline__ float reciprocal(float v) { return __fdividef(1.f, v); }
__device__ __forceinline__ double reciprocal(double v) { return 1.0 / v; }

// 1 / (1 + exp(-z)).  In 32 bits with the short exponential and division, whose errors of a few units relative to
// exp(-z) are multiplied by exp(-z) / (1 + exp(-z)): they fade where they grow.  exp(-z) = infinity gives 0.
__device__ __forceinline__ float logistic(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }
__device__ __forceinline__ double logistic(double z) { return 1.0 / (1.0 + exp(-z)); }

constexpr double kRootHalf = 0.70710678118654752440;     // 1 / sqrt(2)
constexpr double kInvRoot2Pi = 0.39894228040143267794;   // 1 / sqrt(2 pi)

// The normal distribution function at z and exp(-z^2 / 2).  In 32 bits by Abramowitz and Stegun, Handbook of
// Mathematical Functions, 7.1.26: erf(x) = 1 - (a1 t + ... + a5 t^5) exp(-x^2) with t = 1 / (1 + p x), x >= 0, off by
// at most 1.5e-7, so the result is off by little more than a rounding of a number near one.  It has no branches, and
// its exponential is the one that the density needs: slope and value together cost a third of erff and expf.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    const float x = fabsf(z) * static_cast<float>(kRootHalf), t = __fdividef(1.f, fmaf(0.3275911f, x, 1.f));
    e = __expf(-x * x);
    const float poly = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float tail = 0.5f * poly * e;
    return z > 0.f ? 1.f - tail : tail;
}
__device__ __forceinline__ double normal_cdf(double z, double& e) {
    e = exp(-0.5 * z * z);
    return 0.5 * erfc(-z * kRootHalf);
}

template <int ACT, typename A>
__device__ __forceinline__ A activate(A z) {
    if constexpr (ACT == NB200_ACT_RELU) return z > A(0) ? z : (z != z ? z : A(0));
    if constexpr (ACT == NB200_ACT_SILU) return z * logistic(z);
    if constexpr (ACT == NB200_ACT_GELU) {
        A e;
        return z * normal_cdf(z, e);
    }
    if constexpr (ACT == NB200_ACT_TANH) return tanh_acc(z);
    return z;
}

// d activate(z) / dz
template <int ACT, typename A>
__device__ __forceinline__ A activate_slope(A z) {
    if constexpr (ACT == NB200_ACT_RELU) return z > A(0) ? A(1) : (z != z ? z : A(0));
    if constexpr (ACT == NB200_ACT_SILU) {
        const A s = logistic(z);
        return s * (A(1) + z * (A(1) - s));
    }
    if constexpr (ACT == NB200_ACT_GELU) {
        A e;
        const A cdf = normal_cdf(z, e);
        return cdf + z * A(kInvRoot2Pi) * e;
    }
    if constexpr (ACT == NB200_ACT_TANH) {                        // 1 - tanh^2 = 4 e / (1 + e)^2 with e = exp(-2 |z|): nothing cancels
        const A e = exp_acc(A(-2) * abs_acc(z)), r = reciprocal(A(1) + e);
        return A(4) * e * r * r;
    }
    return A(1);
}

// ---- two floats at a time: one instruction for a pair of additions, products or multiply-adds ---------------
struct Pair {
    unsigned long long bits;
    __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(a), "f"(b)); }
    __device__ __forceinline__ explicit Pair(unsigned long long v) : bits(v) {}
    __device__ __forceinline__ void to(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(bits)); }
};
__device__ __forceinline__ Pair operator+(const Pair& a, const Pair& b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.bits), "l"(b.bits));
    return Pair(r);
}
__device__ __forceinline__ Pair operator*(const Pair& a, const Pair& b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.bits), "l"(b.bits));
    return Pair(r);
}
__device__ __forceinline__ Pair fma(const Pair& a, const Pair& b, const Pair& c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
    return Pair(r);
}
__device__ __forceinline__ Pair both(float v) { return Pair(v, v); }

// activate() of two values: the same formulas, the parts outside the special functions done in pairs.
template <int ACT>
__device__ __forceinline__ void activate_pair(float& a, float& b) {
    if constexpr (ACT == NB200_ACT_SILU) {
        float ea = __expf(-a), eb = __expf(-b);
        (Pair(ea, eb) + both(1.f)).to(ea, eb);
        (Pair(a, b) * Pair(__fdividef(1.f, ea), __fdividef(1.f, eb))).to(a, b);
    } else if constexpr (ACT == NB200_ACT_GELU) {
        const Pair z(a, b), x = Pair(fabsf(a), fabsf(b)) * both(static_cast<float>(kRootHalf));
        float ta, tb, ea, eb;
        fma(x, both(0.3275911f), both(1.f)).to(ta, tb);
        const Pair t(__fdividef(1.f, ta), __fdividef(1.f, tb));
        (x * x).to(ea, eb);
        Pair poly = fma(t, both(1.061405429f), both(-1.453152027f));
        poly = fma(t, poly, both(1.421413741f));
        poly = fma(t, poly, both(-0.284496736f));
        poly = fma(t, poly, both(0.254829592f));
        const Pair tail = t * poly * Pair(0.5f * __expf(-ea), 0.5f * __expf(-eb));
        float ca, cb, na, nb;
        tail.to(ca, cb);
        fma(tail, both(-1.f), both(1.f)).to(na, nb);
        (z * Pair(a > 0.f ? na : ca, b > 0.f ? nb : cb)).to(a, b);
    } else {
        a = activate<ACT>(a);
        b = activate<ACT>(b);
    }
}

// The slopes at two values; in pairs only where that is faster (silu's slope pass over a million rows of 128 floats took
// 291 us in pairs against 257).
template <int ACT>
__device__ __forceinline__ void slope_pair(float& a, float& b) {
    if constexpr (ACT == NB200_ACT_GELU) {
        const Pair z(a, b), x = Pair(fabsf(a), fabsf(b)) * both(static_cast<float>(kRootHalf));
        float ta, tb, ea, eb;
        fma(x, both(0.3275911f), both(1.f)).to(ta, tb);
        const Pair t(__fdividef(1.f, ta), __fdividef(1.f, tb));
        (x * x).to(ea, eb);
        Pair poly = fma(t, both(1.061405429f), both(-1.453152027f));
        poly = fma(t, poly, both(1.421413741f));
        poly = fma(t, poly, both(-0.284496736f));
        poly = fma(t, poly, both(0.254829592f));
        const Pair e(__expf(-ea), __expf(-eb)), tail = t * poly * both(0.5f) * e;
        float ca, cb, na, nb;
        tail.to(ca, cb);
        fma(tail, both(-1.f), both(1.f)).to(na, nb);
        fma(z * both(static_cast<float>(kInvRoot2Pi)), e, Pair(a > 0.f ? na : ca, b > 0.f ? nb : cb)).to(a, b);
    } else {
        a = activate_slope<ACT>(a);
        b = activate_slope<ACT>(b);
    }
}

// V values in place.
template <int ACT, typename A, int V>
__device__ __forceinline__ void activate_all(A (&z)[V]) {
    if constexpr (sizeof(A) == 4 && V % 2 == 0) {
#pragma unroll
        for (int q = 0; q < V; q += 2) activate_pair<ACT>(z[q], z[q + 1]);
    } else {
#pragma unroll
        for (int q = 0; q < V; ++q) z[q] = activate<ACT>(z[q]);
    }
}
template <int ACT, typename A, int V>
__device__ __forceinline__ void slope_all(A (&z)[V]) {
    if constexpr (sizeof(A) == 4 && V % 2 == 0) {
#pragma unroll
        for (int q = 0; q < V; q += 2) slope_pair<ACT>(z[q], z[q + 1]);
    } else {
#pragma unroll
        for (int q = 0; q < V; ++q) z[q] = activate_slope<ACT>(z[q]);
    }
}

inline bool known_activation(int act) { return act >= NB200_ACT_NONE && act <= NB200_ACT_TANH; }
inline bool known_dense_dtype(int dtype) { return dtype >= NB200_F32 && dtype <= NB200_F16; }
inline size_t dense_dtype_size(int dtype) { return dtype == NB200_F64 ? 8 : dtype == NB200_F32 ? 4 : 2; }

}  // namespace nb200

// Dispatch on the four value types of the dense operators / on the activation (a constant ACT).
#define NB200_DISPATCH_DENSE(dtype, CALL)                                         \
    [&]() -> int {                                                                \
        if ((dtype) == NB200_F32) { using T = float; return CALL; }               \
        if ((dtype) == NB200_F64) { using T = double; return CALL; }              \
        if ((dtype) == NB200_BF16) { using T = __nv_bfloat16; return CALL; }      \
        if ((dtype) == NB200_F16) { using T = __half; return CALL; }              \
        return NB200_ERR_BAD_ARG;                                                 \
    }()

#define NB200_DISPATCH_ACT(act, CALL)                                             \
    [&]() -> int {                                                                \
        if ((act) == NB200_ACT_NONE) { constexpr int ACT = NB200_ACT_NONE; return CALL; } \
        if ((act) == NB200_ACT_RELU) { constexpr int ACT = NB200_ACT_RELU; return CALL; } \
        if ((act) == NB200_ACT_SILU) { constexpr int ACT = NB200_ACT_SILU; return CALL; } \
        if ((act) == NB200_ACT_GELU) { constexpr int ACT = NB200_ACT_GELU; return CALL; } \
        if ((act) == NB200_ACT_TANH) { constexpr int ACT = NB200_ACT_TANH; return CALL; } \
        return NB200_ERR_BAD_ARG;                                                 \
    }()
