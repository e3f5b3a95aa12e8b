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
__device__ __forceinline__ float exp_acc(float v) { return expf(v); }
__device__ __forceinline__ double exp_acc(double v) { return exp(v); }
__device__ __forceinline__ float erf_acc(float v) { return erff(v); }
__device__ __forceinline__ double erf_acc(double v) { return erf(v); }
__device__ __forceinline__ float tanh_acc(float v) { return tanhf(v); }
__device__ __forceinline__ double tanh_acc(double v) { return tanh(v); }

// 1 / (1 + exp(-z)).  In 32 bits with the short exponential and division, whose errors of a few units relative to
// exp(-z) are multiplied by exp(-z) / (1 + exp(-z)): they fade where they grow.  exp(-z) = infinity gives 0.
__device__ __forceinline__ float logistic(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }
__device__ __forceinline__ double logistic(double z) { return 1.0 / (1.0 + exp(-z)); }

constexpr double kRootHalf = 0.70710678118654752440;     // 1 / sqrt(2)
constexpr double kInvRoot2Pi = 0.39894228040143267794;   // 1 / sqrt(2 pi)

template <int ACT, typename A>
__device__ __forceinline__ A activate(A z) {
    if constexpr (ACT == NB200_ACT_RELU) return z > A(0) ? z : (z != z ? z : A(0));
    if constexpr (ACT == NB200_ACT_SILU) return z * logistic(z);
    if constexpr (ACT == NB200_ACT_GELU) return A(0.5) * z * (A(1) + erf_acc(z * A(kRootHalf)));
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
    if constexpr (ACT == NB200_ACT_GELU)
        return A(0.5) * (A(1) + erf_acc(z * A(kRootHalf))) + z * A(kInvRoot2Pi) * exp_acc(A(-0.5) * z * z);
    if constexpr (ACT == NB200_ACT_TANH) {
        const A t = tanh_acc(z);
        return A(1) - t * t;
    }
    return A(1);
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
