// Interface of the tensor-core product (linear_mma_kernel.cuh) to the entry points in linear.cu.
#pragma once
#include "dense_common.cuh"

namespace nb200 {

// What the epilogue of a product needs; absent parts are NULL.
template <typename T>
struct Epilogue {
    const T* bias;
    const T* residual;
    int64_t ldr;
    T* z;                 // [rows, cols] contiguous
    T* y;                 // [rows, cols] contiguous
    acc_t<T>* partial;    // instead of all of the above: [splits, rows, cols]
};

// The largest finite number of a 16-bit type.
template <typename T> __device__ __forceinline__ float largest_finite();
template <> __device__ __forceinline__ float largest_finite<__nv_bfloat16>() { return 3.3895313892515355e38f; }
template <> __device__ __forceinline__ float largest_finite<__half>() { return 65504.f; }

// Whether the slope of an activation is a number times z: at an infinity it is then 0 * infinity.
template <int ACT> constexpr bool slope_has_z() { return ACT == NB200_ACT_SILU || ACT == NB200_ACT_GELU; }

// z as the backward pass will read it: rounded to the type of the layer, a choice that halves what 16-bit layers write and
// read for it (the slope is then off by up to 0.8 |z| half-steps; measured, dx and dw of a layer of 512 x 512 bfloat16 2.4e-3
// from 64 bits, 1.7e-3 with a 32-bit z and dz).  A finite z
// stays finite in 16 bits: beyond their range the slopes are constant, so the largest number stands for it, where an
// infinity would make a NaN.  For relu only the sign counts, and rounding keeps it, except that a positive z below half
// the smallest fp16 number would become zero.
template <typename T, int ACT>
__device__ __forceinline__ T rounded_z(acc_t<T> v) {
    if constexpr (slope_has_z<ACT>() && sizeof(T) == 2)
        if (isfinite(v)) v = fminf(fmaxf(v, -largest_finite<T>()), largest_finite<T>());
    T r = from_acc<T>(v);
    if constexpr (ACT == NB200_ACT_RELU && sizeof(T) == 2)
        if (v > 0.f && to_acc(r) == 0.f) r = from_acc<T>(5.9604644775390625e-8f);   // 2^-24, representable in both types
    return r;
}

// C[i, j] = sum_k A(i, k) B(k, j).  A(i, k) is a[i * as + k] with A_K or a[i + k * as]; B(k, j) is
// b[k + j * bs] with B_K or b[k * bs + j].  The sum is cut into `splits` parts of `per` (a multiple of 64)
// terms, which needs ep.partial when splits > 1.  T: float, bfloat16 or half.
template <typename T, bool A_K, bool B_K, int ACT>
int mma_product(int64_t rows, int64_t cols, int64_t depth, int64_t splits, int64_t per, const T* a, int64_t as, const T* b, int64_t bs,
                const Epilogue<T>& ep, int32_t* status, cudaStream_t stream);

constexpr int kMmaTile = 128;     // rows and columns of a tile
constexpr int kMmaChunk = 64;     // terms of the sum that are staged together

}  // namespace nb200
