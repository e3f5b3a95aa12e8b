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

// z as the backward pass will read it.  Rounding to 16 bits keeps the sign, which is all that relu's slope
// needs, except that a positive z below half the smallest fp16 number would become zero.
template <typename T, int ACT>
__device__ __forceinline__ T rounded_z(acc_t<T> v) {
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
