// Tensor-core products of bfloat16 operands; one file per type so that they compile side by side.
#include "linear_mma_kernel.cuh"

namespace nb200 {
NB200_MMA_TYPE(__nv_bfloat16)
}  // namespace nb200
