// Tensor-core products of half operands; one file per type so that they compile side by side.
#include "linear_mma_kernel.cuh"

namespace nb200 {
NB200_MMA_TYPE(__half)
}  // namespace nb200
