// Layer norm kernels for bf16 rows (layer_norm.cuh).
#include "layer_norm.cuh"

namespace ccq {

cudaError_t layer_norm_bf16(const LayerNormArgs& a, bool bwd, bool vector, int* launches, int* partials) {
  return vector ? pick<__nv_bfloat16, 8>(a, bwd, launches, partials) : pick<__nv_bfloat16, 1>(a, bwd, launches, partials);
}

}  // namespace ccq
