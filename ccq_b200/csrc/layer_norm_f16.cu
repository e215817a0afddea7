// Layer norm kernels for fp16 rows (layer_norm.cuh).
#include "layer_norm.cuh"

namespace ccq {

cudaError_t layer_norm_f16(const LayerNormArgs& a, bool bwd, bool vector, int* launches, int* partials) {
  return vector ? pick<__half, 8>(a, bwd, launches, partials) : pick<__half, 1>(a, bwd, launches, partials);
}

}  // namespace ccq
