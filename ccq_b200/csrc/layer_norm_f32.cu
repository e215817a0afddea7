// Layer norm kernels for fp32 rows (layer_norm.cuh).
#include "layer_norm.cuh"

namespace ccq {

cudaError_t layer_norm_f32(const LayerNormArgs& a, bool bwd, bool vector, int* launches, int* partials) {
  return vector ? pick<float, 4>(a, bwd, launches, partials) : pick<float, 1>(a, bwd, launches, partials);
}

}  // namespace ccq
