// Layer norm: which kernels a call takes, the sums of the weight gradients, the workspace (layer_norm.cuh has the
// kernels and their reasons).
#include "args.h"
#include "common.cuh"

namespace ccq {

cudaError_t layer_norm_f32(const LayerNormArgs& a, bool bwd, bool vector, int* launches, int* partials);
cudaError_t layer_norm_bf16(const LayerNormArgs& a, bool bwd, bool vector, int* launches, int* partials);
cudaError_t layer_norm_f16(const LayerNormArgs& a, bool bwd, bool vector, int* launches, int* partials);

namespace {

// dweight / dbias: the blocks' partials summed in block order: 32 columns a block, 32 slices of the blocks
__global__ void __launch_bounds__(1024) reduce_kernel(LayerNormArgs a, int blocks) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, which = blockIdx.y;
  float* out = which ? a.dbias : a.dweight;
  if (out == nullptr) return;
  float t = 0.f;
  if (c < a.D) {
    const int per = (blocks + 31) / 32, end = min(blocks, (slice + 1) * per);
#pragma unroll 8
    for (int b = slice * per; b < end; ++b) t += a.partial[((int64_t)b * 2 + which) * a.D + c];
  }
  s[slice][lane] = t;
  __syncthreads();
  if (slice == 0 && c < a.D) {
#pragma unroll
    for (int i = 1; i < 32; ++i) t += s[i][lane];
    out[c] = t;
  }
}

__global__ void zero_kernel(float* p, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (p && i < n) p[i] = 0.f;
}

bool aligned16(const LayerNormArgs& a) {
  const uintptr_t p = (uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.gate | (uintptr_t)a.y | (uintptr_t)a.h |
                      (uintptr_t)a.dy | (uintptr_t)a.dh | (uintptr_t)a.dx | (uintptr_t)a.dgate | (uintptr_t)a.weight |
                      (uintptr_t)a.bias;
  return (p & 15) == 0;
}

cudaError_t dispatch(const LayerNormArgs& a, bool bwd, int* launches) {
  if (a.rows == 0) {
    if (bwd) {
      zero_kernel<<<(a.D + 255) / 256, 256, 0, a.stream>>>(a.dweight, a.D);
      zero_kernel<<<(a.D + 255) / 256, 256, 0, a.stream>>>(a.dbias, a.D);
      *launches += 2;
    }
    return cudaGetLastError();
  }
  const int vec = a.dtype == DT_F32 ? 4 : 8;
  const bool v = a.D % vec == 0 && aligned16(a);
  int partials = 0;
  cudaError_t e = a.dtype == DT_F32 ? layer_norm_f32(a, bwd, v, launches, &partials)
                  : a.dtype == DT_BF16 ? layer_norm_bf16(a, bwd, v, launches, &partials)
                                       : layer_norm_f16(a, bwd, v, launches, &partials);
  if (e == cudaSuccess && bwd && (a.dweight || a.dbias)) {
    reduce_kernel<<<dim3((a.D + 31) / 32, 2), 1024, 0, a.stream>>>(a, partials);
    ++*launches;
    e = cudaGetLastError();
  }
  return e;
}

}  // namespace

size_t layer_norm_bwd_workspace(int64_t rows, int D) {
  if (rows == 0) return 0;
  return ws_align((size_t)(rows < LN_BWD_BLOCKS ? rows : LN_BWD_BLOCKS) * 2 * D * sizeof(float));
}
cudaError_t layer_norm_fwd(const LayerNormArgs& a, int* launches) { return dispatch(a, false, launches); }
cudaError_t layer_norm_bwd(const LayerNormArgs& a, int* launches) { return dispatch(a, true, launches); }

}  // namespace ccq
