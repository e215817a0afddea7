// Layer norm over the last axis, forward and backward, with the forms a mixer block uses:
//
//   h = x (+ residual)     n = (h - mean) r     r = 1 / sqrt(var + eps)      (RMS: mean = 0, var = <h^2>)
//   y = n weight (+ bias)  (gated: y *= gate sigmoid(gate))
//
//   dn = dy' weight,  dy' = dy gate sigmoid(gate)   dweight = sum_rows dy' n   dbias = sum_rows dy'
//   dh = r (dn - <dn> - n <dn n>) + dh_in           (RMS: without <dn>)        <.> = mean over the row
//   dgate = dy (n weight + bias) s (1 + gate (1 - s)),  s = sigmoid(gate)
//
// A row is held in registers by TPR threads (several rows to a warp, one warp, or one block), so x is
// read once in each pass; mean and variance are two reductions over those registers in fp32.  The
// backward recomputes h from x and residual (the rounded h would put 2^-9 into dweight) and takes mean
// and r from the forward.  Blocks walk rows with a fixed stride and keep their columns' dweight and
// dbias in registers; the blocks' partials are summed in block order by a second kernel, so the result
// does not depend on timing.  Every kernel is bound by HBM: one read of each input, one write of each output.
#include "args.h"
#include "common.cuh"

namespace ccq {
namespace {

template <typename T, int VEC> struct Vec;
template <> struct Vec<float, 4> {
  static __device__ __forceinline__ void load(const float* p, float* x) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  }
  static __device__ __forceinline__ void store(float* p, const float* x) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  }
};
template <> struct Vec<__nv_bfloat16, 8> {
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* x) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float* x) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
  }
};
template <> struct Vec<__half, 8> {
  static __device__ __forceinline__ void load(const __half* p, float* x) {
    uint4 v = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void store(__half* p, const float* x) {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
  }
};
template <typename T> struct Vec<T, 1> {
  static __device__ __forceinline__ void load(const T* p, float* x) { x[0] = Act<T>::load(p); }
  static __device__ __forceinline__ void store(T* p, const float* x) { Act<T>::store(p, x[0]); }
};

// sums of two values over the TPR threads of a row (TPR <= 32: inside a warp; else the whole block)
template <int TPR>
__device__ __forceinline__ float2 row_sum(float2 x, float2* red) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) {
    x.x += __shfl_xor_sync(0xffffffffu, x.x, o);
    x.y += __shfl_xor_sync(0xffffffffu, x.y, o);
  }
  if (TPR <= 32) return x;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  float2 s = red[0];
#pragma unroll
  for (int i = 1; i < TPR / 32; ++i) {
    s.x += red[i].x;
    s.y += red[i].y;
  }
  return s;
}

__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + __expf(-x)); }

template <int TPR> constexpr int block_of() { return TPR <= 32 ? 256 : TPR; }

// One row per TPR threads; a thread holds NV vectors of VEC elements, TPR * VEC apart.
template <typename T, int VEC, int NV, int TPR, bool CENTER, bool GATE>
__global__ void __launch_bounds__(block_of<TPR>()) fwd_kernel(LayerNormArgs a) {
  constexpr int BLOCK = block_of<TPR>(), ROWS = BLOCK / TPR;
  __shared__ float2 red[32];
  const int lane = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  const bool live = row < a.rows;
  const int D = a.D;
  const int64_t base = row * D;
  float h[NV * VEC];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * VEC;
    float* x = h + i * VEC;
    if (live && c < D) {
      Vec<T, VEC>::load(reinterpret_cast<const T*>(a.x) + base + c, x);
      if (a.residual) {
        float r[VEC];
        Vec<T, VEC>::load(reinterpret_cast<const T*>(a.residual) + base + c, r);
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] += r[j];
        Vec<T, VEC>::store(reinterpret_cast<T*>(a.h) + base + c, x);
      }
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += x[j];
  }
  float mean = 0.f;
  if (CENTER) mean = row_sum<TPR>(make_float2(s, 0.f), red).x / D;
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * TPR + lane) * VEC < D) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = h[i * VEC + j] - mean;
        ss = fmaf(d, d, ss);
      }
    }
  const float r = 1.f / sqrtf(row_sum<TPR>(make_float2(ss, 0.f), red).x / D + a.eps);
  if (live && lane == 0 && a.stats) a.stats[row] = make_float2(mean, r);
  if (!live) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * VEC;
    if (c < D) {
      float y[VEC], g[VEC];
      if (GATE) Vec<T, VEC>::load(reinterpret_cast<const T*>(a.gate) + base + c, g);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        y[j] = (h[i * VEC + j] - mean) * r;
        if (a.weight) y[j] *= a.weight[c + j];
        if (a.bias) y[j] += a.bias[c + j];
        if (GATE) y[j] *= g[j] * sigmoid(g[j]);
      }
      Vec<T, VEC>::store(reinterpret_cast<T*>(a.y) + base + c, y);
    }
  }
}

// Rows blockIdx.x * ROWS + r, then gridDim.x * ROWS further on, and so on.
template <typename T, int VEC, int NV, int TPR, bool CENTER, bool GATE>
__global__ void __launch_bounds__(block_of<TPR>()) bwd_kernel(LayerNormArgs a) {
  constexpr int BLOCK = block_of<TPR>(), ROWS = BLOCK / TPR;
  __shared__ float2 red[32];
  __shared__ float fold[ROWS > 1 ? BLOCK * VEC : 1];
  const int lane = threadIdx.x % TPR, D = a.D;
  float dw[NV * VEC], db[NV * VEC];
#pragma unroll
  for (int i = 0; i < NV * VEC; ++i) dw[i] = db[i] = 0.f;
  for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < a.rows; row0 += (int64_t)gridDim.x * ROWS) {
    const int64_t row = row0 + threadIdx.x / TPR;
    const bool live = row < a.rows;
    const int64_t base = row * D;
    const float2 st = live ? a.stats[row] : make_float2(0.f, 0.f);
    float n[NV * VEC], dn[NV * VEC];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      float* x = n + i * VEC;
      float* d = dn + i * VEC;
      if (live && c < D) {
        float g[VEC], res[VEC];
        Vec<T, VEC>::load(reinterpret_cast<const T*>(a.x) + base + c, x);
        Vec<T, VEC>::load(reinterpret_cast<const T*>(a.dy) + base + c, d);
        if (GATE) Vec<T, VEC>::load(reinterpret_cast<const T*>(a.gate) + base + c, g);
        if (a.residual) Vec<T, VEC>::load(reinterpret_cast<const T*>(a.residual) + base + c, res);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (a.residual) x[j] += res[j];
          x[j] = (x[j] - st.x) * st.y;
          const float w = a.weight ? a.weight[c + j] : 1.f;
          if (GATE) {
            const float sg = sigmoid(g[j]);
            const float core = fmaf(x[j], w, a.bias ? a.bias[c + j] : 0.f);
            const float dy = d[j];
            d[j] = dy * g[j] * sg;
            g[j] = dy * core * sg * fmaf(g[j], 1.f - sg, 1.f);
          }
          dw[i * VEC + j] = fmaf(d[j], x[j], dw[i * VEC + j]);
          db[i * VEC + j] += d[j];
          d[j] *= w;
          s.x += d[j];
          s.y = fmaf(d[j], x[j], s.y);
        }
        if (GATE) Vec<T, VEC>::store(reinterpret_cast<T*>(a.dgate) + base + c, g);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = d[j] = 0.f;
      }
    }
    s = row_sum<TPR>(s, red);
    const float c1 = CENTER ? s.x / D : 0.f, c2 = s.y / D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (live && c < D) {
        float dx[VEC];
        if (a.dh) Vec<T, VEC>::load(reinterpret_cast<const T*>(a.dh) + base + c, dx);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float v = st.y * (dn[i * VEC + j] - c1 - n[i * VEC + j] * c2);
          dx[j] = a.dh ? dx[j] + v : v;
        }
        Vec<T, VEC>::store(reinterpret_cast<T*>(a.dx) + base + c, dx);
      }
    }
  }
  // this block's partials: [gridDim.x][2][D]
  float* part = a.partial + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* acc = which ? db : dw;
    if (which ? a.dbias == nullptr : a.dweight == nullptr) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (ROWS > 1) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VEC; ++j) fold[(threadIdx.x / TPR) * TPR * VEC + lane * VEC + j] = acc[i * VEC + j];
        __syncthreads();
        for (int e = threadIdx.x; e < TPR * VEC; e += BLOCK) {
          float t = 0.f;
          for (int r = 0; r < ROWS; ++r) t += fold[r * TPR * VEC + e];
          if (i * TPR * VEC + e < D) part[which * D + i * TPR * VEC + e] = t;
        }
      } else if (c < D) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) part[which * D + c + j] = acc[i * VEC + j];
      }
    }
  }
}

// dweight / dbias: the blocks' partials summed in block order, 32 columns a block, 8 slices of blocks
__global__ void __launch_bounds__(256) reduce_kernel(LayerNormArgs a, int blocks) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, which = blockIdx.y;
  float* out = which ? a.dbias : a.dweight;
  if (out == nullptr) return;
  float t = 0.f;
  if (c < a.D)
    for (int b = slice; b < blocks; b += 8) t += a.partial[((int64_t)b * 2 + which) * a.D + c];
  s[slice][lane] = t;
  __syncthreads();
  if (slice == 0 && c < a.D) {
#pragma unroll
    for (int i = 1; i < 8; ++i) t += s[i][lane];
    out[c] = t;
  }
}

__global__ void zero_kernel(float* p, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (p && i < n) p[i] = 0.f;
}

// blocks of the backward: enough to cover 148 SMs a few times, few enough that the partials stay small
inline int bwd_blocks(int64_t rows, int rows_per_block) {
  const int64_t need = (rows + rows_per_block - 1) / rows_per_block;
  const int64_t most = 148 * 4;
  return (int)(need < most ? need : most);
}

template <typename T, int VEC, int NV, int TPR>
cudaError_t run(const LayerNormArgs& a, bool bwd, int* launches) {
  constexpr int BLOCK = block_of<TPR>(), ROWS = BLOCK / TPR;
  const bool center = a.form == LN_LAYER;
  if (!bwd) {
    const unsigned grid = (unsigned)((a.rows + ROWS - 1) / ROWS);
    if (a.gate) {
      if (center) fwd_kernel<T, VEC, NV, TPR, true, true><<<grid, BLOCK, 0, a.stream>>>(a);
      else fwd_kernel<T, VEC, NV, TPR, false, true><<<grid, BLOCK, 0, a.stream>>>(a);
    } else {
      if (center) fwd_kernel<T, VEC, NV, TPR, true, false><<<grid, BLOCK, 0, a.stream>>>(a);
      else fwd_kernel<T, VEC, NV, TPR, false, false><<<grid, BLOCK, 0, a.stream>>>(a);
    }
    ++*launches;
    return cudaGetLastError();
  }
  const int blocks = bwd_blocks(a.rows, ROWS);
  if (a.gate) {
    if (center) bwd_kernel<T, VEC, NV, TPR, true, true><<<blocks, BLOCK, 0, a.stream>>>(a);
    else bwd_kernel<T, VEC, NV, TPR, false, true><<<blocks, BLOCK, 0, a.stream>>>(a);
  } else {
    if (center) bwd_kernel<T, VEC, NV, TPR, true, false><<<blocks, BLOCK, 0, a.stream>>>(a);
    else bwd_kernel<T, VEC, NV, TPR, false, false><<<blocks, BLOCK, 0, a.stream>>>(a);
  }
  ++*launches;
  if (a.dweight || a.dbias) {
    reduce_kernel<<<dim3((a.D + 31) / 32, 2), 256, 0, a.stream>>>(a, blocks);
    ++*launches;
  }
  return cudaGetLastError();
}

// Threads per row by the number of vectors in it: the fewest that keep a row in at most four
// vectors (eight scalars) a thread, so short rows share a warp and long ones take a block.
template <typename T, int VEC>
cudaError_t pick(const LayerNormArgs& a, bool bwd, int* launches) {
  const int n = (a.D + VEC - 1) / VEC;
  if (VEC > 1) {
    if (n <= 8) return run<T, VEC, 1, 8>(a, bwd, launches);
    if (n <= 16) return run<T, VEC, 1, 16>(a, bwd, launches);
    if (n <= 32) return run<T, VEC, 1, 32>(a, bwd, launches);
    if (n <= 64) return run<T, VEC, 2, 32>(a, bwd, launches);
    if (n <= 128) return run<T, VEC, 1, 128>(a, bwd, launches);
    if (n <= 256) return run<T, VEC, 1, 256>(a, bwd, launches);
    if (n <= 512) return run<T, VEC, 2, 256>(a, bwd, launches);
    if (n <= 1024) return run<T, VEC, 2, 512>(a, bwd, launches);
    return run<T, VEC, (VEC == 4 ? 4 : 2), 1024>(a, bwd, launches);
  }
  if (n <= 32) return run<T, VEC, 1, 32>(a, bwd, launches);
  if (n <= 128) return run<T, VEC, 4, 32>(a, bwd, launches);
  if (n <= 1024) return run<T, VEC, 8, 128>(a, bwd, launches);
  if (n <= 4096) return run<T, VEC, 8, 512>(a, bwd, launches);
  if (n <= 8192) return run<T, VEC, 8, 1024>(a, bwd, launches);
  return run<T, VEC, 16, 1024>(a, bwd, launches);
}

bool aligned16(const LayerNormArgs& a) {
  const uintptr_t p = (uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.gate | (uintptr_t)a.y | (uintptr_t)a.h |
                      (uintptr_t)a.dy | (uintptr_t)a.dh | (uintptr_t)a.dx | (uintptr_t)a.dgate;
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
  switch (a.dtype) {
    case DT_F32: return v ? pick<float, 4>(a, bwd, launches) : pick<float, 1>(a, bwd, launches);
    case DT_BF16: return v ? pick<__nv_bfloat16, 8>(a, bwd, launches) : pick<__nv_bfloat16, 1>(a, bwd, launches);
    default: return v ? pick<__half, 8>(a, bwd, launches) : pick<__half, 1>(a, bwd, launches);
  }
}

}  // namespace

size_t layer_norm_bwd_workspace(int64_t rows, int D) {
  if (rows == 0) return 0;
  return ws_align((size_t)bwd_blocks(rows, 1) * 2 * D * sizeof(float));
}
cudaError_t layer_norm_fwd(const LayerNormArgs& a, int* launches) { return dispatch(a, false, launches); }
cudaError_t layer_norm_bwd(const LayerNormArgs& a, int* launches) { return dispatch(a, true, launches); }

}  // namespace ccq
