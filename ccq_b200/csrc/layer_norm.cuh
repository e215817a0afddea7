// Layer norm over the last axis, forward and backward, with the forms a mixer block uses:
//
//   h = x (+ residual)     n = (h - mean) r     r = 1 / sqrt(var + eps)      (RMS: mean = 0, var = <h^2>)
//   y = n weight (+ bias)  (gated: y *= gate sigmoid(gate))
//
//   dn = dy' weight,  dy' = dy gate sigmoid(gate)   dweight = sum_rows dy' n   dbias = sum_rows dy'
//   dh = r (dn - <dn> - n <dn n>) + dh_in           (RMS: without <dn>)        <.> = mean over the row
//   dgate = dy (n weight + bias) s (1 + gate (1 - s)),  s = sigmoid(gate)
//
// A row is held in registers by TPR threads, so x is read once in each pass; mean and variance are two
// reductions over those registers in fp32.  The kernels are bound by HBM (one read of each input, one write of
// each output), which takes enough loads in flight: the forward gives a row to as few threads as hold
// it (a warp up to 2048 16-bit elements: eight loads a thread and no block barrier) and several short rows to
// each; the backward, whose threads also keep their columns' dweight and dbias, gives a thread one vector of a
// row and loads its next row before it reduces the present one.  The backward recomputes h from x and
// residual (the rounded h would put 2^-9 into dweight) and takes mean and r from the forward.  Blocks walk
// rows with a fixed stride, and their partial dweight and dbias are summed in block order by a second
// kernel, so the result does not depend on timing.  bf16, forward and backward: 32768 rows of 2048 with a residual
// (940 MB) 222 us, 4.2 TB/s; 524288 gated rows of 128 (805 MB) 210 us, 3.8 TB/s.
#pragma once

#include "args.h"
#include "common.cuh"

namespace ccq {
namespace {

// VEC elements as they are loaded (Raw) and as fp32
template <typename T, int VEC> struct Vec;
template <> struct Vec<float, 4> {
  using Raw = float4;
  static __device__ __forceinline__ void unpack(const Raw& v, float* x) {
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  }
  static __device__ __forceinline__ Raw pack(const float* x) { return make_float4(x[0], x[1], x[2], x[3]); }
};
template <> struct Vec<__nv_bfloat16, 8> {
  using Raw = uint4;
  static __device__ __forceinline__ void unpack(const Raw& v, float* x) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ Raw pack(const float* x) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    return *reinterpret_cast<Raw*>(h);
  }
};
template <> struct Vec<__half, 8> {
  using Raw = uint4;
  static __device__ __forceinline__ void unpack(const Raw& v, float* x) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ Raw pack(const float* x) {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    return *reinterpret_cast<Raw*>(h);
  }
};
template <typename T> struct Vec<T, 1> {
  using Raw = T;
  static __device__ __forceinline__ void unpack(const Raw& v, float* x) { x[0] = Act<T>::load(&v); }
  static __device__ __forceinline__ Raw pack(const float* x) {
    Raw r;
    Act<T>::store(&r, x[0]);
    return r;
  }
};
template <typename T, int VEC>
__device__ __forceinline__ typename Vec<T, VEC>::Raw load_raw(const void* base, int64_t at) {
  return *reinterpret_cast<const typename Vec<T, VEC>::Raw*>(reinterpret_cast<const T*>(base) + at);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_raw(void* base, int64_t at, const float* x) {
  *reinterpret_cast<typename Vec<T, VEC>::Raw*>(reinterpret_cast<T*>(base) + at) = Vec<T, VEC>::pack(x);
}

// VEC consecutive fp32 parameters (vectors start on 16-byte boundaries)
template <int VEC>
__device__ __forceinline__ void load_param(const float* p, float* x) {
  if (VEC == 1) {
    x[0] = p[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    }
  }
}

// sums of two values over the TPR threads of a row (TPR <= 32: inside a warp; else the whole block, with one
// barrier: calls alternate between two buffers)
template <int TPR>
__device__ __forceinline__ float2 row_sum(float2 x, float2 (*red)[32], int& turn) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) {
    x.x += __shfl_xor_sync(0xffffffffu, x.x, o);
    x.y += __shfl_xor_sync(0xffffffffu, x.y, o);
  }
  if (TPR <= 32) return x;
  float2* r = red[turn];
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = x;
  __syncthreads();
  float2 s = r[0];
#pragma unroll
  for (int i = 1; i < TPR / 32; ++i) {
    s.x += r[i].x;
    s.y += r[i].y;
  }
  return s;
}

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

template <int TPR> constexpr int block_of() { return TPR <= 32 ? 256 : TPR; }
// Blocks of the backward an SM must hold.  With one vector a thread: 1024 threads (64 registers each), but 768
// with the residual forms' five loads, which spill at 64 (bf16, 512 / 768 / 1024 threads: 65536 x 1024 rms
// 109 / 89 / 82 us, 524288 x 128 gated 171 / 130 / 124 us, 32768 x 2048 with residual 146 / 119 / 151 us).
template <int ELEMS, int TPR, bool RES> constexpr int bwd_per_sm() {
  constexpr int threads = RES ? 768 : 1024, block = block_of<TPR>();
  return ELEMS <= 8 && block <= threads ? threads / block : 1;
}

// One row per TPR threads, RPT such rows in turn (their loads first); a thread holds NV vectors of VEC
// elements, TPR * VEC apart.
template <typename T, int VEC, int NV, int TPR, int RPT, bool CENTER, bool GATE, bool RES>
__global__ void __launch_bounds__(block_of<TPR>()) fwd_kernel(LayerNormArgs a) {
  constexpr int BLOCK = block_of<TPR>(), ROWS = BLOCK / TPR;
  using V = Vec<T, VEC>;
  __shared__ float2 red[2][32];
  int turn = 0;
  const int lane = threadIdx.x % TPR, D = a.D;
  const int64_t row0 = (int64_t)blockIdx.x * ROWS * RPT + threadIdx.x / TPR;
  typename V::Raw rx[RPT][NV], rr[RPT][NV];
#pragma unroll
  for (int q = 0; q < RPT; ++q)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      const int64_t row = row0 + (int64_t)q * ROWS;
      if (row < a.rows && c < D) {
        rx[q][i] = load_raw<T, VEC>(a.x, row * D + c);
        if (GATE) rr[q][i] = load_raw<T, VEC>(a.gate, row * D + c);
        else if (RES) rr[q][i] = load_raw<T, VEC>(a.residual, row * D + c);
      }
    }
#pragma unroll
  for (int q = 0; q < RPT; ++q) {
    const int64_t row = row0 + (int64_t)q * ROWS;
    const bool live = row < a.rows;
    const int64_t base = row * D;
    float h[NV * VEC];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      float* x = h + i * VEC;
      if (live && c < D) {
        V::unpack(rx[q][i], x);
        if (RES) {
          float r[VEC];
          V::unpack(rr[q][i], r);
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[j] += r[j];
          store_raw<T, VEC>(a.h, base + c, x);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += x[j];
    }
    float mean = 0.f;
    if (CENTER) mean = row_sum<TPR>(make_float2(s, 0.f), red, turn).x / D;
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
    const float r = 1.f / sqrtf(row_sum<TPR>(make_float2(ss, 0.f), red, turn).x / D + a.eps);
    if (live && lane == 0 && a.stats) a.stats[row] = make_float2(mean, r);
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c < D) {
        float y[VEC], p[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = (h[i * VEC + j] - mean) * r;
        if (a.weight) {
          load_param<VEC>(a.weight + c, p);
#pragma unroll
          for (int j = 0; j < VEC; ++j) y[j] *= p[j];
        }
        if (CENTER && a.bias) {
          load_param<VEC>(a.bias + c, p);
#pragma unroll
          for (int j = 0; j < VEC; ++j) y[j] += p[j];
        }
        if (GATE) {
          V::unpack(rr[q][i], p);
#pragma unroll
          for (int j = 0; j < VEC; ++j) y[j] *= p[j] * sigmoid(p[j]);
        }
        store_raw<T, VEC>(a.y, base + c, y);
      }
    }
  }
}

// Rows blockIdx.x * ROWS + r, then gridDim.x * ROWS further on, and so on.
template <typename T, int VEC, int NV, int TPR, bool CENTER, bool GATE, bool RES>
__global__ void __launch_bounds__(block_of<TPR>(), bwd_per_sm<NV * VEC, TPR, RES>()) bwd_kernel(LayerNormArgs a) {
  constexpr int BLOCK = block_of<TPR>(), ROWS = BLOCK / TPR;
  // the next row's loads go out early where registers allow: one vector a thread
  constexpr bool AHEAD = NV * VEC <= 8;
  using V = Vec<T, VEC>;
  using Raw = typename V::Raw;
  __shared__ float2 red[2][32];
  __shared__ float fold[ROWS > 1 ? BLOCK * VEC : 1];
  int turn = 0;
  const int lane = threadIdx.x % TPR, D = a.D;
  float dw[NV * VEC], db[NV * VEC], wt[NV * VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      dw[i * VEC + j] = db[i * VEC + j] = 0.f;
      wt[i * VEC + j] = 1.f;
    }
    if (a.weight && c < D) load_param<VEC>(a.weight + c, wt + i * VEC);
  }
  Raw rx[NV], ry[NV], rr[NV], rg[NV], rh[NV];
  float2 st;
  auto fetch = [&](int64_t row) {
    const bool live = row < a.rows;
    st = live ? a.stats[row] : make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (live && c < D) {
        rx[i] = load_raw<T, VEC>(a.x, row * D + c);
        ry[i] = load_raw<T, VEC>(a.dy, row * D + c);
        if (GATE) rg[i] = load_raw<T, VEC>(a.gate, row * D + c);
        if (RES) rr[i] = load_raw<T, VEC>(a.residual, row * D + c);
        if (RES && a.dh) rh[i] = load_raw<T, VEC>(a.dh, row * D + c);
      }
    }
  };
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  if (AHEAD) fetch((int64_t)blockIdx.x * ROWS + threadIdx.x / TPR);
  for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < a.rows; row0 += stride) {
    const int64_t row = row0 + threadIdx.x / TPR;
    const bool live = row < a.rows;
    const int64_t base = row * D;
    if (!AHEAD) fetch(row);
    float n[NV * VEC], dn[NV * VEC], dh[NV * VEC];
    const float r = st.y;
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      float* x = n + i * VEC;
      float* d = dn + i * VEC;
      if (live && c < D) {
        float t[VEC];
        V::unpack(rx[i], x);
        V::unpack(ry[i], d);
        if (RES && a.dh) V::unpack(rh[i], dh + i * VEC);
        if (RES) {
          V::unpack(rr[i], t);
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[j] += t[j];
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = (x[j] - st.x) * r;
        if (GATE) {
          float g[VEC];
          V::unpack(rg[i], g);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float sg = sigmoid(g[j]);
            const float core = x[j] * wt[i * VEC + j];
            t[j] = d[j] * core * sg * fmaf(g[j], 1.f - sg, 1.f);
            d[j] *= g[j] * sg;
          }
          store_raw<T, VEC>(a.dgate, base + c, t);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          dw[i * VEC + j] = fmaf(d[j], x[j], dw[i * VEC + j]);
          if (CENTER) db[i * VEC + j] += d[j];
          d[j] *= wt[i * VEC + j];
          if (CENTER) s.x += d[j];
          s.y = fmaf(d[j], x[j], s.y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = d[j] = 0.f;
      }
    }
    if (AHEAD) fetch(row + stride);
    s = row_sum<TPR>(s, red, turn);
    const float c1 = CENTER ? s.x / D : 0.f, c2 = s.y / D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (live && c < D) {
        float dx[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float v = r * ((CENTER ? dn[i * VEC + j] - c1 : dn[i * VEC + j]) - n[i * VEC + j] * c2);
          dx[j] = RES && a.dh ? dh[i * VEC + j] + v : v;
        }
        store_raw<T, VEC>(a.dx, base + c, dx);
      }
    }
  }
  // this block's partials: [gridDim.x][2][D]
  float* part = a.partial + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int which = 0; which < (CENTER ? 2 : 1); ++which) {
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
          for (int q = 0; q < ROWS; ++q) t += fold[q * TPR * VEC + e];
          if (i * TPR * VEC + e < D) part[which * D + i * TPR * VEC + e] = t;
        }
      } else if (c < D) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) part[which * D + c + j] = acc[i * VEC + j];
      }
    }
  }
}

// blocks of the backward: those that run at once, so that none is left for a second wave
inline int bwd_blocks(int64_t rows, int rows_per_block, int per_sm) {
  const int64_t need = (rows + rows_per_block - 1) / rows_per_block, most = 148 * (int64_t)per_sm;
  return (int)(need < most ? need : most);
}

template <typename T, int VEC, int NV, int TPR, int RPT>
cudaError_t run_fwd(const LayerNormArgs& a, int* launches) {
  constexpr int BLOCK = block_of<TPR>(), ROWS = BLOCK / TPR * RPT;
  const unsigned grid = (unsigned)((a.rows + ROWS - 1) / ROWS);
  if (a.gate) fwd_kernel<T, VEC, NV, TPR, RPT, false, true, false><<<grid, BLOCK, 0, a.stream>>>(a);
  else if (a.form == LN_LAYER && a.residual) fwd_kernel<T, VEC, NV, TPR, RPT, true, false, true><<<grid, BLOCK, 0, a.stream>>>(a);
  else if (a.form == LN_LAYER) fwd_kernel<T, VEC, NV, TPR, RPT, true, false, false><<<grid, BLOCK, 0, a.stream>>>(a);
  else if (a.residual) fwd_kernel<T, VEC, NV, TPR, RPT, false, false, true><<<grid, BLOCK, 0, a.stream>>>(a);
  else fwd_kernel<T, VEC, NV, TPR, RPT, false, false, false><<<grid, BLOCK, 0, a.stream>>>(a);
  ++*launches;
  return cudaGetLastError();
}

template <typename T, int VEC, int NV, int TPR>
cudaError_t run_bwd(const LayerNormArgs& a, int* launches, int* partials) {
  constexpr int BLOCK = block_of<TPR>(), ROWS = BLOCK / TPR;
  const int blocks = bwd_blocks(a.rows, ROWS, a.residual ? bwd_per_sm<NV * VEC, TPR, true>() : bwd_per_sm<NV * VEC, TPR, false>());
  if (a.gate) bwd_kernel<T, VEC, NV, TPR, false, true, false><<<blocks, BLOCK, 0, a.stream>>>(a);
  else if (a.form == LN_LAYER && a.residual) bwd_kernel<T, VEC, NV, TPR, true, false, true><<<blocks, BLOCK, 0, a.stream>>>(a);
  else if (a.form == LN_LAYER) bwd_kernel<T, VEC, NV, TPR, true, false, false><<<blocks, BLOCK, 0, a.stream>>>(a);
  else if (a.residual) bwd_kernel<T, VEC, NV, TPR, false, false, true><<<blocks, BLOCK, 0, a.stream>>>(a);
  else bwd_kernel<T, VEC, NV, TPR, false, false, false><<<blocks, BLOCK, 0, a.stream>>>(a);
  ++*launches;
  *partials = blocks;
  return cudaGetLastError();
}

// Forward: short rows four to a thread while there are rows enough to fill the SMs (148, 2048 threads
// each) that way, else one; a warp a row as far as eight vectors a thread go.
template <typename T, int VEC>
cudaError_t pick_fwd(const LayerNormArgs& a, int* launches) {
  const int n = (a.D + VEC - 1) / VEC;
  if (VEC > 1) {
    const bool many = a.rows * n >= 4 * 148 * 2048;
    if (n <= 8) return many ? run_fwd<T, VEC, 1, 8, 4>(a, launches) : run_fwd<T, VEC, 1, 8, 1>(a, launches);
    if (n <= 16) return many ? run_fwd<T, VEC, 1, 16, 4>(a, launches) : run_fwd<T, VEC, 1, 16, 1>(a, launches);
    if (n <= 32) return many ? run_fwd<T, VEC, 1, 32, 4>(a, launches) : run_fwd<T, VEC, 1, 32, 1>(a, launches);
    if (n <= 64) return run_fwd<T, VEC, 2, 32, 1>(a, launches);
    if (n <= 128) return run_fwd<T, VEC, 4, 32, 1>(a, launches);
    if (n <= 256) return run_fwd<T, VEC, 8, 32, 1>(a, launches);
    if (n <= 512) return run_fwd<T, VEC, 4, 128, 1>(a, launches);
    if (n <= 1024) return run_fwd<T, VEC, 4, 256, 1>(a, launches);
    if (n <= 2048) return run_fwd<T, VEC, 4, 512, 1>(a, launches);
    return run_fwd<T, VEC, 4, 1024, 1>(a, launches);
  }
  if (n <= 32) return run_fwd<T, VEC, 1, 32, 1>(a, launches);
  if (n <= 128) return run_fwd<T, VEC, 4, 32, 1>(a, launches);
  if (n <= 1024) return run_fwd<T, VEC, 8, 128, 1>(a, launches);
  if (n <= 4096) return run_fwd<T, VEC, 8, 512, 1>(a, launches);
  if (n <= 8192) return run_fwd<T, VEC, 8, 1024, 1>(a, launches);
  return run_fwd<T, VEC, 16, 1024, 1>(a, launches);
}

// Backward: one vector a thread up to blocks of 512 threads.
template <typename T, int VEC>
cudaError_t pick_bwd(const LayerNormArgs& a, int* launches, int* partials) {
  const int n = (a.D + VEC - 1) / VEC;
  if (VEC > 1) {
    if (n <= 8) return run_bwd<T, VEC, 1, 8>(a, launches, partials);
    if (n <= 16) return run_bwd<T, VEC, 1, 16>(a, launches, partials);
    if (n <= 32) return run_bwd<T, VEC, 1, 32>(a, launches, partials);
    if (n <= 64) return run_bwd<T, VEC, 1, 64>(a, launches, partials);
    if (n <= 128) return run_bwd<T, VEC, 1, 128>(a, launches, partials);
    if (n <= 256) return run_bwd<T, VEC, 1, 256>(a, launches, partials);
    if (n <= 512) return run_bwd<T, VEC, 1, 512>(a, launches, partials);
    if (n <= 1024) return run_bwd<T, VEC, 2, 512>(a, launches, partials);
    return run_bwd<T, VEC, (VEC == 4 ? 4 : 2), 1024>(a, launches, partials);
  }
  if (n <= 32) return run_bwd<T, VEC, 1, 32>(a, launches, partials);
  if (n <= 128) return run_bwd<T, VEC, 4, 32>(a, launches, partials);
  if (n <= 1024) return run_bwd<T, VEC, 8, 128>(a, launches, partials);
  if (n <= 4096) return run_bwd<T, VEC, 8, 512>(a, launches, partials);
  if (n <= 8192) return run_bwd<T, VEC, 8, 1024>(a, launches, partials);
  return run_bwd<T, VEC, 16, 1024>(a, launches, partials);
}

template <typename T, int VEC>
cudaError_t pick(const LayerNormArgs& a, bool bwd, int* launches, int* partials) {
  return bwd ? pick_bwd<T, VEC>(a, launches, partials) : pick_fwd<T, VEC>(a, launches);
}

}  // namespace
}  // namespace ccq
