// Gated delta rule token by token over a cache: the state update and read of gdr.h, fp32 throughout.
//
// A block owns 4 LV columns of one (document, value head) state and keeps them in registers for all its
// tokens: LV lanes of a warp take four neighbouring columns each (one 16-byte access a row), the other
// 32 / LV lane groups and the warps split the K rows, neighbouring rows to a thread, whose k and q it then
// loads eight at a time.  Both products of a token, S^T k and S^T q, are formed in the same pass over the
// decayed state, since the read after the update is
//   S_new^T q = S^T q + (k . q) u,
// so a token costs one reduction over the block.  A state row is read once and written once: with one
// token the kernel is bound by HBM (8 K V bytes a head), with more by instructions, which packed arithmetic
// halves.  256 requests, 16 heads, K = V = 128, 537 MB of state: 4 warps of 16 rows a thread 88 us, 6.1 TB/s
// (four tokens 124 us); 2 of 32 95 us (143), 8 of 8 90 us (174); 128 columns a block instead of 64: 90 us (141).
// With few heads the kernel is bound by latency, so the launcher narrows
// the block to 32 or 16 columns until the grid covers the SMs.  Each element is read and written by one
// thread, so the state may be updated in place.
#include "gdr.h"

namespace ccq {
namespace {

// four columns, two to an instruction
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ void scale4(float4& d, float s) {
  uint64_t lo, hi;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(lo) : "l"(pair(d.x, d.y)), "l"(pair(s, s)));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(hi) : "l"(pair(d.z, d.w)), "l"(pair(s, s)));
  unpair(lo, d.x, d.y);
  unpair(hi, d.z, d.w);
}
__device__ __forceinline__ void fma4(float4& d, const float4& x, float s) {
  uint64_t lo, hi;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(lo) : "l"(pair(x.x, x.y)), "l"(pair(s, s)), "l"(pair(d.x, d.y)));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(hi) : "l"(pair(x.z, x.w)), "l"(pair(s, s)), "l"(pair(d.z, d.w)));
  unpair(lo, d.x, d.y);
  unpair(hi, d.z, d.w);
}
__device__ __forceinline__ void add4(float4& d, const float4& x) {
  d.x += x.x;
  d.y += x.y;
  d.z += x.z;
  d.w += x.w;
}
__device__ __forceinline__ float4 shfl_xor4(const float4& x, int o) {
  return make_float4(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o),
                     __shfl_xor_sync(0xffffffffu, x.z, o), __shfl_xor_sync(0xffffffffu, x.w, o));
}

// four columns from v0 of a row of V values; VEC4: V is a multiple of 4 and rows are 16-byte aligned
template <bool VEC4>
__device__ __forceinline__ float4 load_state(const float* row, int v0, int V) {
  if (VEC4) return v0 < V ? __ldcs(reinterpret_cast<const float4*>(row + v0)) : make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(v0 < V ? row[v0] : 0.f, v0 + 1 < V ? row[v0 + 1] : 0.f, v0 + 2 < V ? row[v0 + 2] : 0.f,
                     v0 + 3 < V ? row[v0 + 3] : 0.f);
}
template <bool VEC4>
__device__ __forceinline__ void store_state(float* row, int v0, int V, const float4& x) {
  if (VEC4) {
    if (v0 < V) __stcs(reinterpret_cast<float4*>(row + v0), x);
    return;
  }
  if (v0 < V) row[v0] = x.x;
  if (v0 + 1 < V) row[v0 + 1] = x.y;
  if (v0 + 2 < V) row[v0 + 2] = x.z;
  if (v0 + 3 < V) row[v0 + 3] = x.w;
}

// ROWS values from r0 of a row of K; VEC: K is a multiple of 8 and the row starts on a 16-byte boundary
template <typename TI, int ROWS, bool VEC>
__device__ __forceinline__ void load_values(const TI* p, int r0, int K, float* x) {
  if (VEC && ROWS % 8 == 0) {
#pragma unroll
    for (int i = 0; i < ROWS; i += 8) {
      uint4 u[sizeof(TI) / 2] = {};
      if (r0 + i < K) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(TI) / 2; ++j) u[j] = reinterpret_cast<const uint4*>(p + r0 + i)[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i + j] = Act<TI>::load(reinterpret_cast<const TI*>(u) + j);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) x[i] = r0 + i < K ? Act<TI>::load(p + r0 + i) : 0.f;
}

// WARPS * (32 / LV) groups of ROWS neighbouring rows
template <typename TI, int LV, int WARPS, int ROWS, bool VEC4>
__global__ void __launch_bounds__(WARPS * 32) step_kernel(GdrArgs a) {
  constexpr int GROUPS = 32 / LV, VT = 4 * LV;
  __shared__ float4 part[2][2][WARPS][LV];  // token parity; S^T k, S^T q; warp; columns
  __shared__ float kq[2][WARPS];
  const int n = blockIdx.x / a.HV, hv = blockIdx.x % a.HV, h = hv / (a.HV / a.H);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lv = lane % LV, row0 = (warp * GROUPS + lane / LV) * ROWS;
  const int v0 = blockIdx.y * VT + 4 * lv;
  const Seq sq = seq_of(n, a.T, a.cu_seqlens);
  const int64_t st = ((int64_t)n * a.HV + hv) * a.K * a.V;
  float4 S[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = row0 + i;
    S[i] = (a.initial_state && r < a.K) ? load_state<VEC4>(a.initial_state + st + (int64_t)r * a.V, v0, a.V)
                                        : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int t = 0; t < sq.len; ++t) {
    const int64_t tok = sq.bos + t;
    const TI* kp = reinterpret_cast<const TI*>(a.k) + (tok * a.H + h) * a.K;
    const TI* qp = reinterpret_cast<const TI*>(a.q) + (tok * a.H + h) * a.K;
    const float decay = expf(gate_load(a.g, a.g_dtype, tok * a.HV + hv));
    const float beta = gate_load(a.beta, a.beta_dtype, tok * a.HV + hv);
    const TI* vp = reinterpret_cast<const TI*>(a.v) + (tok * a.HV + hv) * a.V;
    float vv[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) vv[c] = v0 + c < a.V ? Act<TI>::load(vp + v0 + c) : 0.f;
    float k[ROWS], q[ROWS];
    load_values<TI, ROWS, VEC4>(kp, row0, a.K, k);
    load_values<TI, ROWS, VEC4>(qp, row0, a.K, q);
    float4 sk = make_float4(0.f, 0.f, 0.f, 0.f), sqv = sk;
    float dot = 0.f;
    if (decay == 0.f) {  // empties the state whatever it holds
#pragma unroll
      for (int i = 0; i < ROWS; ++i) S[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      scale4(S[i], decay);
      fma4(sk, S[i], k[i]);
      fma4(sqv, S[i], q[i]);
      dot = fmaf(k[i], q[i], dot);
    }
#pragma unroll
    for (int o = LV; o < 32; o <<= 1) {
      add4(sk, shfl_xor4(sk, o));
      add4(sqv, shfl_xor4(sqv, o));
      dot += __shfl_xor_sync(0xffffffffu, dot, o);
    }
    const int p = t & 1;
    if (lane < LV) {
      part[p][0][warp][lane] = sk;
      part[p][1][warp][lane] = sqv;
    }
    if (lane == 0) kq[p][warp] = dot;
    __syncthreads();
    sk = part[p][0][0][lv];
    sqv = part[p][1][0][lv];
    dot = kq[p][0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) {
      add4(sk, part[p][0][w][lv]);
      add4(sqv, part[p][1][w][lv]);
      dot += kq[p][w];
    }
    const float4 u = make_float4(beta * (vv[0] - sk.x), beta * (vv[1] - sk.y), beta * (vv[2] - sk.z), beta * (vv[3] - sk.w));
#pragma unroll
    for (int i = 0; i < ROWS; ++i) fma4(S[i], u, k[i]);
    if (warp == 0 && lane < LV) {
      fma4(sqv, u, dot);
      TI* op = reinterpret_cast<TI*>(a.o) + (tok * a.HV + hv) * a.V;
      const float o[4] = {sqv.x, sqv.y, sqv.z, sqv.w};
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (v0 + c < a.V) Act<TI>::store(op + v0 + c, a.scale * o[c]);
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = row0 + i;
    if (r < a.K) store_state<VEC4>(a.final_state + st + (int64_t)r * a.V, v0, a.V, S[i]);
  }
}

template <typename TI, int LV, int WARPS, int ROWS>
void launch(const GdrArgs& a) {
  const dim3 grid(a.n_seqs * a.HV, (a.V + 4 * LV - 1) / (4 * LV));
  const bool vec = a.V % 4 == 0 && a.K % 8 == 0 &&
                   (((uintptr_t)a.initial_state | (uintptr_t)a.final_state | (uintptr_t)a.q | (uintptr_t)a.k) & 15) == 0;
  if (vec) step_kernel<TI, LV, WARPS, ROWS, true><<<grid, WARPS * 32, 0, a.stream>>>(a);
  else step_kernel<TI, LV, WARPS, ROWS, false><<<grid, WARPS * 32, 0, a.stream>>>(a);
}

// W64, W128, W256: warps of a block for K up to 64, 128 and 256
template <typename TI, int LV, int W64, int W128, int W256>
void pick_rows(const GdrArgs& a) {
  constexpr int G = 32 / LV;
  if (a.K <= 64) launch<TI, LV, W64, 64 / (W64 * G)>(a);
  else if (a.K <= 128) launch<TI, LV, W128, 128 / (W128 * G)>(a);
  else launch<TI, LV, W256, 256 / (W256 * G)>(a);
}

template <typename TI>
void pick_columns(const GdrArgs& a) {
  // narrower blocks only while the grid would leave SMs idle (148).  192 blocks of 64 columns (8 requests of 8
  // tokens, K = V = 256): 15.8 us, in 32s 18.7; 32 blocks of 64 (4 requests of 16 tokens, K = V = 128): 15.6 us,
  // in 16s 13.8.
  const int64_t heads = (int64_t)a.n_seqs * a.HV;
  if (a.V > 32 && heads * ((a.V + 63) / 64) >= 148) pick_rows<TI, 16, 2, 4, 4>(a);
  else if (a.V > 16 && heads * ((a.V + 31) / 32) >= 148) pick_rows<TI, 8, 2, 4, 8>(a);
  else pick_rows<TI, 4, 2, 4, 8>(a);
}

}  // namespace

cudaError_t gdr_step(const GdrArgs& a, int* launches) {
  switch (a.dtype) {
    case DT_F32: pick_columns<float>(a); break;
    case DT_BF16: pick_columns<__nv_bfloat16>(a); break;
    default: pick_columns<__half>(a); break;
  }
  ++*launches;
  return cudaGetLastError();
}

}  // namespace ccq
