// Gated delta rule: argument bundle and the pieces its kernels share.
//
//   S <- e^{g_t} S;  u_t = beta_t (v_t - S^T k_t);  S <- S + k_t u_t^T;  o_t = scale S^T q_t
//
// per (document, value head), S [K, V] fp32.  A key head serves HV / H value heads.  In chunks of C
// tokens (rows of Q, K, V), with G the running sum of g inside the chunk, Gam = e^G, w = e^{G_C - G},
// D_ij = e^{G_i - G_j} (j <= i) and S0 the state before the chunk:
//
//   R = V - Gam K S0      T = (1 + strict(D_ij k_i.k_j beta_j))^{-1}       E = T R      U = beta E
//   O = scale Gam Q S0 + P U     P = scale tril(D_ij q_i.k_j)                S1 = Gam_C S0 + K^T (w U)
//
// (E, the part of V that the state does not hold yet, rather than U: beta then multiplies and never
// divides, so that beta = 0 needs no case of its own.)  Backwards, from dO and dS1, with L = strict(D k k^T):
//
//   dE = beta (P^T dO + w K dS1)      dV = T^T dE
//   dS0 = Gam_C dS1 + (scale Gam Q)^T dO - (Gam K)^T dV
//   dQ = scale Gam dO S0^T + W K,                 W = scale tril(D dO U^T)
//   dK = -Gam dV S0^T + W^T Q + (N + N^T) K + w U dS1^T,   N_ij = -D_ij dV_i.U_j  (j < i)
//   dbeta_j = sum_i P_ij dO_i.E_j + w_j k_j.(dS1 E_j) - sum_i L_ij dV_i.E_j
//   dg_t = <dS1, S1> + sum_{i >= t} (dO_i . O_i - V_i . dV_i)      (i inside the chunk)
//
// The last line is what collecting every e^G gives: the terms with q sum to dO . O, and those with k, the
// scores and R to -V . dV.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "args.h"
#ifdef __CUDACC__
#include "common.cuh"
#endif

namespace ccq {

struct GdrArgs {
  int dtype, B, T, H, HV, K, V, n_seqs;
  const void* q;     // [B, T, H, K]
  const void* k;     // [B, T, H, K]
  const void* v;     // [B, T, HV, V]
  int g_dtype, beta_dtype;
  const void* g;     // [B, T, HV] log decay
  const void* beta;  // [B, T, HV]
  float scale;
  const int64_t* cu_seqlens;
  const float* initial_state;  // [n_seqs, HV, K, V] or nullptr
  void* o;                     // [B, T, HV, V]
  float* final_state;          // [n_seqs, HV, K, V] or nullptr
  // backward
  const void* d_o;
  const float* dfinal_state;  // or nullptr
  void* dq;
  void* dk;
  void* dv;
  void* dg;             // g's type
  void* dbeta;          // beta's type
  float* dinitial_state;  // or nullptr
  const void* fwd_workspace;  // of the forward on the same inputs, or nullptr (tensor-core path only)
  void* workspace;
  size_t workspace_bytes;
  cudaStream_t stream;
};

// Both paths read their workspaces in 16-byte pieces: the entry points refuse one that is not on such a boundary.
// Exact path: fp32 arithmetic on the CUDA cores, any K <= 256 and any V, fp32 / bf16 / fp16.
size_t gdr_simt_workspace(const GdrArgs& a, bool bwd);
cudaError_t gdr_simt_fwd(const GdrArgs& a, int* launches);
cudaError_t gdr_simt_bwd(const GdrArgs& a, int* launches);

// Tensor-core path (gdr_tc*.cu): 16-bit inputs, K a multiple of 8 up to 128, V a multiple of 8,
// 16-byte aligned tensors but for o.  Word 0 of the workspace receives the device error code.
bool gdr_tc_supported(const GdrArgs& a);
size_t gdr_tc_workspace(const GdrArgs& a, bool bwd);
cudaError_t gdr_tc_fwd(const GdrArgs& a, int* launches);
cudaError_t gdr_tc_bwd(const GdrArgs& a, int* launches);

// Token by token over a cache (any T, meant for a few tokens): state_in may equal state_out.
cudaError_t gdr_step(const GdrArgs& a, int* launches);

#ifdef __CUDACC__
__device__ __forceinline__ float gate_load(const void* p, int dt, int64_t i) {
  if (dt == DT_F32) return reinterpret_cast<const float*>(p)[i];
  if (dt == DT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void gate_store(void* p, int dt, int64_t i, float x) {
  if (dt == DT_F32) reinterpret_cast<float*>(p)[i] = x;
  else if (dt == DT_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(x);
}
// A decay below e^-1000 is zero in every type here; the bound keeps sums of g finite when a
// caller resets the state with g = -inf (a NaN stays one).
__device__ __forceinline__ float clamp_g(float g) { return g < -1000.f ? -1000.f : g; }

// Chunk slots.  Dense: n * ceil(T / C) + c.  Varlen: floor(bos / C) + n + c (see chunk_slot0).
__host__ __device__ inline int64_t gdr_slots(const GdrArgs& a, int C) {
  return a.cu_seqlens ? chunk_slots_total(a.T, a.n_seqs, C) : (int64_t)a.n_seqs * ((a.T + C - 1) / C);
}
__device__ __forceinline__ int64_t gdr_slot0(const GdrArgs& a, int n, const Seq& sq, int C) {
  return a.cu_seqlens ? chunk_slot0(n, sq.bos, C) : (int64_t)n * ((a.T + C - 1) / C);
}
// The document and chunk of a slot; false where the slot holds no chunk.
__device__ __forceinline__ bool gdr_slot_find(const GdrArgs& a, int64_t slot, int C, int* n_out, int* c_out, Seq* sq_out) {
  int n;
  if (a.cu_seqlens == nullptr) {
    n = (int)(slot / ((a.T + C - 1) / C));
  } else {
    int lo = 0, hi = a.n_seqs - 1;  // last n whose first slot is <= slot (first slots increase with n)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      const Seq s = seq_of(mid, a.T, a.cu_seqlens);
      if (chunk_slot0(mid, s.bos, C) <= slot) lo = mid; else hi = mid - 1;
    }
    n = lo;
  }
  const Seq sq = seq_of(n, a.T, a.cu_seqlens);
  const int64_t c = slot - gdr_slot0(a, n, sq, C);
  *n_out = n;
  *c_out = (int)c;
  *sq_out = sq;
  return c >= 0 && c * C < sq.len;
}
#endif

}  // namespace ccq
