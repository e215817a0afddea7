// Gated delta rule, exact path: fp32 arithmetic on the CUDA cores, any K <= 256, any V, every type.
// Formulas: gdr.h, written here with beta on the rows: (1 + strict(beta_i L_ij)) U = beta R, so that its T
// is diag(beta) T diag(beta)^{-1} of gdr.h, and dR = T^T dU, dV = beta dR; dbeta_i = dR_i . R_i - sum_j L_ij
// dR_i . U_j.  Chunks of 32 tokens; four kernels over fp32 buffers in the workspace:
//   prep    per (chunk, value head): D, L = strict(D k k^T), T, P and the per-token factors;
//   scan    per (document, value head, 32 columns of V): the state in shared memory, chunk by chunk;
//           for the backward it also keeps S0, U, V - Gam K S0 and dO . O;
//   rscan   the same in reverse for dS: dV, dR, dS1, V . dV and <dS1, S1>;
//   grads   per (chunk, key head): dq, dk (summed over the value heads of the key head), dg, dbeta.
// This path is for fp32 inputs and for sizes the tensor-core path does not take.  What bounds it is
// the scans: one chunk depends on the one before, so a launch with few heads runs at one block's
// latency (about 6 us a chunk at K = 128).
#include "gdr.h"

namespace ccq {
namespace {

constexpr int C = 32;       // tokens per chunk
constexpr int VT = 32;      // columns of V per block of the scans
constexpr int KB = 64;      // columns of K per pass of the gradient kernel
constexpr int THREADS = 256;

// workspace, in floats
struct Ws {
  float *T, *P, *D, *L;   // [slots, HV, C, C]
  float *aux;             // [slots, HV, 3, C]: beta, Gam, w
  float *S0, *dS1;        // [slots, HV, K, V]
  float *U, *R, *dR;      // [slots, HV, C, V]
  float *dotO, *dotV;     // [NVT, slots, HV, C]
  float *tot;             // [NVT, slots, HV]
};

inline int nvt(int V) { return (V + VT - 1) / VT; }

size_t carve(const GdrArgs& a, bool bwd, Ws* w) {
  const size_t sh = (size_t)gdr_slots(a, C) * a.HV;
  size_t off = 0;
  float* base = reinterpret_cast<float*>(a.workspace);
  auto take = [&](size_t n) {
    float* p = base ? base + off : nullptr;
    off += (n + 63) & ~size_t(63);
    return p;
  };
  Ws t;
  t.T = take(sh * C * C);
  t.P = take(sh * C * C);
  t.aux = take(sh * 3 * C);
  t.D = t.L = t.S0 = t.dS1 = t.U = t.R = t.dR = t.dotO = t.dotV = t.tot = nullptr;
  if (bwd) {
    t.D = take(sh * C * C);
    t.L = take(sh * C * C);
    t.S0 = take(sh * a.K * a.V);
    t.dS1 = take(sh * a.K * a.V);
    t.U = take(sh * C * a.V);
    t.R = take(sh * C * a.V);
    t.dR = take(sh * C * a.V);
    t.dotO = take(sh * C * nvt(a.V));
    t.dotV = take(sh * C * nvt(a.V));
    t.tot = take(sh * nvt(a.V));
  }
  if (w) *w = t;
  return off * sizeof(float);
}

__device__ __forceinline__ float dot4(const float4& a, const float4& b, float s) {
  return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, s))));
}

// rows [t0, t0 + C) of a [tokens, heads, W] tensor into dst[C][ld], columns [c0, c0 + n); zero
// outside the document and past W
template <typename TI>
__device__ __forceinline__ void load_rows(float* dst, int ld, int n, const TI* src, const Seq& sq, int t0, int heads,
                                          int head, int W, int c0) {
  for (int i = threadIdx.x; i < C * n; i += blockDim.x) {
    const int r = i / n, c = i - r * n;
    float x = 0.f;
    if (t0 + r < sq.len && c0 + c < W) x = Act<TI>::load(src + ((sq.bos + t0 + r) * heads + head) * W + c0 + c);
    dst[r * ld + c] = x;
  }
}

// ------------------------------------------------------------------------------------------------
template <typename TI>
__global__ void __launch_bounds__(THREADS) prep_kernel(GdrArgs a, Ws w) {
  extern __shared__ float4 smem4[];
  float* sm = reinterpret_cast<float*>(smem4);
  const int Kp = (a.K + 3) & ~3, ld = Kp + 4;
  float* kt = sm;
  float* qt = kt + C * ld;
  __shared__ double G[C];
  __shared__ float beta[C];
  __shared__ float M[C][C + 1], X[C][C + 1];
  const int64_t slot = blockIdx.x;
  const int hv = blockIdx.y, h = hv / (a.HV / a.H);
  int n, c;
  Seq sq;
  if (!gdr_slot_find(a, slot, C, &n, &c, &sq)) return;
  const int t0 = c * C;
  load_rows(kt, ld, Kp, reinterpret_cast<const TI*>(a.k), sq, t0, a.H, h, a.K, 0);
  load_rows(qt, ld, Kp, reinterpret_cast<const TI*>(a.q), sq, t0, a.H, h, a.K, 0);
  const int64_t sh = slot * a.HV + hv;
  if (threadIdx.x < 32) {
    const int t = t0 + threadIdx.x;
    const bool in = t < sq.len;
    const int64_t at = (sq.bos + t) * a.HV + hv;
    // the running sum in 64 bits: differences of large sums stay exact to fp32
    double s = in ? (double)clamp_g(gate_load(a.g, a.g_dtype, at)) : 0.0;
    const float b = in ? gate_load(a.beta, a.beta_dtype, at) : 0.f;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double u = __shfl_up_sync(0xffffffffu, s, o);
      if ((int)threadIdx.x >= o) s += u;
    }
    const double last = __shfl_sync(0xffffffffu, s, 31);
    G[threadIdx.x] = s;
    beta[threadIdx.x] = b;
    float* ax = w.aux + sh * 3 * C;
    ax[threadIdx.x] = b;
    ax[C + threadIdx.x] = expf((float)s);
    ax[2 * C + threadIdx.x] = expf((float)(last - s));
  }
  __syncthreads();
  const int64_t mat = sh * C * C;
  for (int e = threadIdx.x; e < C * C; e += THREADS) {
    const int i = e / C, j = e % C;
    float kk = 0.f, qk = 0.f, d = 0.f;
    if (j <= i) {
      for (int x = 0; x < Kp; x += 4) {
        const float4 kj = *reinterpret_cast<const float4*>(kt + j * ld + x);
        kk = dot4(*reinterpret_cast<const float4*>(kt + i * ld + x), kj, kk);
        qk = dot4(*reinterpret_cast<const float4*>(qt + i * ld + x), kj, qk);
      }
      // rows past the document keep D = 0: a value of another document never enters
      d = t0 + i < sq.len ? expf((float)(G[i] - G[j])) : 0.f;
    }
    const float l = (j < i && d != 0.f) ? kk * d : 0.f;
    M[i][j] = beta[i] * l;
    w.P[mat + e] = d != 0.f ? a.scale * qk * d : 0.f;
    if (w.D) {
      w.D[mat + e] = d;
      w.L[mat + e] = l;
    }
  }
  __syncthreads();
  if (threadIdx.x < C) {  // column j of T = (1 + M)^{-1} by forward substitution
    const int j = threadIdx.x;
    for (int i = 0; i < C; ++i) {
      float s = i == j ? 1.f : 0.f;
      for (int l = j; l < i; ++l) s = fmaf(-M[i][l], X[l][j], s);
      X[i][j] = i < j ? 0.f : s;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < C * C; e += THREADS) w.T[mat + e] = X[e / C][e % C];
}

// ------------------------------------------------------------------------------------------------
// shared memory of the scans: state [Kp][VT], key and query rows [C][ld], T and P [C][C], four
// [C][VT] tiles, factors
inline size_t scan_smem(int K) {
  const int Kp = (K + 3) & ~3, ld = Kp + 4;
  return sizeof(float) * ((size_t)Kp * VT + 2 * C * ld + 2 * C * C + 4 * C * VT + 3 * C);
}

template <typename TI, bool BWD>
__global__ void __launch_bounds__(THREADS) scan_kernel(GdrArgs a, Ws w) {
  extern __shared__ float4 smem4[];
  float* sm = reinterpret_cast<float*>(smem4);
  const int Kp = (a.K + 3) & ~3, ld = Kp + 4;
  float* S = sm;                    // [Kp][VT]
  float* kt = S + Kp * VT;
  float* qt = kt + C * ld;
  float* Tm = qt + C * ld;
  float* Pm = Tm + C * C;
  float* vt = Pm + C * C;           // V, then R
  float* Ut = vt + C * VT;
  float* Uw = Ut + C * VT;
  float* dO = Uw + C * VT;
  float* ax = dO + C * VT;
  const int n = blockIdx.x / a.HV, hv = blockIdx.x % a.HV, h = hv / (a.HV / a.H);
  const int v0 = blockIdx.y * VT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Seq sq = seq_of(n, a.T, a.cu_seqlens);
  const int64_t slot0 = gdr_slot0(a, n, sq, C), slots = gdr_slots(a, C);
  const int64_t st = ((int64_t)n * a.HV + hv) * a.K * a.V;
  const bool vin = v0 + lane < a.V;
  for (int k = warp; k < Kp; k += 8)
    S[k * VT + lane] = (a.initial_state && k < a.K && vin) ? a.initial_state[st + (int64_t)k * a.V + v0 + lane] : 0.f;
  for (int t0 = 0; t0 < sq.len; t0 += C) {
    const int64_t sh = (slot0 + t0 / C) * a.HV + hv;
    __syncthreads();
    load_rows(kt, ld, Kp, reinterpret_cast<const TI*>(a.k), sq, t0, a.H, h, a.K, 0);
    load_rows(qt, ld, Kp, reinterpret_cast<const TI*>(a.q), sq, t0, a.H, h, a.K, 0);
    load_rows(vt, VT, VT, reinterpret_cast<const TI*>(a.v), sq, t0, a.HV, hv, a.V, v0);
    if (BWD) load_rows(dO, VT, VT, reinterpret_cast<const TI*>(a.d_o), sq, t0, a.HV, hv, a.V, v0);
    for (int i = threadIdx.x; i < C * C; i += THREADS) {
      Tm[i] = w.T[sh * C * C + i];
      Pm[i] = w.P[sh * C * C + i];
    }
    if (threadIdx.x < 3 * C) ax[threadIdx.x] = w.aux[sh * 3 * C + threadIdx.x];
    if (BWD && vin)
      for (int k = warp; k < a.K; k += 8) w.S0[(sh * a.K + k) * a.V + v0 + lane] = S[k * VT + lane];
    __syncthreads();
    float x[4] = {}, y[4] = {};  // K S0 and Q S0 of tokens 4 warp .. 4 warp + 3, column lane
    for (int k = 0; k < Kp; k += 4) {
      const float4 s = make_float4(S[k * VT + lane], S[(k + 1) * VT + lane], S[(k + 2) * VT + lane], S[(k + 3) * VT + lane]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = dot4(*reinterpret_cast<const float4*>(kt + (4 * warp + r) * ld + k), s, x[r]);
        y[r] = dot4(*reinterpret_cast<const float4*>(qt + (4 * warp + r) * ld + k), s, y[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 4 * warp + r;
      const float e = t0 + i < sq.len ? vt[i * VT + lane] - ax[C + i] * x[r] : 0.f;
      if (BWD && vin) w.R[(sh * C + i) * a.V + v0 + lane] = e;
      vt[i * VT + lane] = ax[i] * e;
    }
    __syncthreads();
    float u[4] = {};
    for (int j = 0; j < 4 * warp + 4; ++j) {
      const float rj = vt[j * VT + lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) u[r] = fmaf(Tm[(4 * warp + r) * C + j], rj, u[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 4 * warp + r;
      Ut[i * VT + lane] = u[r];
      Uw[i * VT + lane] = ax[2 * C + i] * u[r];
      if (BWD && vin) w.U[(sh * C + i) * a.V + v0 + lane] = u[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] *= a.scale * ax[C + 4 * warp + r];
    for (int j = 0; j < 4 * warp + 4; ++j) {
      const float uj = Ut[j * VT + lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = fmaf(Pm[(4 * warp + r) * C + j], uj, y[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 4 * warp + r;
      if (BWD) {
        const float d = warp_sum(t0 + i < sq.len ? y[r] * dO[i * VT + lane] : 0.f);
        if (lane == 0) w.dotO[((int64_t)blockIdx.y * slots * a.HV + sh) * C + i] = d;
      } else if (vin && t0 + i < sq.len) {
        Act<TI>::store(reinterpret_cast<TI*>(a.o) + ((sq.bos + t0 + i) * a.HV + hv) * a.V + v0 + lane, y[r]);
      }
    }
    const float gam = ax[C + C - 1];
    for (int k = 4 * warp; k < Kp; k += 32) {
      float s[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = gam * S[(k + r) * VT + lane];
      for (int j = 0; j < C; ++j) {
        const float uj = Uw[j * VT + lane];
        const float4 kj = *reinterpret_cast<const float4*>(kt + j * ld + k);
        s[0] = fmaf(kj.x, uj, s[0]);
        s[1] = fmaf(kj.y, uj, s[1]);
        s[2] = fmaf(kj.z, uj, s[2]);
        s[3] = fmaf(kj.w, uj, s[3]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) S[(k + r) * VT + lane] = s[r];
    }
  }
  if (!BWD && a.final_state && vin) {
    __syncthreads();
    for (int k = warp; k < a.K; k += 8) a.final_state[st + (int64_t)k * a.V + v0 + lane] = S[k * VT + lane];
  }
}

// ------------------------------------------------------------------------------------------------
template <typename TI>
__global__ void __launch_bounds__(THREADS) rscan_kernel(GdrArgs a, Ws w) {
  extern __shared__ float4 smem4[];
  float* sm = reinterpret_cast<float*>(smem4);
  const int Kp = (a.K + 3) & ~3, ld = Kp + 4;
  float* S = sm;                    // dS [Kp][VT]
  float* kt = S + Kp * VT;
  float* qt = kt + C * ld;
  float* Tm = qt + C * ld;
  float* Pm = Tm + C * C;
  float* vt = Pm + C * C;
  float* dU = vt + C * VT;
  float* dR = dU + C * VT;          // then beta Gam dR
  float* dO = dR + C * VT;
  float* ax = dO + C * VT;
  __shared__ float red[8];
  const int n = blockIdx.x / a.HV, hv = blockIdx.x % a.HV, h = hv / (a.HV / a.H);
  const int v0 = blockIdx.y * VT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Seq sq = seq_of(n, a.T, a.cu_seqlens);
  const int64_t slot0 = gdr_slot0(a, n, sq, C), slots = gdr_slots(a, C);
  const int64_t st = ((int64_t)n * a.HV + hv) * a.K * a.V;
  const bool vin = v0 + lane < a.V;
  for (int k = warp; k < Kp; k += 8)
    S[k * VT + lane] = (a.dfinal_state && k < a.K && vin) ? a.dfinal_state[st + (int64_t)k * a.V + v0 + lane] : 0.f;
  for (int t0 = (sq.len - 1) / C * C; t0 >= 0 && sq.len > 0; t0 -= C) {
    const int64_t sh = (slot0 + t0 / C) * a.HV + hv;
    __syncthreads();
    load_rows(kt, ld, Kp, reinterpret_cast<const TI*>(a.k), sq, t0, a.H, h, a.K, 0);
    load_rows(qt, ld, Kp, reinterpret_cast<const TI*>(a.q), sq, t0, a.H, h, a.K, 0);
    load_rows(vt, VT, VT, reinterpret_cast<const TI*>(a.v), sq, t0, a.HV, hv, a.V, v0);
    load_rows(dO, VT, VT, reinterpret_cast<const TI*>(a.d_o), sq, t0, a.HV, hv, a.V, v0);
    for (int i = threadIdx.x; i < C * C; i += THREADS) {
      Tm[i] = w.T[sh * C * C + i];
      Pm[i] = w.P[sh * C * C + i];
    }
    if (threadIdx.x < 3 * C) ax[threadIdx.x] = w.aux[sh * 3 * C + threadIdx.x];
    __syncthreads();
    const float gam = ax[C + C - 1];
    // <dS1, S1> = Gam_C <dS1, S0> + sum_j w_j U_j . (K dS1)_j
    float tot = 0.f;
    if (vin)
      for (int k = warp; k < a.K; k += 8) {
        const int64_t at = (sh * a.K + k) * a.V + v0 + lane;
        const float s = S[k * VT + lane];
        w.dS1[at] = s;
        tot = fmaf(gam * s, w.S0[at], tot);
      }
    float y[4] = {};
    for (int k = 0; k < Kp; k += 4) {
      const float4 s = make_float4(S[k * VT + lane], S[(k + 1) * VT + lane], S[(k + 2) * VT + lane], S[(k + 3) * VT + lane]);
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = dot4(*reinterpret_cast<const float4*>(kt + (4 * warp + r) * ld + k), s, y[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = 4 * warp + r;
      y[r] *= ax[2 * C + j];
      if (vin) tot = fmaf(y[r], w.U[(sh * C + j) * a.V + v0 + lane], tot);
    }
    tot = warp_sum(tot);
    if (lane == 0) red[warp] = tot;
    for (int i = 4 * warp; i < C; ++i) {
      const float d = dO[i * VT + lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = fmaf(Pm[i * C + 4 * warp + r], d, y[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) dU[(4 * warp + r) * VT + lane] = y[r];
    __syncthreads();
    if (threadIdx.x == 0) {
      float s = 0.f;
      for (int i = 0; i < 8; ++i) s += red[i];
      w.tot[(int64_t)blockIdx.y * slots * a.HV + sh] = s;
    }
    float x[4] = {};
    for (int i = 4 * warp; i < C; ++i) {
      const float d = dU[i * VT + lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = fmaf(Tm[i * C + 4 * warp + r], d, x[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = 4 * warp + r;
      const bool in = t0 + j < sq.len;
      const float dv = in ? ax[j] * x[r] : 0.f;
      if (vin) w.dR[(sh * C + j) * a.V + v0 + lane] = in ? x[r] : 0.f;
      if (vin && in) Act<TI>::store(reinterpret_cast<TI*>(a.dv) + ((sq.bos + t0 + j) * a.HV + hv) * a.V + v0 + lane, dv);
      const float d = warp_sum(dv * vt[j * VT + lane]);
      if (lane == 0) w.dotV[((int64_t)blockIdx.y * slots * a.HV + sh) * C + j] = d;
      dR[j * VT + lane] = -ax[C + j] * dv;
      dO[j * VT + lane] *= a.scale * ax[C + j];
    }
    __syncthreads();
    for (int k = 4 * warp; k < Kp; k += 32) {
      float s[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = gam * S[(k + r) * VT + lane];
      for (int j = 0; j < C; ++j) {
        const float dr = dR[j * VT + lane], d = dO[j * VT + lane];
        const float4 kj = *reinterpret_cast<const float4*>(kt + j * ld + k);
        const float4 qj = *reinterpret_cast<const float4*>(qt + j * ld + k);
        s[0] = fmaf(kj.x, dr, fmaf(qj.x, d, s[0]));
        s[1] = fmaf(kj.y, dr, fmaf(qj.y, d, s[1]));
        s[2] = fmaf(kj.z, dr, fmaf(qj.z, d, s[2]));
        s[3] = fmaf(kj.w, dr, fmaf(qj.w, d, s[3]));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) S[(k + r) * VT + lane] = s[r];
    }
  }
  if (a.dinitial_state && vin) {
    __syncthreads();
    for (int k = warp; k < a.K; k += 8) a.dinitial_state[st + (int64_t)k * a.V + v0 + lane] = S[k * VT + lane];
  }
}

// ------------------------------------------------------------------------------------------------
constexpr int LV = VT + 4;  // row stride of the [., VT] tiles here: 16-byte rows, no bank conflicts over rows
inline size_t grads_smem(int K) {
  const int Kp = (K + 3) & ~3, ld = Kp + 4;
  return sizeof(float) * ((size_t)2 * C * ld + 2 * KB * LV + 4 * C * LV + 2 * C * (C + 1) + 3 * C);
}

template <typename TI>
__global__ void __launch_bounds__(THREADS) grads_kernel(GdrArgs a, Ws w) {
  extern __shared__ float4 smem4[];
  float* sm = reinterpret_cast<float*>(smem4);
  const int Kp = (a.K + 3) & ~3, ld = Kp + 4;
  float* kt = sm;
  float* qt = kt + C * ld;
  float* S0 = qt + C * ld;          // [KB][LV]
  float* dS = S0 + KB * LV;
  float* Ut = dS + KB * LV;         // [C][LV]
  float* dR = Ut + C * LV;
  float* dO = dR + C * LV;
  float* Rt = dO + C * LV;
  float* W = Rt + C * LV;           // [C][C + 1] scale D dP
  float* N = W + C * (C + 1);       // -beta D (dR U^T)
  float* ax = N + C * (C + 1);      // 3 C
  const int64_t slot = blockIdx.x, slots = gdr_slots(a, C);
  const int h = blockIdx.y, group = a.HV / a.H;
  int n, c;
  Seq sq;
  if (!gdr_slot_find(a, slot, C, &n, &c, &sq)) return;
  const int t0 = c * C;
  load_rows(kt, ld, Kp, reinterpret_cast<const TI*>(a.k), sq, t0, a.H, h, a.K, 0);
  load_rows(qt, ld, Kp, reinterpret_cast<const TI*>(a.q), sq, t0, a.H, h, a.K, 0);
  const int kc = threadIdx.x & 63, ig = threadIdx.x >> 6;           // column of K, tokens 8 ig .. 8 ig + 7
  const int pi = threadIdx.x >> 3, pj = (threadIdx.x & 7) * 4;      // row and 4 columns of the C x C products
  for (int kb = 0; kb < a.K; kb += KB) {
    float aq[8] = {}, ak[8] = {};
    for (int hv = h * group; hv < (h + 1) * group; ++hv) {
      const int64_t sh = slot * a.HV + hv;
      float xq[8] = {}, xr[8] = {}, xu[8] = {}, dp[4] = {}, da[4] = {}, db = 0.f;
      for (int v0 = 0; v0 < a.V; v0 += VT) {
        __syncthreads();
        for (int i = threadIdx.x; i < KB * VT; i += THREADS) {
          const int r = i / VT, v = i % VT;
          const bool in = kb + r < a.K && v0 + v < a.V;
          const int64_t at = (sh * a.K + kb + r) * a.V + v0 + v;
          S0[r * LV + v] = in ? w.S0[at] : 0.f;
          dS[r * LV + v] = in ? w.dS1[at] : 0.f;
        }
        for (int i = threadIdx.x; i < C * VT; i += THREADS) {
          const int r = i / VT, v = i % VT;
          const bool in = v0 + v < a.V;
          const int64_t at = (sh * C + r) * a.V + v0 + v;
          Ut[r * LV + v] = in ? w.U[at] : 0.f;
          dR[r * LV + v] = in ? w.dR[at] : 0.f;
          Rt[r * LV + v] = in ? w.R[at] : 0.f;
          dO[r * LV + v] = in && t0 + r < sq.len
                               ? Act<TI>::load(reinterpret_cast<const TI*>(a.d_o) + ((sq.bos + t0 + r) * a.HV + hv) * a.V + v0 + v)
                               : 0.f;
        }
        __syncthreads();
        for (int v = 0; v < VT; v += 4) {
          const float4 s = *reinterpret_cast<const float4*>(S0 + kc * LV + v);
          const float4 d = *reinterpret_cast<const float4*>(dS + kc * LV + v);
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int i = 8 * ig + r;
            xq[r] = dot4(*reinterpret_cast<const float4*>(dO + i * LV + v), s, xq[r]);
            xr[r] = dot4(*reinterpret_cast<const float4*>(dR + i * LV + v), s, xr[r]);
            xu[r] = dot4(*reinterpret_cast<const float4*>(Ut + i * LV + v), d, xu[r]);
          }
          const float4 o = *reinterpret_cast<const float4*>(dO + pi * LV + v);
          const float4 rr = *reinterpret_cast<const float4*>(dR + pi * LV + v);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 u = *reinterpret_cast<const float4*>(Ut + (pj + j) * LV + v);
            dp[j] = dot4(o, u, dp[j]);
            da[j] = dot4(rr, u, da[j]);
          }
          if (v == pj) db = dot4(rr, *reinterpret_cast<const float4*>(Rt + pi * LV + v), db);
        }
      }
      if (threadIdx.x < 3 * C) ax[threadIdx.x] = w.aux[sh * 3 * C + threadIdx.x];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float d = w.D[sh * C * C + pi * C + pj + j];
        W[pi * (C + 1) + pj + j] = a.scale * d * dp[j];
        N[pi * (C + 1) + pj + j] = pj + j < pi ? -ax[pi] * d * da[j] : 0.f;
        db = fmaf(-w.L[sh * C * C + pi * C + pj + j], da[j], db);
      }
      if (kb == 0) {
        // dbeta: eight threads share a row
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) db += __shfl_xor_sync(0xffffffffu, db, o);
        if (pj == 0 && t0 + pi < sq.len) gate_store(a.dbeta, a.beta_dtype, (sq.bos + t0 + pi) * a.HV + hv, db);
        if (threadIdx.x < C) {  // dg: reverse running sum over the chunk
          const int i = threadIdx.x;
          float s = 0.f, tot = 0.f;
          for (int vt = 0; vt < (a.V + VT - 1) / VT; ++vt) {
            const int64_t p = (int64_t)vt * slots * a.HV + sh;
            s += w.dotO[p * C + i] - w.dotV[p * C + i];
            tot += w.tot[p];
          }
          if (t0 + i >= sq.len) s = 0.f;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const float u = __shfl_down_sync(0xffffffffu, s, o);
            if (i + o < 32) s += u;
          }
          s += tot;
          // nothing decays at the first token of a document that starts from a zero state
          if (t0 + i == 0 && a.initial_state == nullptr) s = 0.f;
          if (t0 + i < sq.len) gate_store(a.dg, a.g_dtype, (sq.bos + t0 + i) * a.HV + hv, s);
        }
      }
      __syncthreads();
      if (kb + kc < a.K) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int i = 8 * ig + r;
          float x = a.scale * ax[C + i] * xq[r];
          float y = fmaf(-ax[i] * ax[C + i], xr[r], ax[2 * C + i] * xu[r]);
          for (int j = 0; j < C; ++j) {
            const float kj = kt[j * ld + kb + kc], qj = qt[j * ld + kb + kc];
            x = fmaf(W[i * (C + 1) + j], kj, x);
            y = fmaf(W[j * (C + 1) + i], qj, y);
            y = fmaf(N[i * (C + 1) + j] + N[j * (C + 1) + i], kj, y);
          }
          aq[r] += x;
          ak[r] += y;
        }
      }
    }
    if (kb + kc < a.K) {
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int i = 8 * ig + r;
        if (t0 + i >= sq.len) continue;
        const int64_t at = ((sq.bos + t0 + i) * a.H + h) * a.K + kb + kc;
        Act<TI>::store(reinterpret_cast<TI*>(a.dq) + at, aq[r]);
        Act<TI>::store(reinterpret_cast<TI*>(a.dk) + at, ak[r]);
      }
    }
  }
}

template <typename F>
cudaError_t allow_smem(F f, size_t bytes) {
  return bytes > 48 * 1024 ? cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) : cudaSuccess;
}

template <typename TI>
cudaError_t run(const GdrArgs& a, bool bwd, int* launches) {
  Ws w;
  carve(a, bwd, &w);
  const int64_t slots = gdr_slots(a, C);
  const dim3 scan_grid(a.n_seqs * a.HV, nvt(a.V));
  const int ld = ((a.K + 3) & ~3) + 4;
  const size_t s1 = sizeof(float) * 2 * C * ld, s2 = scan_smem(a.K), s3 = grads_smem(a.K);
  cudaError_t e = allow_smem(prep_kernel<TI>, s1);
  if (e == cudaSuccess) e = bwd ? allow_smem(scan_kernel<TI, true>, s2) : allow_smem(scan_kernel<TI, false>, s2);
  if (e == cudaSuccess && bwd) e = allow_smem(rscan_kernel<TI>, s2);
  if (e == cudaSuccess && bwd) e = allow_smem(grads_kernel<TI>, s3);
  if (e != cudaSuccess) return e;
  if (a.T > 0) {
    prep_kernel<TI><<<dim3((unsigned)slots, a.HV), THREADS, s1, a.stream>>>(a, w);
    ++*launches;
  }
  if (!bwd) {
    scan_kernel<TI, false><<<scan_grid, THREADS, s2, a.stream>>>(a, w);
    ++*launches;
    return cudaGetLastError();
  }
  if (a.T > 0) {
    scan_kernel<TI, true><<<scan_grid, THREADS, s2, a.stream>>>(a, w);
    ++*launches;
  }
  rscan_kernel<TI><<<scan_grid, THREADS, s2, a.stream>>>(a, w);
  ++*launches;
  if (a.T > 0) {
    grads_kernel<TI><<<dim3((unsigned)slots, a.H), THREADS, s3, a.stream>>>(a, w);
    ++*launches;
  }
  return cudaGetLastError();
}

cudaError_t dispatch(const GdrArgs& a, bool bwd, int* launches) {
  switch (a.dtype) {
    case DT_F32: return run<float>(a, bwd, launches);
    case DT_BF16: return run<__nv_bfloat16>(a, bwd, launches);
    default: return run<__half>(a, bwd, launches);
  }
}

}  // namespace

size_t gdr_simt_workspace(const GdrArgs& a, bool bwd) {
  GdrArgs b = a;
  b.workspace = nullptr;
  return carve(b, bwd, nullptr);
}
cudaError_t gdr_simt_fwd(const GdrArgs& a, int* launches) { return dispatch(a, false, launches); }
cudaError_t gdr_simt_bwd(const GdrArgs& a, int* launches) { return dispatch(a, true, launches); }

}  // namespace ccq
