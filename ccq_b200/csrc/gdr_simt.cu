// Gated delta rule, exact path: fp32 arithmetic on the CUDA cores, any K <= 256, any V, every type.
// Formulas: gdr.h, written here with beta on the rows: (1 + strict(beta_i L_ij)) U = beta R, so that its T
// is diag(beta) T diag(beta)^{-1} of gdr.h, and dR = T^T dU, dV = beta dR; dbeta_i = dR_i . R_i - sum_j L_ij
// dR_i . U_j.  Chunks of 32 tokens; four kernels over fp32 buffers in the workspace:
//   prep    per (chunk, value head): D, L = strict(D k k^T), T, P and the per-token factors;
//   scan    per (document, value head, VT columns of V): the state in shared memory, chunk by chunk;
//           for the backward it also keeps S0, U, V - Gam K S0 and dO . O;
//   rscan   the same in reverse for dS: dV, dR, dS1, V . dV and <dS1, S1>;
//   grads   per (chunk, key head): dq, dk (summed over the value heads of the key head), dg, dbeta.
// This path is for fp32 inputs and for sizes the tensor-core path does not take.  What bounds it is
// the scans: one chunk depends on the one before, so a launch with few heads runs at one block's
// latency.  VT is then 8 (see tile()): four times the blocks, one token and column a thread in place
// of four, and the next chunk's rows loaded beside this one's products.
#include "gdr.h"

namespace ccq {
namespace {

constexpr int C = 32;       // tokens per chunk
constexpr int VG = 32;      // columns of V per pass of the gradient kernel
constexpr int LT = C + 4;   // row stride of a C x C matrix in shared memory
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
  int nvt;                // NVT
};

// Columns of V per block of the scans: 32, or 8 where that leaves half of the SMs without a block.  Forward and
// backward of 1024 tokens in fp32, 64 blocks of 32: 0.67 ms in eights, 0.92 in 32s at K = V = 64, 0.92 and
// 1.24 at 128, 1.98 and 2.04 at 256; 128 blocks of 32: 1.25 and 1.04, 1.72 and 1.40, 3.87 and 2.39.
inline int tile(const GdrArgs& a) { return 2 * (int64_t)a.n_seqs * a.HV * ((a.V + 31) / 32) <= 148 ? 8 : 32; }
inline int nvt(const GdrArgs& a) { return (a.V + tile(a) - 1) / tile(a); }

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
  t.nvt = nvt(a);
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
    t.dotO = take(sh * C * nvt(a));
    t.dotV = take(sh * C * nvt(a));
    t.tot = take(sh * nvt(a));
  }
  if (w) *w = t;
  return off * sizeof(float);
}

__device__ __forceinline__ float dot4(const float4& a, const float4& b, float s) {
  return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, s))));
}

__device__ __forceinline__ void copy4(float* dst, const float* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(in ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void copy16(float* dst, const float* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <typename TI>
__device__ __forceinline__ void fetch1(float* dst, const TI* src, bool in) {
  if constexpr (sizeof(TI) == 4)
    copy4(dst, src, in);
  else
    *dst = in ? Act<TI>::load(src) : 0.f;
}
// rows [t0, t0 + C) of a [tokens, heads, W] tensor into dst[C][ld], n columns; zero outside the document and
// past W.  A warp a row; for fp32 the copies are asynchronous.
template <typename TI>
__device__ __forceinline__ void fetch_rows(float* dst, int ld, int n, const TI* src, const Seq& sq, int t0, int heads, int head,
                                           int W) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int r = threadIdx.x >> 5; r < C; r += THREADS / 32) {
    const bool row = t0 + r < sq.len;
    const TI* p = src + (row ? ((sq.bos + t0 + r) * heads + head) * W : 0);
    for (int c = lane; c < n; c += 32) fetch1(dst + r * ld + c, p + (c < W ? c : 0), row && c < W);
  }
}
// and VT columns of V from c0
template <typename TI, int VT>
__device__ __forceinline__ void fetch_tile(float* dst, const TI* src, const Seq& sq, int t0, int heads, int head, int W, int c0) {
#pragma unroll
  for (int i = threadIdx.x; i < C * VT; i += THREADS) {
    const int r = i / VT, c = c0 + i % VT;
    const bool in = t0 + r < sq.len && c < W;
    fetch1(dst + i, src + (in ? ((sq.bos + t0 + r) * heads + head) * W + c : 0), in);
  }
}
__device__ __forceinline__ void fetch_mat(float* dst, const float* src) {
  copy16(dst + (threadIdx.x >> 3) * LT + (threadIdx.x & 7) * 4, src + threadIdx.x * 4);
}
static_assert(C * C == THREADS * 4, "a matrix is one 16-byte copy a thread");

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
  __shared__ float X[C][C + 1];
  __shared__ __align__(16) float M[C][LT];
  const int64_t slot = blockIdx.x;
  const int hv = blockIdx.y, h = hv / (a.HV / a.H);
  int n, c;
  Seq sq;
  if (!gdr_slot_find(a, slot, C, &n, &c, &sq)) return;
  const int t0 = c * C;
  fetch_rows(kt, ld, Kp, reinterpret_cast<const TI*>(a.k), sq, t0, a.H, h, a.K);
  fetch_rows(qt, ld, Kp, reinterpret_cast<const TI*>(a.q), sq, t0, a.H, h, a.K);
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
  copies_wait();
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
  if (threadIdx.x < C) {  // column j of T = (1 + M)^{-1} by forward substitution, in registers
    const int j = threadIdx.x;
    float x[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float p[4] = {i == j ? 1.f : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int l = 0; l < i; ++l) p[l & 3] = fmaf(-M[i][l], x[l], p[l & 3]);
      x[i] = i < j ? 0.f : (p[0] + p[1]) + (p[2] + p[3]);
      X[i][j] = x[i];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < C * C; e += THREADS) w.T[mat + e] = X[e / C][e % C];
}

// ------------------------------------------------------------------------------------------------
// The scans: a thread has column `col` of its block's VT and the tokens R g .. R g + R - 1.  Shared memory: the
// state [VT][ld], one or two sets of a chunk's inputs, three [C][VT] tiles.
template <int VT>
struct Scan {
  static constexpr int NG = THREADS / VT, R = C / NG, SETS = VT < 32 ? 2 : 1;
  static __host__ __device__ int set(int ld) { return 2 * C * ld + 2 * C * LT + 2 * C * VT + 3 * C; }
  static size_t smem(int K) {
    const int ld = ((K + 3) & ~3) + 4;
    return sizeof(float) * ((size_t)VT * ld + SETS * set(ld) + 3 * C * VT);
  }
};
struct Chunk {
  float *kt, *qt, *Tm, *Pm, *vt, *dO, *ax;
};
template <int VT>
__device__ __forceinline__ Chunk chunk_at(float* p, int ld) {
  Chunk b;
  b.kt = p;
  b.qt = b.kt + C * ld;
  b.Tm = b.qt + C * ld;
  b.Pm = b.Tm + C * LT;
  b.vt = b.Pm + C * LT;
  b.dO = b.vt + C * VT;
  b.ax = b.dO + C * VT;
  return b;
}
template <typename TI, int VT, bool DO>
__device__ __forceinline__ void fetch(const Chunk& b, const GdrArgs& a, const Ws& w, const Seq& sq, int t0, int64_t sh, int h, int hv,
                                      int v0, int ld) {
  fetch_rows(b.kt, ld, ld - 4, reinterpret_cast<const TI*>(a.k), sq, t0, a.H, h, a.K);
  fetch_rows(b.qt, ld, ld - 4, reinterpret_cast<const TI*>(a.q), sq, t0, a.H, h, a.K);
  fetch_tile<TI, VT>(b.vt, reinterpret_cast<const TI*>(a.v), sq, t0, a.HV, hv, a.V, v0);
  if (DO) fetch_tile<TI, VT>(b.dO, reinterpret_cast<const TI*>(a.d_o), sq, t0, a.HV, hv, a.V, v0);
  fetch_mat(b.Tm, w.T + sh * C * C);
  fetch_mat(b.Pm, w.P + sh * C * C);
  if (threadIdx.x < 3 * C) copy4(b.ax + threadIdx.x, w.aux + sh * 3 * C + threadIdx.x, true);
}
// sum over the VT columns
template <int VT>
__device__ __forceinline__ float col_sum(float x) {
#pragma unroll
  for (int o = VT / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <typename TI, bool BWD, int VT>
__global__ void __launch_bounds__(THREADS) scan_kernel(GdrArgs a, Ws w) {
  using L = Scan<VT>;
  constexpr int R = L::R, NG = L::NG;
  extern __shared__ float4 smem4[];
  float* S = reinterpret_cast<float*>(smem4);  // [VT][ld]
  const int Kp = (a.K + 3) & ~3, ld = Kp + 4;
  float* sets = S + VT * ld;
  float* Rt = sets + L::SETS * L::set(ld);  // [C][VT]
  float* Ut = Rt + C * VT;
  float* Uw = Ut + C * VT;
  const int n = blockIdx.x / a.HV, hv = blockIdx.x % a.HV, h = hv / (a.HV / a.H);
  const int v0 = blockIdx.y * VT;
  const int col = threadIdx.x % VT, g = threadIdx.x / VT;
  const int jm = 4 * (threadIdx.x >> 5) + 4;  // past the last token of this warp
  const Seq sq = seq_of(n, a.T, a.cu_seqlens);
  const int64_t slot0 = gdr_slot0(a, n, sq, C), slots = gdr_slots(a, C);
  const int64_t st = ((int64_t)n * a.HV + hv) * a.K * a.V;
  const bool vin = v0 + col < a.V;
  for (int k = g; k < Kp; k += NG)
    S[col * ld + k] = (a.initial_state && k < a.K && vin) ? a.initial_state[st + (int64_t)k * a.V + v0 + col] : 0.f;
  if (L::SETS == 2 && sq.len > 0) fetch<TI, VT, BWD>(chunk_at<VT>(sets, ld), a, w, sq, 0, slot0 * a.HV + hv, h, hv, v0, ld);
  for (int t0 = 0; t0 < sq.len; t0 += C) {
    const int64_t sh = (slot0 + t0 / C) * a.HV + hv;
    const Chunk b = chunk_at<VT>(sets + (L::SETS == 2 ? (t0 / C & 1) * L::set(ld) : 0), ld);
    if (L::SETS == 1) {
      __syncthreads();
      fetch<TI, VT, BWD>(b, a, w, sq, t0, sh, h, hv, v0, ld);
    }
    copies_wait();
    __syncthreads();
    if (L::SETS == 2 && t0 + C < sq.len)
      fetch<TI, VT, BWD>(chunk_at<VT>(sets + (t0 / C + 1 & 1) * L::set(ld), ld), a, w, sq, t0 + C, sh + a.HV, h, hv, v0, ld);
    if (BWD && vin)
      for (int k = 4 * g; k < a.K; k += 4 * NG) {
        const float4 s = *reinterpret_cast<const float4*>(S + col * ld + k);
        float* p = w.S0 + (sh * a.K + k) * a.V + v0 + col;
        p[0] = s.x;
        if (k + 1 < a.K) p[a.V] = s.y;
        if (k + 2 < a.K) p[2 * a.V] = s.z;
        if (k + 3 < a.K) p[3 * a.V] = s.w;
      }
    float x[R] = {}, y[R] = {};  // K S0 and Q S0
#pragma unroll 4
    for (int k = 0; k < Kp; k += 4) {
      const float4 s = *reinterpret_cast<const float4*>(S + col * ld + k);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        x[r] = dot4(*reinterpret_cast<const float4*>(b.kt + (R * g + r) * ld + k), s, x[r]);
        y[r] = dot4(*reinterpret_cast<const float4*>(b.qt + (R * g + r) * ld + k), s, y[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = R * g + r;
      const float e = t0 + i < sq.len ? b.vt[i * VT + col] - b.ax[C + i] * x[r] : 0.f;
      if (BWD && vin) w.R[(sh * C + i) * a.V + v0 + col] = e;
      Rt[i * VT + col] = b.ax[i] * e;
    }
    __syncthreads();
    float u[R] = {};
#pragma unroll 2
    for (int j = 0; j < jm; j += 4) {
      const float r0 = Rt[j * VT + col], r1 = Rt[(j + 1) * VT + col], r2 = Rt[(j + 2) * VT + col], r3 = Rt[(j + 3) * VT + col];
#pragma unroll
      for (int r = 0; r < R; ++r)
        u[r] = dot4(*reinterpret_cast<const float4*>(b.Tm + (R * g + r) * LT + j), make_float4(r0, r1, r2, r3), u[r]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = R * g + r;
      Ut[i * VT + col] = u[r];
      Uw[i * VT + col] = b.ax[2 * C + i] * u[r];
      if (BWD && vin) w.U[(sh * C + i) * a.V + v0 + col] = u[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) y[r] *= a.scale * b.ax[C + R * g + r];
#pragma unroll 2
    for (int j = 0; j < jm; j += 4) {
      const float u0 = Ut[j * VT + col], u1 = Ut[(j + 1) * VT + col], u2 = Ut[(j + 2) * VT + col], u3 = Ut[(j + 3) * VT + col];
#pragma unroll
      for (int r = 0; r < R; ++r)
        y[r] = dot4(*reinterpret_cast<const float4*>(b.Pm + (R * g + r) * LT + j), make_float4(u0, u1, u2, u3), y[r]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = R * g + r;
      if (BWD) {
        const float d = col_sum<VT>(t0 + i < sq.len ? y[r] * b.dO[i * VT + col] : 0.f);
        if (col == 0) w.dotO[((int64_t)blockIdx.y * slots * a.HV + sh) * C + i] = d;
      } else if (vin && t0 + i < sq.len) {
        Act<TI>::store(reinterpret_cast<TI*>(a.o) + ((sq.bos + t0 + i) * a.HV + hv) * a.V + v0 + col, y[r]);
      }
    }
    const float gam = b.ax[C + C - 1];
    for (int k = 4 * g; k < Kp; k += 4 * NG) {
      float4 s = *reinterpret_cast<const float4*>(S + col * ld + k);
      s = make_float4(gam * s.x, gam * s.y, gam * s.z, gam * s.w);
#pragma unroll 8
      for (int j = 0; j < C; ++j) {
        const float uj = Uw[j * VT + col];
        const float4 kj = *reinterpret_cast<const float4*>(b.kt + j * ld + k);
        s.x = fmaf(kj.x, uj, s.x);
        s.y = fmaf(kj.y, uj, s.y);
        s.z = fmaf(kj.z, uj, s.z);
        s.w = fmaf(kj.w, uj, s.w);
      }
      *reinterpret_cast<float4*>(S + col * ld + k) = s;
    }
  }
  if (!BWD && a.final_state && vin) {
    __syncthreads();
    for (int k = g; k < a.K; k += NG) a.final_state[st + (int64_t)k * a.V + v0 + col] = S[col * ld + k];
  }
}

// ------------------------------------------------------------------------------------------------
template <typename TI, int VT>
__global__ void __launch_bounds__(THREADS) rscan_kernel(GdrArgs a, Ws w) {
  using L = Scan<VT>;
  constexpr int R = L::R, NG = L::NG;
  extern __shared__ float4 smem4[];
  float* S = reinterpret_cast<float*>(smem4);  // dS [VT][ld]
  const int Kp = (a.K + 3) & ~3, ld = Kp + 4;
  float* sets = S + VT * ld;
  float* dU = sets + L::SETS * L::set(ld);  // [C][VT]
  float* dR = dU + C * VT;                  // -Gam dV
  float* dQ = dR + C * VT;                  // scale Gam dO
  __shared__ float red[8];
  const int n = blockIdx.x / a.HV, hv = blockIdx.x % a.HV, h = hv / (a.HV / a.H);
  const int v0 = blockIdx.y * VT;
  const int col = threadIdx.x % VT, g = threadIdx.x / VT, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j0 = 4 * warp;  // first token of this warp
  const Seq sq = seq_of(n, a.T, a.cu_seqlens);
  const int64_t slot0 = gdr_slot0(a, n, sq, C), slots = gdr_slots(a, C);
  const int64_t st = ((int64_t)n * a.HV + hv) * a.K * a.V;
  const bool vin = v0 + col < a.V;
  for (int k = g; k < Kp; k += NG)
    S[col * ld + k] = (a.dfinal_state && k < a.K && vin) ? a.dfinal_state[st + (int64_t)k * a.V + v0 + col] : 0.f;
  const int nch = (sq.len + C - 1) / C;
  // the sum over the warps of the chunk before, between two barriers of this one
  auto put_tot = [&](int64_t sh) {
    if (threadIdx.x == 0) {
      float s = 0.f;
      for (int i = 0; i < 8; ++i) s += red[i];
      w.tot[(int64_t)blockIdx.y * slots * a.HV + sh] = s;
    }
  };
  if (L::SETS == 2 && nch > 0)
    fetch<TI, VT, true>(chunk_at<VT>(sets + (nch - 1 & 1) * L::set(ld), ld), a, w, sq, (nch - 1) * C, (slot0 + nch - 1) * a.HV + hv, h, hv,
                        v0, ld);
  for (int c = nch - 1; c >= 0; --c) {
    const int t0 = c * C;
    const int64_t sh = (slot0 + c) * a.HV + hv;
    const Chunk b = chunk_at<VT>(sets + (L::SETS == 2 ? (c & 1) * L::set(ld) : 0), ld);
    if (L::SETS == 1) {
      __syncthreads();
      fetch<TI, VT, true>(b, a, w, sq, t0, sh, h, hv, v0, ld);
    }
    float us[R];
#pragma unroll
    for (int r = 0; r < R; ++r) us[r] = vin ? w.U[(sh * C + R * g + r) * a.V + v0 + col] : 0.f;
    copies_wait();
    __syncthreads();
    if (c + 1 < nch) put_tot(sh + a.HV);
    if (L::SETS == 2 && c > 0)
      fetch<TI, VT, true>(chunk_at<VT>(sets + (c - 1 & 1) * L::set(ld), ld), a, w, sq, t0 - C, sh - a.HV, h, hv, v0, ld);
    const float gam = b.ax[C + C - 1];
    float y[R] = {};
#pragma unroll 4
    for (int k = 0; k < Kp; k += 4) {
      const float4 s = *reinterpret_cast<const float4*>(S + col * ld + k);
#pragma unroll
      for (int r = 0; r < R; ++r) y[r] = dot4(*reinterpret_cast<const float4*>(b.kt + (R * g + r) * ld + k), s, y[r]);
    }
    // <dS1, S1> = Gam_C <dS1, S0> + sum_j w_j U_j . (K dS1)_j
    float tot = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      y[r] *= b.ax[2 * C + R * g + r];
      if (vin) tot = fmaf(y[r], us[r], tot);
    }
#pragma unroll 4
    for (int i = j0; i < C; ++i) {
      const float d = b.dO[i * VT + col];
#pragma unroll
      for (int r = 0; r < R; ++r) y[r] = fmaf(b.Pm[i * LT + R * g + r], d, y[r]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) dU[(R * g + r) * VT + col] = y[r];
    __syncthreads();
    float x[R] = {};
#pragma unroll 4
    for (int i = j0; i < C; ++i) {
      const float d = dU[i * VT + col];
#pragma unroll
      for (int r = 0; r < R; ++r) x[r] = fmaf(b.Tm[i * LT + R * g + r], d, x[r]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = R * g + r;
      const bool in = t0 + j < sq.len;
      const float dv = in ? b.ax[j] * x[r] : 0.f;
      if (vin) w.dR[(sh * C + j) * a.V + v0 + col] = in ? x[r] : 0.f;
      if (vin && in) Act<TI>::store(reinterpret_cast<TI*>(a.dv) + ((sq.bos + t0 + j) * a.HV + hv) * a.V + v0 + col, dv);
      const float d = col_sum<VT>(dv * b.vt[j * VT + col]);
      if (col == 0) w.dotV[((int64_t)blockIdx.y * slots * a.HV + sh) * C + j] = d;
      dR[j * VT + col] = -b.ax[C + j] * dv;
      dQ[j * VT + col] = a.scale * b.ax[C + j] * b.dO[j * VT + col];
    }
    __syncthreads();
    for (int k = 4 * g; k < Kp; k += 4 * NG) {
      float4 s = *reinterpret_cast<const float4*>(S + col * ld + k);
      const float old[4] = {s.x, s.y, s.z, s.w};
      float s0[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t at = (sh * a.K + k + r) * a.V + v0 + col;
        const bool in = vin && k + r < a.K;
        s0[r] = in ? w.S0[at] : 0.f;
        if (in) w.dS1[at] = old[r];
      }
      s = make_float4(gam * s.x, gam * s.y, gam * s.z, gam * s.w);
#pragma unroll 8
      for (int j = 0; j < C; ++j) {
        const float dr = dR[j * VT + col], d = dQ[j * VT + col];
        const float4 kj = *reinterpret_cast<const float4*>(b.kt + j * ld + k);
        const float4 qj = *reinterpret_cast<const float4*>(b.qt + j * ld + k);
        s.x = fmaf(kj.x, dr, fmaf(qj.x, d, s.x));
        s.y = fmaf(kj.y, dr, fmaf(qj.y, d, s.y));
        s.z = fmaf(kj.z, dr, fmaf(qj.z, d, s.z));
        s.w = fmaf(kj.w, dr, fmaf(qj.w, d, s.w));
      }
      *reinterpret_cast<float4*>(S + col * ld + k) = s;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (vin && k + r < a.K) tot = fmaf(gam * old[r], s0[r], tot);
    }
    tot = warp_sum(tot);
    if (lane == 0) red[warp] = tot;
  }
  __syncthreads();
  if (nch > 0) put_tot(slot0 * a.HV + hv);
  if (a.dinitial_state && vin)
    for (int k = g; k < a.K; k += NG) a.dinitial_state[st + (int64_t)k * a.V + v0 + col] = S[col * ld + k];
}

// ------------------------------------------------------------------------------------------------
constexpr int LV = VG + 4;  // row stride of the [., VG] tiles here: 16-byte rows, no bank conflicts over rows
inline size_t grads_smem(int K) {
  const int Kp = (K + 3) & ~3, ld = Kp + 4;
  return sizeof(float) * ((size_t)2 * C * ld + 2 * KB * LV + 4 * C * LV + 3 * C * LT + 3 * C);
}

template <typename TI>
__global__ void __launch_bounds__(THREADS, 2) grads_kernel(GdrArgs a, Ws w) {
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
  float* W = Rt + C * LV;           // [C][LT] scale D dP
  float* Wt = W + C * LT;           // its transpose
  float* N = Wt + C * LT;           // Z + Z^T, Z = -beta D (dR U^T) below the diagonal
  float* ax = N + C * LT;           // 3 C
  const int64_t slot = blockIdx.x, slots = gdr_slots(a, C);
  const int h = blockIdx.y, group = a.HV / a.H;
  int n, c;
  Seq sq;
  if (!gdr_slot_find(a, slot, C, &n, &c, &sq)) return;
  const int t0 = c * C;
  fetch_rows(kt, ld, Kp, reinterpret_cast<const TI*>(a.k), sq, t0, a.H, h, a.K);
  fetch_rows(qt, ld, Kp, reinterpret_cast<const TI*>(a.q), sq, t0, a.H, h, a.K);
  const int kc = threadIdx.x & 63, ig = threadIdx.x >> 6;           // column of K, tokens 8 ig .. 8 ig + 7
  const int pi = threadIdx.x >> 3, pj = threadIdx.x & 7;            // row and columns pj + 8 j of the C x C products
  for (int kb = 0; kb < a.K; kb += KB) {
    float aq[8] = {}, ak[8] = {};
    for (int hv = h * group; hv < (h + 1) * group; ++hv) {
      const int64_t sh = slot * a.HV + hv;
      float xq[8] = {}, xr[8] = {}, xu[8] = {}, dp[4] = {}, da[4] = {}, db = 0.f;
      for (int v0 = 0; v0 < a.V; v0 += VG) {
        __syncthreads();
        {
          const int v = threadIdx.x % VG;
          const bool vin = v0 + v < a.V;
          const int64_t at = v0 + (vin ? v : 0);
#pragma unroll
          for (int r = threadIdx.x / VG; r < KB; r += THREADS / VG) {
            const bool in = vin && kb + r < a.K;
            const int64_t p = (sh * a.K + (in ? kb + r : 0)) * a.V + at;
            copy4(S0 + r * LV + v, w.S0 + p, in);
            copy4(dS + r * LV + v, w.dS1 + p, in);
          }
#pragma unroll
          for (int r = threadIdx.x / VG; r < C; r += THREADS / VG) {
            const int64_t p = (sh * C + r) * a.V + at;
            copy4(Ut + r * LV + v, w.U + p, vin);
            copy4(dR + r * LV + v, w.dR + p, vin);
            copy4(Rt + r * LV + v, w.R + p, vin);
            const bool in = vin && t0 + r < sq.len;
            fetch1(dO + r * LV + v, reinterpret_cast<const TI*>(a.d_o) + (in ? ((sq.bos + t0 + r) * a.HV + hv) * a.V + at : 0), in);
          }
        }
        copies_wait();
        __syncthreads();
        for (int v = 0; v < VG; v += 4) {
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
            const float4 u = *reinterpret_cast<const float4*>(Ut + (pj + 8 * j) * LV + v);
            dp[j] = dot4(o, u, dp[j]);
            da[j] = dot4(rr, u, da[j]);
          }
          if (v == 4 * pj) db = dot4(rr, *reinterpret_cast<const float4*>(Rt + pi * LV + v), db);
        }
      }
      if (threadIdx.x < 3 * C) ax[threadIdx.x] = w.aux[sh * 3 * C + threadIdx.x];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int cj = pj + 8 * j;
        const float d = w.D[sh * C * C + pi * C + cj];
        const float wij = a.scale * d * dp[j], z = -ax[pi] * d * da[j];
        W[pi * LT + cj] = Wt[cj * LT + pi] = wij;
        if (cj < pi) N[pi * LT + cj] = N[cj * LT + pi] = z;
        if (cj == pi) N[pi * LT + pi] = 0.f;
        db = fmaf(-w.L[sh * C * C + pi * C + cj], da[j], db);
      }
      if (kb == 0) {
        // dbeta: eight threads share a row
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) db += __shfl_xor_sync(0xffffffffu, db, o);
        if (pj == 0 && t0 + pi < sq.len) gate_store(a.dbeta, a.beta_dtype, (sq.bos + t0 + pi) * a.HV + hv, db);
        if (threadIdx.x < C) {  // dg: reverse running sum over the chunk
          const int i = threadIdx.x;
          float s = 0.f, tot = 0.f;
          for (int vt = 0; vt < w.nvt; ++vt) {
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
          aq[r] = fmaf(a.scale * ax[C + i], xq[r], aq[r]);
          ak[r] += fmaf(-ax[i] * ax[C + i], xr[r], ax[2 * C + i] * xu[r]);
        }
        for (int j = 0; j < C; j += 4) {
          const float* kp = kt + j * ld + kb + kc;
          const float* qp = qt + j * ld + kb + kc;
          const float4 kj = make_float4(kp[0], kp[ld], kp[2 * ld], kp[3 * ld]);
          const float4 qj = make_float4(qp[0], qp[ld], qp[2 * ld], qp[3 * ld]);
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int at = (8 * ig + r) * LT + j;
            aq[r] = dot4(*reinterpret_cast<const float4*>(W + at), kj, aq[r]);
            ak[r] = dot4(*reinterpret_cast<const float4*>(Wt + at), qj, ak[r]);
            ak[r] = dot4(*reinterpret_cast<const float4*>(N + at), kj, ak[r]);
          }
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
  // 48 KB without asking, the static arrays (up to 10 KB) counted in
  return bytes > 38 * 1024 ? cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) : cudaSuccess;
}

template <typename TI, int VT>
cudaError_t run_tiled(const GdrArgs& a, const Ws& w, bool bwd, int* launches) {
  const int64_t slots = gdr_slots(a, C);
  const dim3 scan_grid(a.n_seqs * a.HV, (a.V + VT - 1) / VT);
  const int ld = ((a.K + 3) & ~3) + 4;
  const size_t s1 = sizeof(float) * 2 * C * ld, s2 = Scan<VT>::smem(a.K), s3 = grads_smem(a.K);
  cudaError_t e = allow_smem(prep_kernel<TI>, s1);
  if (e == cudaSuccess) e = bwd ? allow_smem(scan_kernel<TI, true, VT>, s2) : allow_smem(scan_kernel<TI, false, VT>, s2);
  if (e == cudaSuccess && bwd) e = allow_smem(rscan_kernel<TI, VT>, s2);
  if (e == cudaSuccess && bwd) e = allow_smem(grads_kernel<TI>, s3);
  if (e != cudaSuccess) return e;
  if (a.T > 0) {
    prep_kernel<TI><<<dim3((unsigned)slots, a.HV), THREADS, s1, a.stream>>>(a, w);
    ++*launches;
  }
  if (!bwd) {
    scan_kernel<TI, false, VT><<<scan_grid, THREADS, s2, a.stream>>>(a, w);
    ++*launches;
    return cudaGetLastError();
  }
  if (a.T > 0) {
    scan_kernel<TI, true, VT><<<scan_grid, THREADS, s2, a.stream>>>(a, w);
    ++*launches;
  }
  rscan_kernel<TI, VT><<<scan_grid, THREADS, s2, a.stream>>>(a, w);
  ++*launches;
  if (a.T > 0) {
    grads_kernel<TI><<<dim3((unsigned)slots, a.H), THREADS, s3, a.stream>>>(a, w);
    ++*launches;
  }
  return cudaGetLastError();
}

template <typename TI>
cudaError_t run(const GdrArgs& a, bool bwd, int* launches) {
  Ws w;
  carve(a, bwd, &w);
  return tile(a) == 8 ? run_tiled<TI, 8>(a, w, bwd, launches) : run_tiled<TI, 32>(a, w, bwd, launches);
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
