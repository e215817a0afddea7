// Tensor-core path of the gated delta rule, per (chunk, value head): with G the running sum of g,
//
//   T = (1 + strict(D_ij k_i.k_j beta_j))^{-1}    P beta = scale tril(D_ij q_i.k_j) beta_j    D_ij = e^{G_i - G_j}
//
// as hi + lo pairs of 16-bit matrices in the swizzled layout the scans' MMAs read, and the per-token factors.  The pairs
// are bfloat16 for either type of input; for float16 a second pair of P beta, in that type, goes straight to memory.
//
// One block of four warps per chunk and value head.  The rows come by TMA; k k^T and q k^T (operands the
// inputs themselves, fp32 sums) run on mma.sync, whose fragments are where the elementwise step wants
// them: a block has 2 x 64 x 64 x 128 multiply-adds, too few to pay for a TMEM round trip.  The inverse is
// formed in fp32 accuracy: the four 16 x 16 diagonal blocks by forward substitution, one warp each, then
// T_21 = -T_22 A_21 T_11 for 16- and for 32-row blocks as three-term TF32 products (2^-21).  What bounds the
// kernel is latency, six short stages with barriers between them: 1.65 instructions a cycle with the five blocks
// that fit an SM.  8192 (chunk, head) pairs of K = 128 take 140 us, where their 540 MB alone would take 83.
// (Bands of 16 rows that rotate over the warps, to even out the schedulers: no change.)  float16: 162 us, 16 KB more written.
#include "gdr_tc.cuh"

namespace ccq {
namespace gdrtc {
namespace {
using namespace tc;

constexpr int LDA = 68;  // floats per row: 16-byte rows, fragment loads without bank conflicts

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <int AB16>
__device__ __forceinline__ void mma16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (AB16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x as two TF32 numbers: the upper 11 significant bits and the rest
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xFFFFE000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
// d[NT][4] (16 x 8 NT) += A[16 x 8 KS] B[8 KS x 8 NT], fp32 operands in shared memory, three TF32 terms
template <int KS, int NT>
__device__ __forceinline__ void mm3(float (*d)[4], const float* A, int lda, const float* B, int ldb, int lane) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    uint32_t ah[4], al[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split_tf32(A[(g + 8 * (i & 1)) * lda + 8 * ks + t + 4 * (i >> 1)], ah[i], al[i]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t bh[2], bl[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) split_tf32(B[(8 * ks + t + 4 * i) * ldb + 8 * nt + g], bh[i], bl[i]);
      mma_tf32(d[nt], ah, bl[0], bl[1]);
      mma_tf32(d[nt], al, bh[0], bh[1]);
      mma_tf32(d[nt], ah, bh[0], bh[1]);
    }
  }
}
template <int NT>
__device__ __forceinline__ void put(const float (*d)[4], float sign, float* out, int ld, int lane) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    *reinterpret_cast<float2*>(out + g * ld + 8 * nt + 2 * t) = make_float2(sign * d[nt][0], sign * d[nt][1]);
    *reinterpret_cast<float2*>(out + (g + 8) * ld + 8 * nt + 2 * t) = make_float2(sign * d[nt][2], sign * d[nt][3]);
  }
}

struct Small {
  uint64_t full;
  float gh[C], gl[C], beta[C];  // G log2(e) as hi + lo
  float pb, top[2][4];          // float16: largest |scale D beta| (a bound); largest |k|^2 and |q_x| of each warp
};

// The rows (up to 32 KB) make room, once read, for A and for the images of P; the images of T then replace
// A.  41 KB in all: five blocks on an SM.
constexpr uint32_t OFF_P = (C * LDA * 4 + 1023) & ~1023u;
constexpr uint32_t OFF_X = OFF_P + 2 * PANEL;           // [32][36]
constexpr uint32_t OFF_S = OFF_X + 32 * 36 * 4;
constexpr uint32_t BYTES = OFF_S + sizeof(Small) + 1024;
static_assert(2 * TILE <= OFF_X, "rows fit");

template <int AB16, int KD>
__global__ void __launch_bounds__(128, 5)
    prep_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk, GdrArgs a, Ws w) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* A = reinterpret_cast<float*>(sm);  // [C][LDA]: A, then T
  float* X = reinterpret_cast<float*>(sm + OFF_X);
  Small& S = *reinterpret_cast<Small*>(sm + OFF_S);
  const int64_t slot = blockIdx.x;
  const int hv = blockIdx.y, h = hv / (a.HV / a.H);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int n, c;
  Seq sq;
  if (!gdr_slot_find(a, slot, C, &n, &c, &sq)) return;
  const int t0 = c * C, valid = min(C, sq.len - t0);
  const int64_t sh = slot * a.HV + hv;
  constexpr int NP = KD / 64;
  const uint32_t sk = smem_u32(sm), sq_ = sk + NP * PANEL;
  if (tid == 32) {
    mbar_init(&S.full, 1);
    fence_barrier_init();
    mbar_arrive_expect_tx(&S.full, 2 * NP * PANEL);
    for (int i = 0; i < NP; ++i) {
      tma_load_3d(sm + i * PANEL, &tmk, &S.full, 64 * i, h, (int)(sq.bos + t0));
      tma_load_3d(sm + (NP + i) * PANEL, &tmq, &S.full, 64 * i, h, (int)(sq.bos + t0));
    }
  }
  if (tid < 32) {
    // running sums of g in 64 bits, two tokens a lane, kept as two fp32 parts: their differences, which
    // are all that enters, are then exact to fp32 however large the sums are
    double g[2];
    float b[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = 2 * lane + j;
      const int64_t at = (sq.bos + t0 + t) * a.HV + hv;
      g[j] = t < valid ? (double)clamp_g(gate_load(a.g, a.g_dtype, at)) * 1.4426950408889634 : 0.0;
      b[j] = t < valid ? gate_load(a.beta, a.beta_dtype, at) : 0.f;
    }
    double s = g[0] + g[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    const double last = __shfl_sync(0xffffffffu, s, 31);
    float* ax = w.aux + sh * AX_N;
    const double Gs[2] = {s - g[1], s};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = 2 * lane + j;
      const double x = Gs[j];
      const float gam = ex2((float)x), wt = ex2((float)(last - x));
      S.gh[t] = ax[AX_GH + t] = (float)x;
      S.gl[t] = ax[AX_GL + t] = (float)(x - (double)(float)x);
      S.beta[t] = ax[AX_B + t] = b[j];
      ax[AX_G + t] = gam;
      ax[AX_SG + t] = a.scale * gam;
      ax[AX_WB + t] = wt * b[j];
      ax[AX_W + t] = wt;
    }
    if constexpr (!AB16) {
      const float top = warp_max(fmaxf(ex2((float)Gs[0]), ex2((float)Gs[1])));
      // the largest G_i - G_j, j <= i, from the smallest G of the lanes before
      const float G0 = (float)Gs[0], G1 = (float)Gs[1];
      float low = fminf(G0, G1);
      const float bt = warp_max(fmaxf(fabsf(b[0]), fabsf(b[1])));
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float u = __shfl_up_sync(0xffffffffu, low, o);
        if (lane >= o) low = fminf(low, u);
      }
      low = __shfl_up_sync(0xffffffffu, low, 1);
      low = lane == 0 ? G0 : fminf(low, G0);
      const float rise = warp_max(fmaxf(G0 - low, G1 - fminf(low, G1)));
      if (lane == 0) {
        ax[AX_SM] = fabsf(a.scale) * top;
        S.pb = fabsf(a.scale) * bt * ex2(rise);
      }
    }
    if (lane < (AB16 ? AX_N - AX_GC : 1)) ax[AX_GC + lane] = lane == 0 ? ex2((float)last) : 0.f;
  }
  __syncthreads();
  // the copy's bytes always arrive; the bound only keeps a broken launch from hanging
  if (!mbar_wait(&S.full, 0)) {
    if (tid == 0) atomicOr(w.err, 0x100000);
    return;
  }
  auto top = [&](int x) { return fmaxf(fmaxf(S.top[x][0], S.top[x][1]), fmaxf(S.top[x][2], S.top[x][3])); };
  // rows 16 warp .. +15 of k k^T and q k^T, columns up to the diagonal
  float kk[8][4] = {}, qk[8][4] = {};
  [[maybe_unused]] uint32_t qm[2] = {0, 0};  // float16: largest |q_x| of rows (lane >> 2) and + 8, in pairs
  {
    const uint32_t r = 16 * warp + (lane & 15), ac = lane >> 4;                  // A fragments: row, 16-byte chunk
    const uint32_t br = (lane & 7) + ((lane >> 4) << 3), bc = (lane >> 3) & 1;   // B fragments of two 8-column tiles
#pragma unroll
    for (int ks = 0; ks < KD / 16; ++ks) {
      uint32_t fk[4], fq[4];
      const uint32_t p = (ks >> 2) * PANEL, ch = (ks & 3) * 2;
      ldsm4(fk, sk + p + sw128(r, ch + ac));
      ldsm4(fq, sq_ + p + sw128(r, ch + ac));
      if constexpr (!AB16) {
#pragma unroll
        for (int e = 0; e < 4; ++e) qm[e & 1] = max2_f16(qm[e & 1], fq[e] & 0x7FFF7FFFu);
      }
#pragma unroll
      for (int np = 0; np < 4; ++np) {
        if (np <= warp) {
          uint32_t b[4];
          ldsm4(b, sk + p + sw128(16 * np + br, ch + bc));
          mma16<AB16>(kk[2 * np], fk, b[0], b[1]);
          mma16<AB16>(kk[2 * np + 1], fk, b[2], b[3]);
          mma16<AB16>(qk[2 * np], fq, b[0], b[1]);
          mma16<AB16>(qk[2 * np + 1], fq, b[2], b[3]);
        }
      }
    }
  }
  if constexpr (!AB16) {
    const int i0 = 16 * warp + (lane >> 2);
    float kn = 0.f, qn = 0.f;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + 8 * (e >> 1), j = 8 * nt + 2 * (lane & 3) + (e & 1);
        if (j == i && i < valid) kn = fmaxf(kn, kk[nt][e]);
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float2 x = unpack2<AB16>(qm[e]);
      if (i0 + 8 * e < valid) qn = fmaxf(qn, fmaxf(x.x, x.y));
    }
    kn = warp_max(kn);
    qn = warp_max(qn);
    if (lane == 0) {
      S.top[0][warp] = kn;
      S.top[1][warp] = qn;
    }
  }
  __syncthreads();  // the rows are read: their space becomes A and the images of P
  Pow2 fp{1.f, 1.f};
  if constexpr (!AB16) {
    const float kn = sqrtf(top(0)), qn = top(1) * sqrtf((float)KD);
    fp = pow2_of(S.pb * kn * qn);
    if (tid < 3) w.aux[sh * AX_N + AX_UP + tid] = tid == 0 ? fp.u : tid == 1 ? kn : qn;
  }
  uint8_t* p16 = w.mats + sh * mats_bytes(AB16) + MATS;
  {
    const int i0 = 16 * warp + (lane >> 2);
    const float gh[2] = {S.gh[i0], S.gh[i0 + 8]}, gl[2] = {S.gl[i0], S.gl[i0 + 8]};
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      const int j0 = 8 * nt + 2 * (lane & 3);
      if (nt >= 2 * warp + 2) {  // above the diagonal block
#pragma unroll
        for (int hr = 0; hr < 2; ++hr) {
          const uint32_t at = sw128(i0 + 8 * hr, nt) + (lane & 3) * 4;
          *reinterpret_cast<uint32_t*>(sm + OFF_P + at) = 0;
          *reinterpret_cast<uint32_t*>(sm + OFF_P + PANEL + at) = 0;
          if (!AB16) *reinterpret_cast<uint32_t*>(p16 + at) = *reinterpret_cast<uint32_t*>(p16 + PANEL + at) = 0;
          *reinterpret_cast<float2*>(A + (i0 + 8 * hr) * LDA + j0) = make_float2(0.f, 0.f);
        }
        continue;
      }
      const float2 hj = *reinterpret_cast<const float2*>(S.gh + j0), lj = *reinterpret_cast<const float2*>(S.gl + j0);
      const float2 bj = *reinterpret_cast<const float2*>(S.beta + j0);
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {
        const int i = i0 + 8 * hr;
        const bool in = i < valid;
        const float d0 = ex2((gh[hr] - hj.x) + (gl[hr] - lj.x)) * bj.x, d1 = ex2((gh[hr] - hj.y) + (gl[hr] - lj.y)) * bj.y;
        const float a0 = in && j0 < i ? d0 * kk[nt][2 * hr] : 0.f, a1 = in && j0 + 1 < i ? d1 * kk[nt][2 * hr + 1] : 0.f;
        const float p0 = in && j0 <= i ? a.scale * d0 * qk[nt][2 * hr] : 0.f;
        const float p1 = in && j0 + 1 <= i ? a.scale * d1 * qk[nt][2 * hr + 1] : 0.f;
        *reinterpret_cast<float2*>(A + i * LDA + j0) = make_float2(a0, a1);
        const float p[2] = {p0, p1};
        uint32_t hi, lo;
        split<1, 1>(p, &hi, &lo);
        const uint32_t at = sw128(i, nt) + (lane & 3) * 4;
        *reinterpret_cast<uint32_t*>(sm + OFF_P + at) = hi;
        *reinterpret_cast<uint32_t*>(sm + OFF_P + PANEL + at) = lo;
        if constexpr (!AB16) {
          const float ps[2] = {p0 * fp.s, p1 * fp.s};
          split<0, 1>(ps, &hi, &lo);
          *reinterpret_cast<uint32_t*>(p16 + at) = hi;
          *reinterpret_cast<uint32_t*>(p16 + PANEL + at) = lo;
        }
      }
    }
  }
  __syncwarp();  // a warp's diagonal block is its own
  {  // diagonal block `warp`: column `lane` by forward substitution
    float x[16];
    float* Ab = A + (16 * warp) * LDA + 16 * warp;
    const int col = lane & 15;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s0 = i == col ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
      for (int l = 0; l < (i + 3) / 4; ++l) {
        const float4 r = *reinterpret_cast<const float4*>(Ab + i * LDA + 4 * l);
        s0 = fmaf(-r.x, x[4 * l], s0);
        if (4 * l + 1 < i) s1 = fmaf(-r.y, x[4 * l + 1], s1);
        if (4 * l + 2 < i) s0 = fmaf(-r.z, x[4 * l + 2], s0);
        if (4 * l + 3 < i) s1 = fmaf(-r.w, x[4 * l + 3], s1);
      }
      x[i] = s0 + s1;
    }
    __syncwarp();
    if (lane < 16) {
#pragma unroll
      for (int i = 0; i < 16; ++i) Ab[i * LDA + lane] = x[i];
    }
  }
  __syncthreads();
  {  // rows 16..31 by columns 0..15 (warps 0, 1) and rows 48..63 by 32..47 (warps 2, 3), eight columns a warp
    const int b = warp >> 1, j0 = 8 * (warp & 1);
    float* B21 = A + (32 * b + 16) * LDA + 32 * b;
    float* Xb = X + 16 * b * 36;
    float d[1][4] = {};
    mm3<2, 1>(d, B21, LDA, A + (32 * b) * LDA + 32 * b + j0, LDA, lane);
    put<1>(d, 1.f, Xb + j0, 36, lane);
    __syncthreads();
    float u[1][4] = {};
    mm3<2, 1>(u, B21 + 16, LDA, Xb + j0, 36, lane);
    put<1>(u, -1.f, B21 + j0, LDA, lane);
  }
  __syncthreads();
  {  // rows 32..63 by columns 0..31: a 16 x 16 tile a warp
    const int i0 = 16 * (warp >> 1), j0 = 16 * (warp & 1);
    float* B21 = A + (32 + i0) * LDA;
    float d[2][4] = {};
    mm3<4, 2>(d, B21, LDA, A + j0, LDA, lane);
    put<2>(d, 1.f, X + i0 * 36 + j0, 36, lane);
    __syncthreads();
    float u[2][4] = {};
    mm3<4, 2>(u, B21 + 32, LDA, X + j0, 36, lane);
    put<2>(u, -1.f, B21 + j0, LDA, lane);
  }
  __syncthreads();
  {
    const int i = tid >> 1, half = tid & 1;
    const float* row = A + i * LDA + 32 * half;
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int cc = 0; cc < 4; ++cc) {
      const float4 u = *reinterpret_cast<const float4*>(row + 8 * cc), v = *reinterpret_cast<const float4*>(row + 8 * cc + 4);
      const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
      split<1, 4>(x, hi + 4 * cc, lo + 4 * cc);
    }
    __syncthreads();
#pragma unroll
    for (int cc = 0; cc < 4; ++cc) {
      const uint32_t at = sw128(i, 4 * half + cc);
      *reinterpret_cast<uint4*>(sm + at) = make_uint4(hi[4 * cc], hi[4 * cc + 1], hi[4 * cc + 2], hi[4 * cc + 3]);
      *reinterpret_cast<uint4*>(sm + PANEL + at) = make_uint4(lo[4 * cc], lo[4 * cc + 1], lo[4 * cc + 2], lo[4 * cc + 3]);
    }
  }
  fence_async_smem();
  __syncthreads();
  if (tid == 0) {
    uint8_t* dst = w.mats + sh * mats_bytes(AB16);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst + i * 2 * PANEL),
                   "r"(sk + i * OFF_P), "r"(2 * PANEL)
                   : "memory");
    bulk_commit();
    bulk_wait_read();  // shared memory must outlive the copy's reads; the writes end with the kernel
  }
}

template <int AB16, int KD>
cudaError_t launch(const GdrArgs& a, const Ws& w) {
  CUtensorMap q, k;
  cudaError_t e = token_map(&q, a, a.q, a.H, a.K);
  if (e == cudaSuccess) e = token_map(&k, a, a.k, a.H, a.K);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(prep_kernel<AB16, KD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)BYTES);
  if (e != cudaSuccess) return e;
  prep_kernel<AB16, KD><<<dim3((unsigned)gdr_slots(a, C), a.HV), 128, BYTES, a.stream>>>(q, k, a, w);
  return cudaGetLastError();
}

}  // namespace

cudaError_t prep(const GdrArgs& a, const Ws& w, int* launches) {
  ++*launches;
  const bool small = a.K <= 64;
  if (a.dtype == DT_BF16) return small ? launch<1, 64>(a, w) : launch<1, 128>(a, w);
  return small ? launch<0, 64>(a, w) : launch<0, 128>(a, w);
}

}  // namespace gdrtc
}  // namespace ccq
