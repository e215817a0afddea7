// Tensor-core path of the gated delta rule, gradients inside a chunk, per (chunk, key head):
//
//   dQ = scale Gam dO S0^T + W K                       W_ij = scale D_ij beta_j (dO E^T)_ij, j <= i
//   dK = -Gam dV S0^T + w beta E dS1^T + W^T Q + (N + N^T) K    N_ij = -D_ij beta_j (dV E^T)_ij, j < i
//   dbeta_j = sum_i scale D_ij (q_i.k_j) (dO E^T)_ij + w_j k_j.(E dS1^T)_j - sum_i D_ij (k_i.k_j) (dV E^T)_ij
//   dg_t = sum_{i >= t} (dO_i . O_i - V_i . dV_i) + <dS, S>, over the tokens up to the next anchor and there
//
// summed over the value heads of the key head in registers.  The chunks are independent: persistent
// blocks of 16 warps walk (chunk, key head) items; each item runs over (value head, 64 columns of V)
// steps whose tiles are loaded by TMA two steps ahead, across items.  A warp holds a 16 x 32 tile of the
// 64 x 128 products and a 16 x 16 tile of the 64 x 64 ones, on mma.sync: an item reads 144 KB for 29 MFLOP, so
// HBM and mma.sync are about equally near; five products with 64-row operands would leave half of
// each tcgen05 tile empty.  Operands are single 16-bit values: what is formed here is rounded to 16 bits next.
#include "gdr_tc.cuh"

namespace ccq {
namespace gdrtc {
namespace {
using namespace tc;

constexpr int THREADS = 512;
constexpr uint32_t B_S = 0, B_DS = 2 * PANEL, B_DO = 4 * PANEL, B_E = 5 * PANEL, B_DV = 6 * PANEL, B_SIZE = 7 * PANEL;  // one step
constexpr uint32_t L_QK = 0;                       // two buffers of Q (2 panels) and K (2 panels)
constexpr uint32_t L_B = 8 * PANEL;                // two steps
constexpr uint32_t L_W = L_B + 2 * B_SIZE, L_N = L_W + PANEL;
constexpr uint32_t L_AX = L_N + PANEL;             // two
constexpr uint32_t AX_BYTES = (AX_N * 4 + 127) & ~127u;

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
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

// A [16 x 16] fragments of a row-major panel tile (rows r0.., 16-byte chunks c0, c0 + 1)
__device__ __forceinline__ uint32_t a_addr(uint32_t panel, int r0, int c0, int lane) {
  return panel + sw128(r0 + (lane & 15), c0 + (lane >> 4));
}
// the same of the transposed matrix: A[m][k] = P[k][m], rows k0.. of the panel, columns m from chunk c0
__device__ __forceinline__ uint32_t at_addr(uint32_t panel, int k0, int c0, int lane) {
  return panel + sw128(k0 + (lane & 7) + ((lane >> 4) << 3), c0 + ((lane >> 3) & 1));
}
// B fragments of two 8-column tiles, B[k][n] = P[n][k]: rows n0.., k from chunk c0 (non-transposed load)
__device__ __forceinline__ uint32_t b_addr(uint32_t panel, int n0, int c0, int lane) {
  return panel + sw128(n0 + (lane & 7) + ((lane >> 4) << 3), c0 + ((lane >> 3) & 1));
}
// B[k][n] = P[k][n]: rows k0.., n from chunk c0 (transposed load)
__device__ __forceinline__ uint32_t bt_addr(uint32_t panel, int k0, int c0, int lane) {
  return panel + sw128(k0 + (lane & 15), c0 + (lane >> 4));
}

// One step as the block's warps see it, written by thread 0 two steps ahead.
struct Step {
  int live, hv, h, row0, valid, first_v, last_v, first, last, qk, ax, more, zero_first;
  int64_t sh, anchor;
};

__device__ __forceinline__ int nvt128(const GdrArgs& a) { return (a.V + VT - 1) / VT; }

// The position of the next step to load (thread 0's; in shared memory to spare the others its registers).
struct Walk {
  int item, items, count, n, c, g, vt, loaded;  // item = slot * H + key head
  Seq sq;
  bool live;
  __device__ __forceinline__ void find(const GdrArgs& a) {
    for (; item < items; item += gridDim.x)
      if (gdr_slot_find(a, item / a.H, C, &n, &c, &sq)) {
        live = true;
        g = vt = 0;
        return;
      }
    live = false;
  }
  __device__ __forceinline__ void next(const GdrArgs& a, int group, int nvt) {
    if (++vt < nvt) return;
    vt = 0;
    if (++g < group) return;
    item += gridDim.x;
    ++count;
    find(a);
  }
};

struct Small {
  uint64_t full[2];
  Step step[2];
  Walk walk;
  float ke[4][C], db[4][C], dg[17];
  int abort;
};
constexpr uint32_t L_SMALL = L_AX + 2 * AX_BYTES;
constexpr uint32_t BYTES = L_SMALL + sizeof(Small) + 1024;
static_assert(BYTES <= 232448, "shared memory");

// ONE: a key head serves one value head, so nothing is carried from one value head to the next
template <int AB16, int KD, bool ONE>
__global__ void __launch_bounds__(THREADS, 1)
    grads_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                 const __grid_constant__ CUtensorMap tmo, const __grid_constant__ CUtensorMap tmdv,
                 const __grid_constant__ CUtensorMap tme, const __grid_constant__ CUtensorMap tms,
                 const __grid_constant__ CUtensorMap tmds, const __grid_constant__ CUtensorMap tmdq,
                 const __grid_constant__ CUtensorMap tmdk, GdrArgs a, Ws w) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Small& S_ = *reinterpret_cast<Small*>(sm + L_SMALL);
  const uint32_t sb = smem_u32(sm);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int mt = warp >> 2, nq = warp & 3;  // rows 16 mt.., columns KD / 4 nq.. of K (16 nq.. of the 64 x 64 products)
  const int g = lane >> 2, tq = lane & 3;
  constexpr int NP = KD / 64, NT = KD / 32;  // panels of K; 8-column tiles of K a warp holds
  const int group = a.HV / a.H, nvt = (a.V + 63) / 64;
  if (tid == 0) {
    mbar_init(&S_.full[0], 1);
    mbar_init(&S_.full[1], 1);
    S_.abort = 0;
    fence_barrier_init();
  }
  __syncthreads();
  Walk& pf = S_.walk;
  // thread 0: describes and loads the next step
  auto load = [&]() {
    const int b = pf.loaded & 1;
    Step& s = S_.step[b];
    s.live = pf.live;
    if (!pf.live) return;
    {
      uint64_t* bar = &S_.full[b];
      uint8_t* p = sm + L_B + b * B_SIZE;
      const int slot = pf.item / a.H, h = pf.item - slot * a.H, hv = h * group + pf.g;
      const int64_t sh = (int64_t)slot * a.HV + hv;
      const int row = (int)(pf.sq.bos + (int64_t)pf.c * C);
      const int nch = (pf.sq.len + C - 1) / C;
      s.hv = hv;
      s.h = h;
      s.row0 = row;
      s.valid = min(C, pf.sq.len - pf.c * C);
      s.first_v = pf.vt == 0;
      s.last_v = pf.vt == nvt - 1;
      s.first = s.first_v && pf.g == 0;
      s.last = s.last_v && pf.g == group - 1;
      s.qk = pf.count & 1;
      s.ax = (pf.count * group + pf.g) & 1;
      s.more = min(ANCHOR - 1 - pf.c % ANCHOR, nch - 1 - pf.c);
      s.zero_first = pf.c == 0 && a.initial_state == nullptr;
      s.sh = sh;
      s.anchor = (gdr_slot0(a, pf.n, pf.sq, C * ANCHOR) + pf.c / ANCHOR) * a.HV + hv;
      mbar_arrive_expect_tx(bar, 2 * NP * PANEL + 3 * PANEL + (s.first_v ? AX_N * 4 : 0) + (s.first ? 2 * NP * PANEL : 0));
      if (s.first) {
        uint8_t* d = sm + L_QK + s.qk * 4 * PANEL;
        for (int i = 0; i < NP; ++i) {
          tma_load_3d(d + i * PANEL, &tmq, bar, 64 * i, h, row);
          tma_load_3d(d + (2 + i) * PANEL, &tmk, bar, 64 * i, h, row);
        }
      }
      if (s.first_v) bulk_load(sm + L_AX + s.ax * AX_BYTES, w.aux + sh * AX_N, AX_N * 4, bar);
      tma_load_3d(p + B_DO, &tmo, bar, 64 * pf.vt, hv, row);
      tma_load_3d(p + B_DV, &tmdv, bar, 64 * pf.vt, hv, row);
      tma_load_3d(p + B_E, &tme, bar, 0, 64 * pf.vt, (int)sh);
      for (int i = 0; i < NP; ++i) {
        tma_load_3d(p + B_S + i * PANEL, &tms, bar, 64 * i, 64 * pf.vt, (int)sh);
        tma_load_3d(p + B_DS + i * PANEL, &tmds, bar, 64 * i, 64 * pf.vt, (int)sh);
      }
    }
    ++pf.loaded;
    pf.next(a, group, nvt);
  };
  if (tid == 0) {
    pf.loaded = 0;
    pf.items = (int)(gdr_slots(a, C) * a.H);
    pf.item = blockIdx.x;
    pf.count = 0;
    pf.find(a);
    load();
    load();
  }
  __syncthreads();
  float dq[NT][4], dk[NT][4];  // ONE: dO S0^T and dV S0^T grow into them
  float xq[NT][4], xv[NT][4], xe[NT][4], pe[2][4], ve[2][4];  // dO S0^T, dV S0^T, E dS1^T, dO E^T, dV E^T
  float dot = 0.f, later = 0.f;
  for (int step = 0;; ++step) {
    const int b = step & 1;
    const Step& s = S_.step[b];
    if (!s.live) break;
    // what is read after the step's last barrier, when thread 0 may already describe the step after the next
    const int valid = s.valid, row0 = s.row0, head = s.h;
    const bool last = s.last;
    const uint32_t p = sb + L_B + b * B_SIZE;
    const uint32_t Q = sb + L_QK + s.qk * 4 * PANEL, K = Q + 2 * PANEL;
    const float* ax = reinterpret_cast<const float*>(sm + L_AX + s.ax * AX_BYTES);
    if (s.first_v) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          xq[i][j] = xv[i][j] = xe[i][j] = 0.f;
          if (!ONE && s.first) dq[i][j] = dk[i][j] = 0.f;
        }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) pe[i][j] = ve[i][j] = 0.f;
      // dO . O - V . dV: of this chunk's tokens in warps 0 and 1, of the chunks up to the next anchor in the
      // others; and <dS, S> there
      dot = later = 0.f;
      const int64_t vs = gdr_slots(a, C) * a.HV, va = gdr_slots(a, C * ANCHOR) * a.HV;
      for (int v = 0; v < nvt128(a); ++v) {
        if ((tid >> 6) <= s.more) {
          const int64_t at = (v * vs + s.sh + (int64_t)(tid >> 6) * a.HV) * C + (tid & 63);
          dot += w.dotO[at] - w.dotV[at];
        }
        if (tid < CHAIN_WARPS) later += w.anchor[(v * va + s.anchor) * CHAIN_WARPS + tid];
      }
    }
    pipe_wait(&S_.full[b], (step >> 1) & 1, &S_.abort, w.err, 0x200000);
    if (valid < C && s.first) {
      // the rows past the document belong to another one: what a product sums over must be zero
      for (int i = 0; i < NP; ++i) {
        zero_rows(Q + i * PANEL, 1, valid, tid, THREADS);
        zero_rows(K + i * PANEL, 1, valid, tid, THREADS);
      }
      __syncthreads();
    }
#pragma unroll 1
    for (int ks = 0; ks < 4; ++ks) {
      uint32_t fo[4], fv[4], fe[4], be[4];
      ldsm4(fo, a_addr(p + B_DO, 16 * mt, 2 * ks, lane));
      ldsm4(fv, a_addr(p + B_DV, 16 * mt, 2 * ks, lane));
      ldsm4t(fe, at_addr(p + B_E, 16 * ks, 2 * mt, lane));
      ldsm4t(be, bt_addr(p + B_E, 16 * ks, 2 * nq, lane));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mma16<AB16>(pe[j], fo, be[2 * j], be[2 * j + 1]);
        mma16<AB16>(ve[j], fv, be[2 * j], be[2 * j + 1]);
      }
#pragma unroll
      for (int j = 0; j < NT / 2; ++j) {
        const int col = (KD / 4) * nq + 16 * j;
        uint32_t bs[4], bd[4];
        ldsm4t(bs, bt_addr(p + B_S + (col >> 6) * PANEL, 16 * ks, (col & 63) >> 3, lane));
        ldsm4t(bd, bt_addr(p + B_DS + (col >> 6) * PANEL, 16 * ks, (col & 63) >> 3, lane));
        mma16<AB16>(xq[2 * j], fo, bs[0], bs[1]);
        mma16<AB16>(xq[2 * j + 1], fo, bs[2], bs[3]);
        mma16<AB16>(xv[2 * j], fv, bs[0], bs[1]);
        mma16<AB16>(xv[2 * j + 1], fv, bs[2], bs[3]);
        mma16<AB16>(xe[2 * j], fe, bd[0], bd[1]);
        mma16<AB16>(xe[2 * j + 1], fe, bd[2], bd[3]);
      }
    }
    if (s.last_v) {
      // q k^T and k k^T of this warp's 16 x 16 tile, where it reaches the lower triangle
      float qk[2][4] = {}, kk[2][4] = {};
      if (nq <= mt) {
#pragma unroll 1
        for (int ks = 0; ks < KD / 16; ++ks) {
          uint32_t fq[4], fk[4], bk[4];
          const uint32_t pan = (ks >> 2) * PANEL;
          ldsm4(fq, a_addr(Q + pan, 16 * mt, 2 * (ks & 3), lane));
          ldsm4(fk, a_addr(K + pan, 16 * mt, 2 * (ks & 3), lane));
          ldsm4(bk, b_addr(K + pan, 16 * nq, 2 * (ks & 3), lane));
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            mma16<AB16>(qk[j], fq, bk[2 * j], bk[2 * j + 1]);
            mma16<AB16>(kk[j], fk, bk[2 * j], bk[2 * j + 1]);
          }
        }
      }
      const int i0 = 16 * mt + g;
      const float gh[2] = {ax[AX_GH + i0], ax[AX_GH + i0 + 8]}, gl[2] = {ax[AX_GL + i0], ax[AX_GL + i0 + 8]};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int j0 = 16 * nq + 8 * j + 2 * tq;
        float db[2] = {0.f, 0.f};
#pragma unroll
        for (int hr = 0; hr < 2; ++hr) {
          const int i = i0 + 8 * hr;
          float W[2], N[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int jj = j0 + e;
            const bool on = jj <= i && i < valid;
            const float d = on ? exp2f((gh[hr] - ax[AX_GH + jj]) + (gl[hr] - ax[AX_GL + jj])) : 0.f;
            const float x = on ? d * pe[j][2 * hr + e] : 0.f, y = on && jj < i ? d * ve[j][2 * hr + e] : 0.f;
            const float be = ax[AX_B + jj];
            W[e] = a.scale * be * x;
            N[e] = -be * y;
            db[e] += a.scale * x * qk[j][2 * hr + e] - y * kk[j][2 * hr + e];
          }
          const uint32_t at = sw128(i, 2 * nq + j) + tq * 4;
          *reinterpret_cast<uint32_t*>(sm + L_W + at) = pack2<AB16>(W[0], W[1]);
          *reinterpret_cast<uint32_t*>(sm + L_N + at) = pack2<AB16>(N[0], N[1]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) db[e] += __shfl_xor_sync(0xffffffffu, db[e], o);
          if (g == 0) S_.db[mt][j0 + e] = db[e];
        }
      }
      // the state's part of dq and dk, and k_j . (E dS1^T)_j
      float ke[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int col = (KD / 4) * nq + 8 * j;
#pragma unroll
        for (int hr = 0; hr < 2; ++hr) {
          const int i = i0 + 8 * hr;
          const float2 kf = unpack2<AB16>(*reinterpret_cast<const uint32_t*>(
              sm + (K - sb) + (col >> 6) * PANEL + sw128(i, (col & 63) >> 3) + tq * 4));
          ke[hr] = fmaf(kf.x, xe[j][2 * hr], fmaf(kf.y, xe[j][2 * hr + 1], ke[hr]));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = ax[AX_SG + i] * xq[j][2 * hr + e];
            const float y = ax[AX_WB + i] * xe[j][2 * hr + e] - ax[AX_G + i] * xv[j][2 * hr + e];
            dq[j][2 * hr + e] = ONE ? x : dq[j][2 * hr + e] + x;
            dk[j][2 * hr + e] = ONE ? y : dk[j][2 * hr + e] + y;
          }
        }
      }
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {
        ke[hr] += __shfl_xor_sync(0xffffffffu, ke[hr], 1);
        ke[hr] += __shfl_xor_sync(0xffffffffu, ke[hr], 2);
        if (tq == 0) S_.ke[nq][i0 + 8 * hr] = ke[hr];
      }
      {
        const float r = warp_sum(warp < 2 ? later : dot + later);
        if (lane == 0) S_.dg[warp] = r;
      }
      __syncthreads();
      // W K, W^T Q, N K, N^T K
#pragma unroll 1
      for (int ks = 0; ks < 4; ++ks) {
        uint32_t fw[4], fwt[4], fn[4], fnt[4];
        ldsm4(fw, a_addr(sb + L_W, 16 * mt, 2 * ks, lane));
        ldsm4t(fwt, at_addr(sb + L_W, 16 * ks, 2 * mt, lane));
        ldsm4(fn, a_addr(sb + L_N, 16 * mt, 2 * ks, lane));
        ldsm4t(fnt, at_addr(sb + L_N, 16 * ks, 2 * mt, lane));
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) {
          const int col = (KD / 4) * nq + 16 * j;
          uint32_t bk[4], bq[4];
          ldsm4t(bk, bt_addr(K + (col >> 6) * PANEL, 16 * ks, (col & 63) >> 3, lane));
          ldsm4t(bq, bt_addr(Q + (col >> 6) * PANEL, 16 * ks, (col & 63) >> 3, lane));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mma16<AB16>(dq[2 * j + e], fw, bk[2 * e], bk[2 * e + 1]);
            mma16<AB16>(dk[2 * j + e], fwt, bq[2 * e], bq[2 * e + 1]);
            mma16<AB16>(dk[2 * j + e], fn, bk[2 * e], bk[2 * e + 1]);
            mma16<AB16>(dk[2 * j + e], fnt, bk[2 * e], bk[2 * e + 1]);
          }
        }
      }
      if (warp < 2) {
        const int j = tid;
        const float ke4 = S_.ke[0][j] + S_.ke[1][j] + S_.ke[2][j] + S_.ke[3][j];
        if (j < valid)
          gate_store(a.dbeta, a.beta_dtype, (int64_t)(s.row0 + j) * a.HV + s.hv,
                     S_.db[0][j] + S_.db[1][j] + S_.db[2][j] + S_.db[3][j] + ax[AX_W + j] * ke4);
        // dg: reverse running sum; warp 1 holds tokens 32..63, whose sum warp 0 adds
        float r = dot;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float u = __shfl_down_sync(0xffffffffu, r, o);
          if (lane + o < 32) r += u;
        }
        if (lane == 0 && warp == 1) S_.dg[16] = r;
        bar_sync<2, 64>();
        float rest = S_.dg[lane & 15];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
        r += rest + (warp == 0 ? S_.dg[16] : 0.f);
        // nothing decays at the first token of a document that starts from a zero state
        if (j == 0 && s.zero_first) r = 0.f;
        if (j < valid) gate_store(a.dg, a.g_dtype, (int64_t)(s.row0 + j) * a.HV + s.hv, r);
      }
    }
    __syncthreads();  // the step's tiles, W, N and, after the last step, Q and K have been read
    if (last) {
      // dq over Q and dk over K, then out
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int col = (KD / 4) * nq + 8 * j;
#pragma unroll
        for (int hr = 0; hr < 2; ++hr) {
          const uint32_t at = (col >> 6) * PANEL + sw128(16 * mt + g + 8 * hr, (col & 63) >> 3) + tq * 4;
          *reinterpret_cast<uint32_t*>(sm + (Q - sb) + at) = pack2<AB16>(dq[j][2 * hr], dq[j][2 * hr + 1]);
          *reinterpret_cast<uint32_t*>(sm + (K - sb) + at) = pack2<AB16>(dk[j][2 * hr], dk[j][2 * hr + 1]);
        }
      }
      fence_async_smem();
      __syncthreads();
      if (valid == C) {
        if (tid == 0) {
          for (int i = 0; i < NP; ++i)
            if (64 * i < a.K) {
              tma_store_3d(&tmdq, sm + (Q - sb) + i * PANEL, 64 * i, head, row0);
              tma_store_3d(&tmdk, sm + (K - sb) + i * PANEL, 64 * i, head, row0);
            }
          bulk_commit();
          bulk_wait_read();
        }
      } else {
        copy_rows(Q, reinterpret_cast<uint16_t*>(a.dq), row0, a.H, head, a.K, 0, valid, tid, THREADS);
        copy_rows(K, reinterpret_cast<uint16_t*>(a.dk), row0, a.H, head, a.K, 0, valid, tid, THREADS);
        __syncthreads();
      }
    }
    // the step is done: its description and buffers go to the one after the next.  A last step's dq and dk
    // have left Q and K (thread 0 waited); the barrier at the end of the next step publishes the description.
    if (tid == 0) load();
  }
  if (tid == 0) bulk_wait_all();
}

template <int AB16, int KD, bool ONE>
cudaError_t launch(const GdrArgs& a, const Ws& w) {
  const int64_t slots = gdr_slots(a, C), sh = slots * a.HV;
  CUtensorMap q, k, o, dv, e, s, ds, dq, dk;
  cudaError_t r = token_map(&q, a, a.q, a.H, a.K);
  if (r == cudaSuccess) r = token_map(&k, a, a.k, a.H, a.K);
  if (r == cudaSuccess) r = token_map(&o, a, a.d_o, a.HV, a.V);
  if (r == cudaSuccess) r = token_map(&dv, a, a.dv, a.HV, a.V);
  if (r == cudaSuccess) r = matrix_map(&e, a, w.E, C, sh);
  if (r == cudaSuccess) r = matrix_map(&s, a, w.S0, a.K, sh);
  if (r == cudaSuccess) r = matrix_map(&ds, a, w.dS1, a.K, sh);
  if (r == cudaSuccess) r = token_map(&dq, a, a.dq, a.H, a.K);
  if (r == cudaSuccess) r = token_map(&dk, a, a.dk, a.H, a.K);
  if (r == cudaSuccess) r = cudaFuncSetAttribute(grads_kernel<AB16, KD, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)BYTES);
  if (r != cudaSuccess) return r;
  const int64_t items = slots * a.H;
  const unsigned grid = (unsigned)(items < 148 ? items : 148);  // one persistent block per SM
  grads_kernel<AB16, KD, ONE><<<grid, THREADS, BYTES, a.stream>>>(q, k, o, dv, e, s, ds, dq, dk, a, w);
  return cudaGetLastError();
}

template <int AB16>
cudaError_t pick(const GdrArgs& a, const Ws& w) {
  const bool one = a.H == a.HV;
  if (a.K <= 64) return one ? launch<AB16, 64, true>(a, w) : launch<AB16, 64, false>(a, w);
  return one ? launch<AB16, 128, true>(a, w) : launch<AB16, 128, false>(a, w);
}

}  // namespace

cudaError_t grads(const GdrArgs& a, const Ws& w, int* launches) {
  ++*launches;
  return a.dtype == DT_BF16 ? pick<1>(a, w) : pick<0>(a, w);
}

}  // namespace gdrtc
}  // namespace ccq
