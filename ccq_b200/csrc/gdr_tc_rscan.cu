// Tensor-core path of the gated delta rule, reverse scan: one block per (document, value head, 128
// columns of V) walks the document backwards in chunks of 64 tokens with dS, the gradient of the state
// after the chunk.  Transposed as in the scan, one column of V per TMEM lane:
//
//   Z^T  = dO^T (P beta)        [128 x 64]   A: the dO tile, read MN-major, B: P beta hi, lo, read MN-major
//   Y^T  = dS^T K^T             [128 x 64]   A: dS hi + lo (TMEM), B: the K rows
//   dE^T = Z^T + w beta Y^T                  (chain warps; split to hi + lo, back to TMEM)
//   dV^T = dE^T T               [128 x 128]  A: dE hi, B: [T hi | T lo]; and dE lo with T hi
//   D^T  = (scale Gam dO)^T Q   [128 x K]    A: hi + lo (output warps, beside the chain), B: Q, MN-major
//        + (-Gam dV)^T K                     A: hi + lo (chain warps), B: the K rows, MN-major
//   dS^T = Gam_C dS^T + D^T                  (chain warps: dS is kept in their registers in fp32)
//
// Written out: dV, V . dV per token, for the gradient kernel dS (16-bit, transposed) of every chunk, and every
// ANCHOR chunks <dS, S>.
// Bound, as the scan, by the latency of one chunk's chain: 8 x 4096 tokens, 16 heads, K = V = 128 take 333 us,
// 5.2 us a chunk.  float16 422 us: the two terms of D have factors of their own and are read one after the other, dV is
// also written with a factor a token, and the instructions for both stand in the chain.  TMEM columns: dS hi, lo
// (64 each), Y and Z (64 each), then dV (128), D (128), dE, then Gam dV as operand (64), scaled dO (64).
#include "gdr_tc.cuh"

namespace ccq {
namespace gdrtc {
namespace {
using namespace tc;

constexpr uint32_t T_SH = 0, T_SL = 64, T_Y = 128, T_Z = 192, T_D = 256, T_EH = 384, T_EL = 416, T_GH = 448, T_GL = 480;

struct Small {
  uint64_t full[2], empty[2], s_ready, y_full, e_ready, f_full, f_ready, f_read, g_ready, d_full, kz, done;
  uint64_t d1_full, d1_read;  // float16: the first product of D^T
  float red[4][C];
  alignas(16) float top[2][16];  // float16: largest dS and Gam dV of each chain warp
  alignas(16) float vtop[4][C];  // largest dV of each token, by quadrant
  float undo[2];      // by the chunk's parity: what undoes the factor of the scaled dO
  uint32_t tmem;
  int abort;
};

constexpr uint32_t L_KQ = 0, L_V = 2 * TILE, L_DO = 3 * TILE, L_M = 4 * TILE, L_AX = L_M + MATS;
constexpr uint32_t L_STAGE = (L_AX + AX_N * 4 + 1023) & ~1023u;
constexpr uint32_t L_OUT = 2 * L_STAGE, L_SMALL = L_OUT + TILE;
constexpr uint32_t L_BYTES = L_SMALL + sizeof(Small) + 1024;
static_assert(L_BYTES <= 232448, "shared memory");

// SUM: nothing is written but the gradient at the segment's start, from a zero one at its end (the document's
// last segment: the given one)
template <int AB16, int KD, bool SUM>
__global__ void __launch_bounds__(BwdWarps::THREADS, 1)
    rscan_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                 const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmo,
                 const __grid_constant__ CUtensorMap tmdv, const __grid_constant__ CUtensorMap tms,
                 const __grid_constant__ CUtensorMap tmdvs, GdrArgs a, Ws w) {
  using G = BwdWarps;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Small& S_ = *reinterpret_cast<Small*>(sm + L_SMALL);
  const uint32_t sb = smem_u32(sm);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the V tiles of a head are neighbours, which read the same K, Q, T and P
  const int nvt = (a.V + VT - 1) / VT, vt = blockIdx.x % nvt, seg = blockIdx.x / nvt % w.nseg, head = blockIdx.x / nvt / w.nseg;
  const int n = doc_of_slot(head / a.HV, w.order), hv = head % a.HV, h = hv / (a.HV / a.H);
  const int v0 = vt * VT;
  const Segment part(a, w, n, seg);
  if (!part.live || (SUM && seg == 0)) return;
  const Seq sq = part.sq;
  const int nch = part.c1 - part.c0;
  const int64_t sh0 = (gdr_slot0(a, n, part.doc, C) + part.c0) * a.HV + hv;  // chunk c is at sh0 + c * HV
  const int64_t heads = (int64_t)a.n_seqs * a.HV, nh = (int64_t)n * a.HV + hv;
  const float* last = part.last() ? (a.dfinal_state ? a.dfinal_state + nh * a.K * a.V : nullptr)
                      : SUM ? nullptr : w.dSend + (seg * heads + nh) * a.K * a.V;
  float* start = SUM ? w.Bs + (seg * heads + nh) * a.K * a.V
                 : (seg == 0 && a.dinitial_state ? a.dinitial_state + nh * a.K * a.V : nullptr);
  constexpr int NP = KD / 64;  // panels of K and Q
  constexpr int CT = G::CT, OT = G::OT;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S_.full[i], 1);
      mbar_init(&S_.empty[i], 1 + G::CHAIN_WARPS + G::OUT_WARPS);  // last commit, every chain and output warp
    }
    mbar_init(&S_.s_ready, G::CHAIN_WARPS);
    mbar_init(&S_.e_ready, G::CHAIN_WARPS);
    mbar_init(&S_.f_ready, G::CHAIN_WARPS);
    mbar_init(&S_.f_read, G::OUT_WARPS);
    mbar_init(&S_.g_ready, G::OUT_WARPS);
    mbar_init(&S_.kz, G::OUT_WARPS);
    mbar_init(&S_.y_full, 1);
    mbar_init(&S_.f_full, 1);
    mbar_init(&S_.d_full, 1);
    mbar_init(&S_.done, 1);
    mbar_init(&S_.d1_full, 1);
    mbar_init(&S_.d1_read, G::CHAIN_WARPS);
    S_.abort = 0;
    fence_barrier_init();
  }
  if (warp == G::MMA) tmem_alloc(&S_.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tb = S_.tmem;
  volatile int* ab = &S_.abort;
  int* err = w.err;
  const bool partial = sq.len % C != 0;  // the last chunk, the first one here, is partial

  if (warp >= G::TMA) G::rest_regs();
  if (warp == G::TMA) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int issued = 0;
      for (int t = 0; t < nch; ++t) {
        const int s = t & 1, c = nch - 1 - t;
        if (t >= 2 && !pipe_wait(&S_.empty[s], ((t - 2) >> 1) & 1, ab, err, 1)) break;
        if (*ab) break;
        uint8_t* p = sm + s * L_STAGE;
        uint64_t* bar = &S_.full[s];
        mbar_arrive_expect_tx(bar, 2 * NP * PANEL + (SUM ? 1 : 2) * TILE + MATS + AX_N * 4);
        const int row = (int)(sq.bos + (int64_t)c * C);
        const int64_t sh = sh0 + (int64_t)c * a.HV;
        for (int i = 0; i < NP; ++i) tma_load_3d(p + L_KQ + 2 * i * PANEL, &tmk, bar, 64 * i, h, row);
        tma_load_3d(p + L_DO, &tmo, bar, v0, hv, row);
        tma_load_3d(p + L_DO + PANEL, &tmo, bar, v0 + 64, hv, row);
        bulk_load(p + L_AX, w.aux + sh * AX_N, AX_N * 4, bar);
        const uint8_t* mats = w.mats + sh * mats_bytes(AB16);
        if (AB16) {
          bulk_load(p + L_M, mats, MATS, bar);
        } else {  // T, and P beta in float16
          bulk_load(p + L_M, mats, MATS / 2, bar);
          bulk_load(p + L_M + MATS / 2, mats + MATS, MATS / 2, bar);
        }
        for (int i = 0; i < NP; ++i) tma_load_3d(p + L_KQ + (2 * i + 1) * PANEL, &tmq, bar, 64 * i, h, row);
        if (!SUM) {
          tma_load_3d(p + L_V, &tmv, bar, v0, hv, row);
          tma_load_3d(p + L_V + PANEL, &tmv, bar, v0 + 64, hv, row);
        }
        ++issued;
      }
      // never leave the block with copies in flight
      for (int t = (issued > 2 ? issued - 2 : 0); t < issued; ++t) own_copy_wait(&S_.full[t & 1], (t >> 1) & 1, ab, err, 2);
    }
  } else if (warp == G::MMA) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t id_y = idesc_f16(128, 64, AB16, 0, 0), id_z = idesc_f16(128, 64, AB16, 1, 1);
      const uint32_t id_d = idesc_f16(128, KD, AB16, 0, 1);
      const uint32_t id_f = idesc_f16(128, 128, 1, 0, 1), id_f2 = idesc_f16(128, 64, 1, 0, 1);  // T is bfloat16
      for (int t = 0; t < nch; ++t) {
        const int s = t & 1, ph = t & 1;
        const uint32_t p = sb + s * L_STAGE;
        const uint32_t T = p + L_M, P = T + 2 * PANEL;
        if (!spin_wait(&S_.full[s], (t >> 1) & 1, ab, err, 4)) break;
        if (t == 0 && partial && !spin_wait(&S_.kz, 0, ab, err, 8)) break;
        // Z^T over the dV of the chunk before
        if (t > 0 && !SUM && !spin_wait(&S_.f_read, (t - 1) & 1, ab, err, 0x20)) break;
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma(tb + T_Z, sdesc(p + L_DO + ks * 2048, PANEL, 1024), sdesc(P + x * PANEL + ks * 2048, PANEL, 1024), id_z,
                 x + ks > 0);
        // Y^T
        if (!spin_wait(&S_.s_ready, ph, ab, err, 0x10)) break;
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int ks = 0; ks < KD / 16; ++ks)
            umma_ts(tb + T_Y, tb + (x ? T_SL : T_SH) + 8 * ks,
                    sdesc(p + L_KQ + (ks >> 2) * 2 * PANEL + (ks & 3) * 32, 16, 1024), id_y, x + ks > 0);
        umma_commit(&S_.y_full);
        // dV^T = dE^T T; the hi and lo halves are added on reading
        if (!spin_wait(&S_.e_ready, ph, ab, err, 0x80)) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          umma_ts(tb + T_Y, tb + T_EH + 8 * ks, sdesc(T + ks * 2048, PANEL, 1024), id_f, ks > 0);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) umma_ts(tb + T_Y, tb + T_EL + 8 * ks, sdesc(T + ks * 2048, PANEL, 1024), id_f2, 1);
        umma_commit(&S_.f_full);
        // D^T = (scale Gam dO)^T Q
        if (!spin_wait(&S_.g_ready, ph, ab, err, 0x40)) break;
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma_ts(tb + T_D, tb + (x ? T_GL : T_GH) + 8 * ks, sdesc(p + L_KQ + PANEL + ks * 2048, 2 * PANEL, 1024), id_d,
                    x + ks > 0);
        if (!AB16) {  // the next product has a factor of its own: this one is read first
          umma_commit(&S_.d1_full);
          if (!spin_wait(&S_.d1_read, ph, ab, err, 0x100)) break;
        }
        // D^T += (-Gam dV)^T K
        if (!spin_wait(&S_.f_ready, ph, ab, err, 0x200)) break;
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma_ts(tb + T_D, tb + (x ? T_EL : T_EH) + 8 * ks, sdesc(p + L_KQ + ks * 2048, 2 * PANEL, 1024), id_d,
                    AB16 || x + ks > 0);
        umma_commit(&S_.d_full);
        umma_commit(&S_.empty[s]);
      }
      umma_commit(&S_.done);  // TMEM is freed only after every issued MMA has completed
      mbar_wait(&S_.done, 0);
    }
  } else if (warp > G::MMA) {
    // completes the warpgroup
  } else if (warp >= G::CHAIN) {
    // ------------------------------------------------------------------ chain: dE, Gam dV, dS
    G::chain_regs();
    constexpr int KH = 4 * KD / G::CHAIN_WARPS;  // columns of K this thread keeps
    const int quad = warp & 3, hh = (warp - G::CHAIN) >> 2;
    const int vl = quad * 32 + lane;
    const bool vin = v0 + vl < a.V;
    const uint32_t tl = tb + ((uint32_t)(quad * 32) << 16);
    float S[KH];
#pragma unroll
    for (int i = 0; i < KH; ++i) {
      const int k = KH * hh + i;
      S[i] = (last && vin && k < a.K) ? last[(int64_t)k * a.V + v0 + vl] : 0.f;
    }
    const int cw = warp - G::CHAIN;
    [[maybe_unused]] float* fx = factors_of(a, w) + ((int64_t)vt * gdr_slots(a, C) * a.HV + sh0) * FX_N;  // of the first chunk
    float uS = 1.f, bS = 0.f;  // float16: what undoes the factor of dS, and a bound on dS
    // dS as the operand of chunk c; its hi part also goes to `tile` (two panels of 128 rows), or straight
    // to the workspace for the first chunk
    auto put_state = [&](uint32_t tile, int c) {
      Pow2 f{1.f, 1.f};
      if constexpr (!AB16) {
        if ((nch - 1 - c) % EXACT == 0) bS = warps_max<2, G::CHAIN_WARPS>(abs_max<KH>(S), S_.top[0], cw);
        f = pow2_of(bS);
        uS = f.u;
        if (!SUM && threadIdx.x == 32 * G::CHAIN) fx[(int64_t)c * a.HV * FX_N + FX_DS] = f.u;
      }
#pragma unroll
      for (int i = 0; i < KH; i += 16) {
        uint32_t hi[8], lo[8];
        if constexpr (AB16) {
          split<AB16, 8>(S + i, hi, lo);
        } else {
          float x[16];
          const float ss[2] = {f.s, f.s};
#pragma unroll
          for (int j = 0; j < 16; j += 2) mul2f(x + j, S + i + j, ss);
          split<AB16, 8>(x, hi, lo);
        }
        tmem_st8(tl + T_SH + hh * (KH / 2) + i / 2, hi);
        tmem_st8(tl + T_SL + hh * (KH / 2) + i / 2, lo);
        const int k = KH * hh + i;
        const uint4 u = make_uint4(hi[0], hi[1], hi[2], hi[3]), v = make_uint4(hi[4], hi[5], hi[6], hi[7]);
        if (tile != 0) {
          const uint32_t pan = tile + (k >> 6) * 2 * PANEL;
          sts128(pan + sw128(vl, (k & 63) >> 3), u);
          sts128(pan + sw128(vl, ((k & 63) >> 3) + 1), v);
        } else if (vin && !SUM) {
          uint16_t* g = w.dS1 + ((sh0 + (int64_t)(nch - 1) * a.HV) * a.V + v0 + vl) * a.K + k;
          if (k < a.K) *reinterpret_cast<uint4*>(g) = u;
          if (k + 8 < a.K) *reinterpret_cast<uint4*>(g + 8) = v;
        }
      }
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&S_.s_ready);
    };
    // <dS, S> at the end of anchor group b, this warp's part
    const int64_t anchors = gdr_slots(a, C * ANCHOR);
    auto put_anchor = [&](int b, bool zero) {
      const int64_t at = (gdr_slot0(a, n, part.doc, C * ANCHOR) + b) * a.HV + hv;
      float d = 0.f;
      if (vin && !zero) {
        const float* g = w.Sf + at * a.K * a.V + v0 + vl;
#pragma unroll
        for (int i = 0; i < KH; ++i)
          if (KH * hh + i < a.K) d = fmaf(S[i], g[(int64_t)(KH * hh + i) * a.V], d);
      }
      d = warp_sum(d);
      if (lane == 0) w.anchor[((int64_t)vt * anchors * a.HV + at) * G::CHAIN_WARPS + warp - G::CHAIN] = d;
    };
    if (nch > 0) {
      put_state(0, nch - 1);
      if (!SUM && part.last()) put_anchor((part.nch - 1) / ANCHOR, a.dfinal_state == nullptr);
    }
    const int i0 = CT * hh;
    for (int t = 0; t < nch; ++t) {
      const int s = t & 1, ph = t & 1, c = nch - 1 - t;
      const float* ax = reinterpret_cast<const float*>(sm + s * L_STAGE + L_AX);
      pipe_wait(&S_.full[s], (t >> 1) & 1, ab, err, 0x400);
      pipe_wait(&S_.y_full, ph, ab, err, 0x800);
      tc_fence_after();
      if constexpr (AB16) {
#pragma unroll
        for (int i = 0; i < CT; i += 16) {
          float x[16];
          tmem_ld16(tl + T_Z + i0 + i, x);
#pragma unroll
          for (int k = 0; k < 16; k += 8) {
            float y[8];
            tmem_ld8(tl + T_Y + i0 + i + k, y);
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
              const float4 b = *reinterpret_cast<const float4*>(ax + AX_WB + i0 + i + k + j);
              const float bb[4] = {b.x, b.y, b.z, b.w};
              float* z = x + k + j;
              fma2(z, bb, y + j, z);
              fma2(z + 2, bb + 2, y + j + 2, z + 2);
            }
          }
          st_split16<AB16>(tl + T_EH + (i0 + i) / 2, tl + T_EL + (i0 + i) / 2, x);
        }
      } else {
        static_assert(CT == 16, "one load");
        const float uP = ax[AX_UP];
        float x[16];
        tmem_ld16(tl + T_Z + i0, x);
#pragma unroll
        for (int k = 0; k < 16; k += 8) {
          float y[8];
          tmem_ld8(tl + T_Y + i0 + k, y);
#pragma unroll
          for (int j = 0; j < 8; j += 4) {
            const float4 b = *reinterpret_cast<const float4*>(ax + AX_WB + i0 + k + j);
            x[k + j] = fmaf(b.x * uS, y[j], x[k + j] * uP);
            x[k + j + 1] = fmaf(b.y * uS, y[j + 1], x[k + j + 1] * uP);
            x[k + j + 2] = fmaf(b.z * uS, y[j + 2], x[k + j + 2] * uP);
            x[k + j + 3] = fmaf(b.w * uS, y[j + 3], x[k + j + 3] * uP);
          }
        }
        st_split16<1>(tl + T_EH + i0 / 2, tl + T_EL + i0 / 2, x);
      }
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&S_.e_ready);
      pipe_wait(&S_.f_full, ph, ab, err, 0x1000);
      tc_fence_after();
      [[maybe_unused]] float uG[2] = {1.f, 1.f};  // float16: what undoes the factor of Gam dV
#pragma unroll
      for (int i = 0; i < CT; i += 16) {
        float x[16];
        tmem_ld16(tl + T_Y + i0 + i, x);
#pragma unroll
        for (int k = 0; k < 16; k += 8) {
          float y[8];
          tmem_ld8(tl + T_Y + 64 + i0 + i + k, y);
#pragma unroll
          for (int j = 0; j < 8; j += 4) {
            const float4 b = *reinterpret_cast<const float4*>(ax + AX_G + i0 + i + k + j);
            const float bb[4] = {-b.x, -b.y, -b.z, -b.w};
            float* z = x + k + j;
            add2f(z, z, y + j);
            add2f(z + 2, z + 2, y + j + 2);
            mul2f(z, z, bb);
            mul2f(z + 2, z + 2, bb + 2);
          }
        }
        if constexpr (!AB16) {
          const float m = warps_max<2, G::CHAIN_WARPS>(abs_max<16>(x), S_.top[1], cw);
          const Pow2 f = pow2_of(m);
          const float ss[2] = {f.s, f.s};
          uG[0] = uG[1] = f.u;
          bS = fmaf(64.f * ax[AX_KN], m, ax[AX_GC] * bS);
#pragma unroll
          for (int j = 0; j < 16; j += 2) mul2f(x + j, x + j, ss);
        }
        st_split16<AB16>(tl + T_EH + (i0 + i) / 2, tl + T_EL + (i0 + i) / 2, x);
      }
      const float gam[2] = {ax[AX_GC], ax[AX_GC]};
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&S_.f_ready);
      if constexpr (!AB16) {  // dS = Gam_C dS + the first product
        pipe_wait(&S_.d1_full, ph, ab, err, 0x2000);
        pipe_wait(&S_.g_ready, ph, ab, err, 0x2000);  // the factor was left before; the phase lasts until d1_read of this chunk
        tc_fence_after();
        const float u = S_.undo[t & 1], uo[2] = {u, u};
        bS = fmaf(64.f * ax[AX_QN], 32768.f * u, bS);
#pragma unroll
        for (int i = 0; i < KH; i += 16) {
          float x[16];
          tmem_ld16(tl + T_D + KH * hh + i, x);
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            mul2f(x + j, x + j, uo);
            fma2(S + i + j, gam, S + i + j, x + j);
          }
        }
        tc_fence_before();
        warp_arrive(&S_.d1_read);
      }
      if (warp != G::CHAIN) warp_arrive(&S_.empty[s]);
      pipe_wait(&S_.d_full, ph, ab, err, 0x2000);
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < KH; i += 16) {
        float x[16];
        tmem_ld16(tl + T_D + KH * hh + i, x);
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          if constexpr (AB16) fma2(S + i + j, gam, S + i + j, x + j);
          else fma2(S + i + j, uG, x + j, S + i + j);
        }
      }
      if (c > 0) put_state(sb + s * L_STAGE + L_KQ, c - 1);  // every product with the K and Q rows is done: their space is the staging
      fence_async_smem();
      bar_sync<2, G::CHAIN_THREADS>();
      if (threadIdx.x == 32 * G::CHAIN) {
        if (c > 0 && !SUM)
          for (int i = 0; i < NP; ++i)
            if (64 * i < a.K)
              store_panel(&tms, sm + s * L_STAGE + L_KQ + 2 * i * PANEL, 64 * i, v0, a.V, sh0 + (int64_t)(c - 1) * a.HV);
        bulk_wait_read();  // then the stage may be loaded again
        mbar_arrive(&S_.empty[s]);
      }
      if (const int cd = part.c0 + c; !SUM && cd > 0 && cd % ANCHOR == 0) put_anchor(cd / ANCHOR - 1, false);
    }
    if (threadIdx.x == 32 * G::CHAIN) bulk_wait_all();
    if (start && vin) {
#pragma unroll
      for (int i = 0; i < KH; ++i) {
        const int k = KH * hh + i;
        if (k < a.K) start[(int64_t)k * a.V + v0 + vl] = S[i];
      }
    }
  } else {
    // ------------------------------------------------------------------ output: scaled dO, dV, V . dV
    G::out_regs();
    const int quad = warp & 3, j0 = OT * (warp >> 2);  // tokens j0 .. j0 + OT - 1
    const int vl = quad * 32 + lane;
    const uint32_t tl = tb + ((uint32_t)(quad * 32) << 16);
    const int64_t slots = gdr_slots(a, C);
    [[maybe_unused]] float* fx = factors_of(a, w) + ((int64_t)vt * slots * a.HV + sh0) * FX_N;  // of the first chunk
    [[maybe_unused]] float top = !AB16 && nch > 0 ? fx[(int64_t)(nch - 1) * a.HV * FX_N + FX_DO] : 0.f;
    for (int t = 0; t < nch; ++t) {
      const int s = t & 1, ph = t & 1, c = nch - 1 - t;
      const int valid = min(C, sq.len - c * C);
      const uint32_t p = sb + s * L_STAGE;
      const float* ax = reinterpret_cast<const float*>(sm + s * L_STAGE + L_AX);
      const int64_t row0 = sq.bos + (int64_t)c * C;
      pipe_wait(&S_.full[s], (t >> 1) & 1, ab, err, 0x4000);
      if (valid < C) {
        // the rows past the document belong to another one: what a product sums over must be zero
        for (int i = 0; i < 2 * NP; ++i) zero_rows(p + L_KQ + i * PANEL, 1, valid, threadIdx.x, G::OUT_THREADS);
        zero_rows(p + L_DO, 2, valid, threadIdx.x, G::OUT_THREADS);
        fence_async_smem();
        warp_arrive(&S_.kz);
      }
      if (t > 0) pipe_wait(&S_.d_full, (t - 1) & 1, ab, err, 0x8000);  // the operand of the chunk before is read
      tc_fence_after();
      Pow2 fo{1.f, 1.f};
      if constexpr (!AB16) {  // from a bound: largest |dO|, which the forward scan left, by the largest scale Gam
        fo = pow2_of(ax[AX_SM] * top);
        if (threadIdx.x == 0) S_.undo[t & 1] = fo.u;
        top = c > 0 ? fx[(int64_t)(c - 1) * a.HV * FX_N + FX_DO] : 0.f;
      }
      {
        const Column D(p + L_DO, vl);
#pragma unroll
        for (int i = j0; i < j0 + OT; i += 16) {
          float x[16];
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 b = *reinterpret_cast<const float4*>(ax + AX_SG + i + j);
            const float bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[j + e] = i + j + e < valid ? bb[e] * h2f<AB16>(lds16(D.at(i + j + e))) : 0.f;
              if (!AB16) x[j + e] *= fo.s;
            }
          }
          st_split16<AB16>(tl + T_GH + i / 2, tl + T_GL + i / 2, x);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&S_.g_ready);
      if (SUM) {
        warp_arrive(&S_.empty[s]);
        continue;
      }
      float y[OT];
      pipe_wait(&S_.f_full, ph, ab, err, 0x10000);
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < OT; i += 16) {
        float x[16];
        tmem_ld16(tl + T_Y + j0 + i, y + i);
        tmem_ld16(tl + T_Y + 64 + j0 + i, x);
#pragma unroll
        for (int j = 0; j < 16; j += 2) add2f(y + i + j, y + i + j, x + j);
      }
      tc_fence_before();
      warp_arrive(&S_.f_read);
      if (!AB16) token_max_put<OT>(y, S_.vtop, j0, quad, lane);
      if (threadIdx.x == 0) bulk_wait_read();  // the stores of the chunk before have read the tile
      bar_sync<1, G::OUT_THREADS>();
      const Column O(sb + L_OUT, vl), V(p + L_V, vl);
#pragma unroll
      for (int i = 0; i < OT; ++i) sts16(O.at(j0 + i), f2h<AB16>(y[i]));
      if constexpr (AB16) {
#pragma unroll
        for (int i = 0; i < OT; ++i) y[i] = j0 + i < valid ? y[i] * h2f<AB16>(lds16(V.at(j0 + i))) : 0.f;
        warp_arrive(&S_.empty[s]);
      } else {  // dV with its factor, for the gradient kernel, takes the place of V
        static_assert(OT == 32, "a token a lane");
        const Pow2 f = pow2_of(token_max_get(S_.vtop, j0 + lane));
        if (quad == 0) fx[(int64_t)c * a.HV * FX_N + FX_DV + j0 + lane] = f.u;
#pragma unroll
        for (int i = 0; i < OT; ++i) {
          const uint32_t at = V.at(j0 + i);
          const float v = h2f<AB16>(lds16(at));
          sts16(at, f2h<AB16>(y[i] * __shfl_sync(0xffffffffu, f.s, i)));
          y[i] = j0 + i < valid ? y[i] * v : 0.f;
        }
        if (warp > 0) warp_arrive(&S_.empty[s]);  // warp 0: once the tile is stored
      }
      lane_sums<OT>(y, lane);
#pragma unroll
      for (int i = 0; i < OT / 32; ++i) S_.red[quad][j0 + lane * (OT / 32) + i] = y[i];
      fence_async_smem();
      bar_sync<1, G::OUT_THREADS>();
      if (valid == C) {
        if (threadIdx.x == 0) {
          tma_store_3d(&tmdv, sm + L_OUT, v0, hv, (int)row0);
          if (v0 + 64 < a.V) tma_store_3d(&tmdv, sm + L_OUT + PANEL, v0 + 64, hv, (int)row0);
          if (!AB16) {
            tma_store_3d(&tmdvs, sm + s * L_STAGE + L_V, v0, hv, (int)row0);
            if (v0 + 64 < a.V) tma_store_3d(&tmdvs, sm + s * L_STAGE + L_V + PANEL, v0 + 64, hv, (int)row0);
          }
          bulk_commit();
        }
      } else {
        copy_rows(sb + L_OUT, reinterpret_cast<uint16_t*>(a.dv), row0, a.HV, hv, a.V, v0, valid, threadIdx.x, G::OUT_THREADS);
        if (!AB16) copy_rows(p + L_V, scaled_dv_of(a, w), row0, a.HV, hv, a.V, v0, valid, threadIdx.x, G::OUT_THREADS);
      }
      if (threadIdx.x < C) {
        const int i = threadIdx.x;
        w.dotV[((int64_t)vt * slots * a.HV + sh0 + (int64_t)c * a.HV) * C + i] =
            S_.red[0][i] + S_.red[1][i] + S_.red[2][i] + S_.red[3][i];
      }
      bar_sync<1, G::OUT_THREADS>();  // the sums are read before the next chunk's are written
      if (!AB16 && warp == 0) {
        if (lane == 0) bulk_wait_read();
        warp_arrive(&S_.empty[s]);
      }
    }
    if (threadIdx.x == 0) bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == G::MMA) tmem_dealloc(tb, 512);
}

template <int AB16, int KD, bool SUM>
cudaError_t launch(const GdrArgs& a, const Ws& w) {
  CUtensorMap q, k, v, o, dv, st, dvs;
  cudaError_t e = token_map(&q, a, a.q, a.H, a.K);
  if (e == cudaSuccess) e = token_map(&k, a, a.k, a.H, a.K);
  if (e == cudaSuccess) e = token_map(&v, a, a.v, a.HV, a.V);
  if (e == cudaSuccess) e = token_map(&o, a, a.d_o, a.HV, a.V);
  if (e == cudaSuccess) e = token_map(&dv, a, a.dv, a.HV, a.V);
  if (e == cudaSuccess) e = matrix_map(&st, a, w.dS1, a.K, gdr_slots(a, C) * a.HV);
  dvs = dv;
  if (!AB16 && e == cudaSuccess) e = token_map(&dvs, a, scaled_dv_of(a, w), a.HV, a.V);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(rscan_kernel<AB16, KD, SUM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L_BYTES);
  if (e != cudaSuccess) return e;
  const int64_t blocks = (int64_t)a.n_seqs * a.HV * w.nseg * ((a.V + VT - 1) / VT);
  rscan_kernel<AB16, KD, SUM><<<(unsigned)blocks, BwdWarps::THREADS, L_BYTES, a.stream>>>(q, k, v, o, dv, st, dvs, a, w);
  return cudaGetLastError();
}

template <int AB16, int KD>
cudaError_t pick(const GdrArgs& a, const Ws& w, bool sum) {
  return sum ? launch<AB16, KD, true>(a, w) : launch<AB16, KD, false>(a, w);
}

}  // namespace

cudaError_t rscan(const GdrArgs& a, const Ws& w, bool sum, int* launches) {
  ++*launches;
  const bool small = a.K <= 64;
  if (a.dtype == DT_BF16) return small ? pick<1, 64>(a, w, sum) : pick<1, 128>(a, w, sum);
  return small ? pick<0, 64>(a, w, sum) : pick<0, 128>(a, w, sum);
}

}  // namespace gdrtc
}  // namespace ccq
