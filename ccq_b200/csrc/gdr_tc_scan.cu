// Tensor-core path of the gated delta rule, forward scan: one block per (document, value head, 128
// columns of V) walks the document in chunks of 64 tokens.  Everything is held transposed, one column of V
// per TMEM lane, so that the three products of a chunk chain through TMEM without a transposition:
//
//   X^T | Y^T = S^T [K ; Q]^T   [128 x 128]  A: S hi + lo (TMEM), B: the K and Q rows, one above the other
//   E^T  = V^T T^T              [128 x 128]  A: the V tile, read MN-major, B: [T hi | T lo] side by side
//        + (-Gam X)^T T^T                    A: Gam X hi + lo (chain warps, back to TMEM), B: T hi, lo
//   dS^T = (w beta E)^T K       [128 x K]    A: hi + lo (chain warps), B: the K rows, read MN-major
//   S^T  = Gam_C S^T + dS^T                  (chain warps: S is kept in their registers in fp32)
//   O^T  = scale Gam Y^T + E^T (P beta)^T    (beside the chain; output warps)
//
// The chunks are sequential, so the kernel is bound by the latency of that chain (three MMA groups, three
// TMEM round trips) and not by the MMA rate or by memory; a second block on an SM does not fit (TMEM is
// full), and splitting K or V further would not shorten the chain.  An MMA with its A operand in TMEM
// takes about 64 cycles for any N up to 128 here, so what can share an A operand is put side by side in N.
// The rest of a chunk's period is instructions of the chain warps between the products, so V enters by an MMA
// of its own (beside the chain) and the factors by packed two-value arithmetic.  8 x 4096 tokens, 16 heads,
// K = V = 128: 233 us, 3.6 us a chunk; 331 us with what the backward reads (BWD), 256 MB more written.
//
// float16 (its factors: gdr_tc.cuh): the chain warps form R = V - Gam X, and E^T = R^T T^T is one product in bfloat16.
// What the factors cost is instructions of the chain warps and their barriers: 287 us, and 439 us for the backward, where E
// is staged behind S, beside the next chunk's first product, since its tokens' factors take a barrier of their own.
//
// BWD: instead of O it writes what the backward reads: S0 (16-bit, transposed), E (hi + lo), dO . O and,
// every ANCHOR chunks, S in fp32.
//
// TMEM columns: S hi, S lo (64 each), X | Y, then dS (128), E, then E P^T
// (128), Gam X / E as operands (64), w beta E as operand (64): all 512.  Every wait is bounded; see tc_common.cuh.
#include <type_traits>

#include "gdr_tc.cuh"

namespace ccq {
namespace gdrtc {
namespace {
using namespace tc;

constexpr uint32_t T_SH = 0, T_SL = 64, T_X = 128, T_D = 256, T_RH = 384, T_RL = 416, T_WH = 448, T_WL = 480;

struct Small {
  uint64_t full[2], empty[2], s_ready, x_full, r_ready, u_full, u_ready, d_full, o1_read, o_full, o2_free, kz, done;
  float red[4][C];
  alignas(16) float top[2][16];  // float16: largest S and w beta E of each chain warp
  alignas(16) float etop[4][C];  // largest E of each token, by quadrant
  float dtop[8];              // largest dO of each output warp
  float undo[2];        // by the chunk's parity: what undoes the factor of S
  uint32_t tmem;
  int abort;
};

template <bool BWD>
using Warps = std::conditional_t<BWD, BwdWarps, FwdWarps>;

template <bool BWD>
struct Lay {  // offsets of one stage, then of the rest
  static constexpr uint32_t KQ = 0, V = 2 * TILE, DO = 3 * TILE, M = (BWD ? 4 : 3) * TILE, AX = M + MATS;
  static constexpr uint32_t STAGE = (AX + AX_N * 4 + 1023) & ~1023u;
  static constexpr uint32_t OUT = 2 * STAGE, SMALL = OUT + TILE;
  static constexpr uint32_t BYTES = SMALL + sizeof(Small) + 1024;
};
static_assert(Lay<true>::BYTES <= 232448 && Lay<false>::BYTES <= 232448, "shared memory");

// SUM: no output; the state at the segment's end from a zero state (the first segment: the given one) over its V,
// or, in a head's last tile, as a linear map of the state at its start: the same walk from the identity without V.
template <int AB16, int KD, bool BWD, bool SUM>
__global__ void __launch_bounds__(Warps<BWD>::THREADS, 1)
    scan_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmo,
                const __grid_constant__ CUtensorMap tms, const __grid_constant__ CUtensorMap tme, GdrArgs a, Ws w) {
  using L = Lay<BWD>;
  using G = Warps<BWD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Small& S_ = *reinterpret_cast<Small*>(sm + L::SMALL);
  const uint32_t sb = smem_u32(sm);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the V tiles of a head are neighbours, which read the same K, Q, T and P
  const int nvt = (a.V + VT - 1) / VT, tiles = SUM ? nvt + 1 : nvt, segs = SUM ? w.nseg - 1 : w.nseg;
  const int vt = blockIdx.x % tiles, seg = blockIdx.x / tiles % segs, head = blockIdx.x / tiles / segs;
  const int n = doc_of_slot(head / a.HV, w.order), hv = head % a.HV, h = hv / (a.HV / a.H);
  const bool map = SUM && vt == nvt;
  const int v0 = map ? 0 : vt * VT, width = map ? a.K : a.V;  // of the state: columns it has
  const Segment part(a, w, n, seg);
  if (!part.live || (SUM && (part.last() || (map && seg == 0)))) return;
  const Seq sq = part.sq;
  const int nch = part.c1 - part.c0;
  const int64_t sh0 = (gdr_slot0(a, n, part.doc, C) + part.c0) * a.HV + hv;  // chunk c is at sh0 + c * HV
  const int64_t heads = (int64_t)a.n_seqs * a.HV, nh = (int64_t)n * a.HV + hv;
  const float* first = seg == 0 ? (a.initial_state ? a.initial_state + nh * a.K * a.V : nullptr)
                       : SUM ? nullptr : w.Sin + (seg * heads + nh) * a.K * a.V;
  float* final = SUM ? (map ? w.Ms : w.Bs) + (seg * heads + nh) * a.K * width
                 : (part.last() && a.final_state ? a.final_state + nh * a.K * a.V : nullptr);
  constexpr int NP = KD / 64;  // panels of K and Q
  constexpr int CT = G::CT, OT = G::OT;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S_.full[i], 1);
      mbar_init(&S_.empty[i], 1 + G::CHAIN_WARPS + (SUM ? 0 : G::OUT_WARPS));  // last commit, every chain and output warp
    }
    mbar_init(&S_.s_ready, G::CHAIN_WARPS);
    mbar_init(&S_.r_ready, G::CHAIN_WARPS);
    mbar_init(&S_.u_ready, G::CHAIN_WARPS);
    mbar_init(&S_.x_full, 1);
    mbar_init(&S_.u_full, 1);
    mbar_init(&S_.d_full, 1);
    mbar_init(&S_.o_full, 1);
    mbar_init(&S_.o1_read, G::OUT_WARPS);
    mbar_init(&S_.o2_free, G::OUT_WARPS);
    mbar_init(&S_.kz, G::OUT_WARPS);
    mbar_init(&S_.done, 1);
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

  if (warp >= G::TMA) G::rest_regs();
  if (warp == G::TMA) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int issued = 0;
      for (int c = 0; c < nch; ++c) {
        const int s = c & 1;
        if (c >= 2 && !pipe_wait(&S_.empty[s], ((c - 2) >> 1) & 1, ab, err, 1)) break;
        if (*ab) break;
        uint8_t* p = sm + s * L::STAGE;
        uint64_t* bar = &S_.full[s];
        if (SUM) mbar_arrive_expect_tx(bar, NP * PANEL + (map ? 0 : TILE) + MATS / 2 + AX_N * 4);
        else mbar_arrive_expect_tx(bar, 2 * NP * PANEL + (BWD ? 2 : 1) * TILE + MATS + AX_N * 4);
        const int row = (int)(sq.bos + (int64_t)c * C);
        const int64_t sh = sh0 + (int64_t)c * a.HV;
        for (int i = 0; i < NP; ++i) tma_load_3d(p + L::KQ + 2 * i * PANEL, &tmk, bar, 64 * i, h, row);
        if (!map) {
          tma_load_3d(p + L::V, &tmv, bar, v0, hv, row);
          tma_load_3d(p + L::V + PANEL, &tmv, bar, v0 + 64, hv, row);
        }
        bulk_load(p + L::AX, w.aux + sh * AX_N, AX_N * 4, bar);
        bulk_load(p + L::M, w.mats + sh * mats_bytes(AB16), SUM ? MATS / 2 : MATS, bar);
        for (int i = 0; i < NP && !SUM; ++i) tma_load_3d(p + L::KQ + (2 * i + 1) * PANEL, &tmq, bar, 64 * i, h, row);
        if (BWD) {
          tma_load_3d(p + L::DO, &tmo, bar, v0, hv, row);
          tma_load_3d(p + L::DO + PANEL, &tmo, bar, v0 + 64, hv, row);
        }
        ++issued;
      }
      // never leave the block with copies in flight
      for (int c = (issued > 2 ? issued - 2 : 0); c < issued; ++c) own_copy_wait(&S_.full[c & 1], (c >> 1) & 1, ab, err, 2);
    }
  } else if (warp == G::MMA) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t id64 = idesc_f16(128, 64, AB16, 0, 0), id128 = idesc_f16(128, 128, AB16, 0, 0);
      const uint32_t ib64 = idesc_f16(128, 64, 1, 0, 0), ib128 = idesc_f16(128, 128, 1, 0, 0);  // T and P beta are bfloat16
      const uint32_t id_d = idesc_f16(128, KD, AB16, 0, 1), id_v = idesc_f16(128, 128, AB16, 1, 0);
      for (int c = 0; c < nch; ++c) {
        const int s = c & 1, ph = c & 1;
        const uint32_t p = sb + s * L::STAGE;
        const uint32_t T = p + L::M, P = T + 2 * PANEL;
        // X^T | Y^T
        if (!spin_wait(&S_.full[s], (c >> 1) & 1, ab, err, 4)) break;
        if (!SUM && (c + 1) * C > sq.len && !spin_wait(&S_.kz, 0, ab, err, 8)) break;
        if (!spin_wait(&S_.s_ready, ph, ab, err, 0x10)) break;
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int ks = 0; ks < KD / 16; ++ks)
            umma_ts(tb + T_X, tb + (x ? T_SL : T_SH) + 8 * ks,
                    sdesc(p + L::KQ + (ks >> 2) * 2 * PANEL + (ks & 3) * 32, 16, 1024), SUM ? id64 : id128, x + ks > 0);
        umma_commit(&S_.x_full);
        // E^T = V^T T^T, then + (-Gam X)^T T^T (float16: R^T T^T); the hi and lo halves are added on reading
        if (!SUM && c > 0 && !spin_wait(&S_.o2_free, (c - 1) & 1, ab, err, 0x20)) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < 4 && AB16 && !map; ++ks)
          umma(tb + T_D, sdesc(p + L::V + ks * 2048, PANEL, 1024), sdesc(T + ks * 32, 16, 1024), id_v, ks > 0);
        if (!spin_wait(&S_.r_ready, ph, ab, err, 0x40)) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) umma_ts(tb + T_D, tb + T_RH + 8 * ks, sdesc(T + ks * 32, 16, 1024), ib128, (AB16 && !map) || ks > 0);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) umma_ts(tb + T_D, tb + T_RL + 8 * ks, sdesc(T + ks * 32, 16, 1024), ib64, 1);
        umma_commit(&S_.u_full);
        // dS^T = (w beta E)^T K over X | Y, then E^T (P beta)^T over E
        if (!SUM && !spin_wait(&S_.o1_read, ph, ab, err, 0x200)) break;
        if (!spin_wait(&S_.u_ready, ph, ab, err, 0x80)) break;
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma_ts(tb + T_X, tb + (x ? T_WL : T_WH) + 8 * ks, sdesc(p + L::KQ + ks * 2048, 2 * PANEL, 1024), id_d, x + ks > 0);
        umma_commit(&S_.d_full);
        if (!SUM) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) umma_ts(tb + T_D, tb + T_RH + 8 * ks, sdesc(P + ks * 32, 16, 1024), ib128, ks > 0);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) umma_ts(tb + T_D, tb + T_RL + 8 * ks, sdesc(P + ks * 32, 16, 1024), ib64, 1);
          umma_commit(&S_.o_full);
        }
        umma_commit(&S_.empty[s]);
      }
      umma_commit(&S_.done);  // TMEM is freed only after every issued MMA has completed
      mbar_wait(&S_.done, 0);
    }
  } else if (warp > G::MMA) {
    // completes the warpgroup
  } else if (warp >= G::CHAIN) {
    // ------------------------------------------------------------------ chain: Gam X, E, S
    G::chain_regs();
    constexpr int KH = 4 * KD / G::CHAIN_WARPS;  // columns of K this thread keeps
    constexpr int NY = G::CT >= 32 ? 16 : 8;  // columns per load where registers are short
    const int quad = warp & 3, hh = (warp - G::CHAIN) >> 2;
    const int vl = quad * 32 + lane;
    const bool vin = v0 + vl < width;
    const uint32_t tl = tb + ((uint32_t)(quad * 32) << 16);
    float S[KH];
#pragma unroll
    for (int i = 0; i < KH; ++i) {
      const int k = KH * hh + i;
      S[i] = (first && vin && k < a.K) ? first[(int64_t)k * a.V + v0 + vl] : map && k == vl && vin ? 1.f : 0.f;
    }
    const int cw = warp - G::CHAIN;
    [[maybe_unused]] float* fx = factors_of(a, w) + ((int64_t)vt * gdr_slots(a, C) * a.HV + sh0) * FX_N;  // of the first chunk
    float uS = 1.f, bS = 0.f;  // float16: what undoes the factor of S, and a bound on S
    // S as the operand of chunk c; for the backward its hi part also goes to `tile` (two panels of
    // 128 rows), or straight to the workspace for the first chunk
    auto put_state = [&](uint32_t tile, int c) {
      Pow2 f{1.f, 1.f};
      if constexpr (!AB16) {
        if (c % EXACT == 0) bS = warps_max<2, G::CHAIN_WARPS>(abs_max<KH>(S), S_.top[0], cw);
        f = pow2_of(bS);
        uS = f.u;
        if (threadIdx.x == 32 * G::CHAIN) {
          S_.undo[c & 1] = f.u;
          if (BWD) fx[(int64_t)c * a.HV * FX_N + FX_S] = f.u;
        }
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
        if (BWD) {
          const int k = KH * hh + i;
          const uint4 u = make_uint4(hi[0], hi[1], hi[2], hi[3]), v = make_uint4(hi[4], hi[5], hi[6], hi[7]);
          if (tile != 0) {
            const uint32_t pan = tile + (k >> 6) * 2 * PANEL;
            sts128(pan + sw128(vl, (k & 63) >> 3), u);
            sts128(pan + sw128(vl, ((k & 63) >> 3) + 1), v);
          } else if (vin) {
            uint16_t* g = w.S0 + (sh0 * a.V + v0 + vl) * a.K + k;
            if (k < a.K) *reinterpret_cast<uint4*>(g) = u;
            if (k + 8 < a.K) *reinterpret_cast<uint4*>(g + 8) = v;
          }
        }
      }
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&S_.s_ready);
    };
    const int i0 = CT * hh;
    // E of tokens i0 + i .. + 15, its two halves added
    auto load_e = [&](int i, float* x) {
      tmem_ld16(tl + T_D + i0 + i, x);
#pragma unroll
      for (int k = 0; k < 16; k += NY) {
        float y[NY];
        if (NY == 16) tmem_ld16(tl + T_D + 64 + i0 + i + k, y);
        else tmem_ld8(tl + T_D + 64 + i0 + i + k, y);
#pragma unroll
        for (int j = 0; j < NY; j += 2) add2f(x + k + j, x + k + j, y + j);
      }
    };
    // float16, backward: E of this thread's 16 tokens from the operand, hi + lo, which stays until the next chunk's R
    [[maybe_unused]] auto read_e = [&](float* x) {
      static_assert(!BWD || CT == 16, "one piece");
      float h[8], l[8];
      tmem_ld8(tl + T_RH + i0 / 2, h);
      tmem_ld8(tl + T_RL + i0 / 2, l);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 u = unpack2<1>(__float_as_uint(h[j])), v = unpack2<1>(__float_as_uint(l[j]));
        x[2 * j] = u.x + v.x;
        x[2 * j + 1] = u.y + v.y;
      }
    };
    // E, transposed, to the staging panel (hi) and over the V tile, whose product is done (lo)
    auto stage_e = [&](uint32_t p, int i, const uint32_t* hi, const uint32_t* lo) {
      sts128(sb + L::OUT + sw128(vl, (i0 + i) >> 3), make_uint4(hi[0], hi[1], hi[2], hi[3]));
      sts128(sb + L::OUT + sw128(vl, ((i0 + i) >> 3) + 1), make_uint4(hi[4], hi[5], hi[6], hi[7]));
      sts128(p + L::V + sw128(vl, (i0 + i) >> 3), make_uint4(lo[0], lo[1], lo[2], lo[3]));
      sts128(p + L::V + sw128(vl, ((i0 + i) >> 3) + 1), make_uint4(lo[4], lo[5], lo[6], lo[7]));
    };
    if (nch > 0) put_state(0, 0);
    for (int c = 0; c < nch; ++c) {
      const int s = c & 1, ph = c & 1;
      const uint32_t p = sb + s * L::STAGE;
      const float* ax = reinterpret_cast<const float*>(sm + s * L::STAGE + L::AX);
      pipe_wait(&S_.full[s], (c >> 1) & 1, ab, err, 0x400);
      [[maybe_unused]] uint32_t v[AB16 ? 1 : CT / 2];  // float16: this thread's part of V, asked for before X is there
      if constexpr (!AB16) {
        const int valid = map ? 0 : min(C, sq.len - c * C);
        const Column V(p + L::V, vl);
#pragma unroll
        for (int i = 0; i < CT; i += 2) {
          const uint32_t lo = lds16_early(V.at(i0 + i)), hi = lds16_early(V.at(i0 + i + 1));
          v[i / 2] = (i0 + i < valid ? lo : 0) | (i0 + i + 1 < valid ? hi << 16 : 0);  // behind the document: anything
        }
      }
      pipe_wait(&S_.x_full, ph, ab, err, 0x800);
      tc_fence_after();
      if constexpr (AB16) {
#pragma unroll
        for (int i = 0; i < CT; i += 16) {
          float x[16];
          tmem_ld16(tl + T_X + i0 + i, x);
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 b = *reinterpret_cast<const float4*>(ax + AX_G + i0 + i + j);
            const float bb[4] = {-b.x, -b.y, -b.z, -b.w};
            mul2f(x + j, x + j, bb);
            mul2f(x + j + 2, x + j + 2, bb + 2);
          }
          st_split16<AB16>(tl + T_RH + (i0 + i) / 2, tl + T_RL + (i0 + i) / 2, x);
        }
      } else {
#pragma unroll
        for (int i = 0; i < CT; i += 16) {
          float x[16];
          tmem_ld16(tl + T_X + i0 + i, x);
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 b = *reinterpret_cast<const float4*>(ax + AX_G + i0 + i + j);
            const float2 v0 = unpack2<AB16>(v[(i + j) / 2]), v1 = unpack2<AB16>(v[(i + j) / 2 + 1]);
            x[j] = fmaf(-b.x * uS, x[j], v0.x);
            x[j + 1] = fmaf(-b.y * uS, x[j + 1], v0.y);
            x[j + 2] = fmaf(-b.z * uS, x[j + 2], v1.x);
            x[j + 3] = fmaf(-b.w * uS, x[j + 3], v1.y);
          }
          st_split16<1>(tl + T_RH + (i0 + i) / 2, tl + T_RL + (i0 + i) / 2, x);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&S_.r_ready);
      if (!AB16 && BWD && c > 0 && threadIdx.x == 32 * G::CHAIN) {
        bulk_wait_read();  // the chunk before is stored: its stage, and the panel of E, may be written again
        mbar_arrive(&S_.empty[s ^ 1]);
      }
      pipe_wait(&S_.u_full, ph, ab, err, 0x1000);
      tc_fence_after();
      const float gam[2] = {ax[AX_GC], ax[AX_GC]};
      [[maybe_unused]] float uW[2] = {1.f, 1.f};        // float16: what undoes the factor of w beta E
      auto weigh = [&](int i, float* x) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 b = *reinterpret_cast<const float4*>(ax + AX_WB + i0 + i + j);
          const float bb[4] = {b.x, b.y, b.z, b.w};
          mul2f(x + j, x + j, bb);
          mul2f(x + j + 2, x + j + 2, bb + 2);
        }
      };
      if constexpr (AB16) {
#pragma unroll
        for (int i = 0; i < CT; i += 16) {
          float x[16];
          load_e(i, x);
          uint32_t hi[8], lo[8];
          split<AB16, 8>(x, hi, lo);
          tmem_st8(tl + T_RH + (i0 + i) / 2, hi);
          tmem_st8(tl + T_RL + (i0 + i) / 2, lo);
          if (BWD) stage_e(p, i, hi, lo);
          weigh(i, x);
          st_split16<AB16>(tl + T_WH + (i0 + i) / 2, tl + T_WL + (i0 + i) / 2, x);
        }
      } else {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < CT; i += 16) {
          float x[16];
          load_e(i, x);
          st_split16<1>(tl + T_RH + (i0 + i) / 2, tl + T_RL + (i0 + i) / 2, x);
          weigh(i, x);
          m = fmaxf(m, abs_max<16>(x));
        }
        m = warps_max<2, G::CHAIN_WARPS>(m, S_.top[1], cw);
        const Pow2 f = pow2_of(m);
        const float ss[2] = {f.s, f.s};
        uW[0] = uW[1] = f.u;
        bS = fmaf(64.f * ax[AX_KN], m, gam[0] * bS);
#pragma unroll
        for (int i = 0; i < CT; i += 16) {  // E once more rather than kept: registers
          float x[16];
          load_e(i, x);
          weigh(i, x);
#pragma unroll
          for (int j = 0; j < 16; j += 2) mul2f(x + j, x + j, ss);
          st_split16<AB16>(tl + T_WH + (i0 + i) / 2, tl + T_WL + (i0 + i) / 2, x);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&S_.u_ready);
      if constexpr (!AB16 && BWD) {
        float e[16];
        read_e(e);
        token_max_put<CT>(e, S_.etop, i0, quad, lane);  // got below
      }
      constexpr bool LATE = !AB16 && BWD;  // E is staged behind S, with its tokens' factors
      if (!LATE && (!BWD || warp != G::CHAIN)) warp_arrive(&S_.empty[s]);
      if (BWD && !LATE) {
        fence_async_smem();
        bar_sync<2, G::CHAIN_THREADS>();
        if (threadIdx.x == 32 * G::CHAIN) {
          store_panel(&tme, sm + L::OUT, 0, v0, a.V, sh0 + (int64_t)c * a.HV);
          store_panel(&tme, sm + s * L::STAGE + L::V, C, v0, a.V, sh0 + (int64_t)c * a.HV);
        }
      }
      pipe_wait(&S_.d_full, ph, ab, err, 0x2000);
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < KH; i += 16) {
        float x[16];
        tmem_ld16(tl + T_X + KH * hh + i, x);
        if (!AB16) {
#pragma unroll
          for (int j = 0; j < 16; j += 2) mul2f(x + j, x + j, uW);
        }
#pragma unroll
        for (int j = 0; j < 16; j += 2) fma2(S + i + j, gam, S + i + j, x + j);
      }
      if (c + 1 < nch) put_state(p + L::KQ, c + 1);  // every product with the K and Q rows is done: their space is the staging
      if constexpr (LATE) {
        bar_sync_quad<4, 128>(hh);  // the four warps with these tokens
        const Pow2 f = pow2_of(token_max_get(S_.etop, i0 + (lane & (CT - 1))));
        if (quad == 0 && lane < CT) fx[(int64_t)c * a.HV * FX_N + FX_E + i0 + lane] = f.u;
        float e[16];
        read_e(e);
#pragma unroll
        for (int j = 0; j < 16; ++j) e[j] *= __shfl_sync(0xffffffffu, f.s, j);
        uint32_t hi[8], lo[8];
        split<AB16, 8>(e, hi, lo);
        stage_e(p, 0, hi, lo);
        fence_async_smem();
        bar_sync<2, G::CHAIN_THREADS>();
        if (threadIdx.x == 32 * G::CHAIN) {
          store_panel(&tme, sm + L::OUT, 0, v0, a.V, sh0 + (int64_t)c * a.HV);
          store_panel(&tme, sm + s * L::STAGE + L::V, C, v0, a.V, sh0 + (int64_t)c * a.HV);
          if (c + 1 < nch)
            for (int i = 0; i < NP; ++i)
              if (64 * i < a.K)
                store_panel(&tms, sm + s * L::STAGE + L::KQ + 2 * i * PANEL, 64 * i, v0, a.V, sh0 + (int64_t)(c + 1) * a.HV);
        }
        if (warp != G::CHAIN) warp_arrive(&S_.empty[s]);
      }
      if (BWD && !LATE) {
        fence_async_smem();
        bar_sync<2, G::CHAIN_THREADS>();
        if (threadIdx.x == 32 * G::CHAIN) {
          if (c + 1 < nch)
            for (int i = 0; i < NP; ++i)
              if (64 * i < a.K)
                store_panel(&tms, sm + s * L::STAGE + L::KQ + 2 * i * PANEL, 64 * i, v0, a.V, sh0 + (int64_t)(c + 1) * a.HV);
          bulk_wait_read();  // then the stage, and the panel of E, may be written again
          mbar_arrive(&S_.empty[s]);
        }
        bar_sync<2, G::CHAIN_THREADS>();
      }
      if (const int cd = part.c0 + c; BWD && vin && ((cd + 1) % ANCHOR == 0 || cd + 1 == part.nch)) {
        float* g = w.Sf + ((gdr_slot0(a, n, part.doc, C * ANCHOR) + cd / ANCHOR) * a.HV + hv) * a.K * a.V + v0 + vl;
#pragma unroll
        for (int i = 0; i < KH; ++i)
          if (KH * hh + i < a.K) g[(int64_t)(KH * hh + i) * a.V] = S[i];
      }
    }
    if (BWD && threadIdx.x == 32 * G::CHAIN) bulk_wait_all();
    if (!BWD && final && vin) {
#pragma unroll
      for (int i = 0; i < KH; ++i) {
        const int k = KH * hh + i;
        if (k < a.K) final[(int64_t)k * width + v0 + vl] = S[i];
      }
    }
  } else if (!SUM) {
    // ------------------------------------------------------------------ output
    G::out_regs();
    const int quad = warp & 3, j0 = OT * (warp >> 2);  // tokens j0 .. j0 + OT - 1
    const int vl = quad * 32 + lane;
    const uint32_t tl = tb + ((uint32_t)(quad * 32) << 16);
    const int64_t slots = gdr_slots(a, C);
    for (int c = 0; c < nch; ++c) {
      const int s = c & 1, ph = c & 1;
      const int valid = min(C, sq.len - c * C);
      const uint32_t p = sb + s * L::STAGE;
      const float* ax = reinterpret_cast<const float*>(sm + s * L::STAGE + L::AX);
      const int64_t row0 = sq.bos + (int64_t)c * C;
      pipe_wait(&S_.full[s], (c >> 1) & 1, ab, err, 0x4000);
      if (valid < C) {
        // the rows past the document belong to another one: what a product sums over must be zero
        for (int i = 0; i < NP; ++i) zero_rows(p + L::KQ + 2 * i * PANEL, 1, valid, threadIdx.x, G::OUT_THREADS);
        zero_rows(p + L::V, 2, valid, threadIdx.x, G::OUT_THREADS);
        fence_async_smem();
        warp_arrive(&S_.kz);
      }
      float y[OT];
      pipe_wait(&S_.x_full, ph, ab, err, 0x8000);
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < OT; i += 32) tmem_ld32(tl + T_X + 64 + j0 + i, y + i);
      tc_fence_before();
      // the factor was left before S was ready, the phase of which lasts until o1_read of this chunk
      if (!AB16) pipe_wait(&S_.s_ready, ph, ab, err, 0x8000);
      const float uY = AB16 ? 1.f : S_.undo[c & 1];
      warp_arrive(&S_.o1_read);
#pragma unroll
      for (int i = 0; i < OT; i += 4) {
        const float4 b = *reinterpret_cast<const float4*>(ax + AX_SG + j0 + i);
        y[i] *= AB16 ? b.x : b.x * uY;
        y[i + 1] *= AB16 ? b.y : b.y * uY;
        y[i + 2] *= AB16 ? b.z : b.z * uY;
        y[i + 3] *= AB16 ? b.w : b.w * uY;
      }
      pipe_wait(&S_.o_full, ph, ab, err, 0x10000);
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < OT; i += 16) {
        float x[16];
        tmem_ld16(tl + T_D + j0 + i, x);
#pragma unroll
        for (int j = 0; j < 16; j += 2) add2f(y + i + j, y + i + j, x + j);
        tmem_ld16(tl + T_D + 64 + j0 + i, x);
#pragma unroll
        for (int j = 0; j < 16; j += 2) add2f(y + i + j, y + i + j, x + j);
      }
      tc_fence_before();
      warp_arrive(&S_.o2_free);
      if (!BWD) {
        warp_arrive(&S_.empty[s]);
        const uint32_t out = sb + L::OUT;
        if (threadIdx.x == 0) bulk_wait_read();  // the stores of the chunk before have read the tile
        bar_sync<1, G::OUT_THREADS>();
        const Column O(out, vl);
#pragma unroll
        for (int i = 0; i < OT; ++i) sts16(O.at(j0 + i), f2h<AB16>(y[i]));
        if (valid == C && ((uintptr_t)a.o & 15) == 0) {
          fence_async_smem();
          bar_sync<1, G::OUT_THREADS>();
          if (threadIdx.x == 0) {
            tma_store_3d(&tmo, sm + L::OUT, v0, hv, (int)row0);
            if (v0 + 64 < a.V) tma_store_3d(&tmo, sm + L::OUT + PANEL, v0 + 64, hv, (int)row0);
            bulk_commit();
          }
        } else {
          bar_sync<1, G::OUT_THREADS>();
          copy_rows<true>(out, reinterpret_cast<uint16_t*>(a.o), row0, a.HV, hv, a.V, v0, valid, threadIdx.x, G::OUT_THREADS);
        }
      } else {
        const Column D(p + L::DO, vl);
        [[maybe_unused]] float top = 0.f;
#pragma unroll
        for (int i = 0; i < OT; ++i) {
          const float d = j0 + i < valid ? h2f<AB16>(lds16(D.at(j0 + i))) : 0.f;
          if (!AB16) top = fmaxf(top, fabsf(d));
          y[i] = j0 + i < valid ? y[i] * d : 0.f;
        }
        warp_arrive(&S_.empty[s]);
        if (!AB16) {
          top = warp_max(top);
          if (lane == 0) S_.dtop[warp] = top;
        }
        lane_sums<OT>(y, lane);
#pragma unroll
        for (int i = 0; i < OT / 32; ++i) S_.red[quad][j0 + lane * (OT / 32) + i] = y[i];
        bar_sync<1, G::OUT_THREADS>();
        if (threadIdx.x < C) {
          const int i = threadIdx.x;
          w.dotO[((int64_t)vt * slots * a.HV + sh0 + (int64_t)c * a.HV) * C + i] =
              S_.red[0][i] + S_.red[1][i] + S_.red[2][i] + S_.red[3][i];
          if (!AB16 && i == 0) {
#pragma unroll
            for (int o = 1; o < G::OUT_WARPS; ++o) top = fmaxf(top, S_.dtop[o]);
            factors_of(a, w)[((int64_t)vt * slots * a.HV + sh0 + (int64_t)c * a.HV) * FX_N + FX_DO] = top;
          }
        }
        bar_sync<1, G::OUT_THREADS>();
      }
    }
    if (!BWD && threadIdx.x == 0) bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == G::MMA) tmem_dealloc(tb, 512);
}

template <int AB16, int KD, bool BWD, bool SUM>
cudaError_t launch(const GdrArgs& a, const Ws& w) {
  CUtensorMap q, k, v, o, st, e16;
  cudaError_t e = token_map(&q, a, a.q, a.H, a.K);
  if (e == cudaSuccess) e = token_map(&k, a, a.k, a.H, a.K);
  if (e == cudaSuccess) e = token_map(&v, a, a.v, a.HV, a.V);
  // (an o off 16 bytes takes no map; its place is then not used)
  if (e == cudaSuccess) e = token_map(&o, a, BWD ? a.d_o : SUM || ((uintptr_t)a.o & 15) ? a.v : a.o, a.HV, a.V);
  st = e16 = o;  // unused by the forward
  const int64_t sh = gdr_slots(a, C) * a.HV;
  if (BWD && e == cudaSuccess) e = matrix_map(&st, a, w.S0, a.K, sh);
  if (BWD && e == cudaSuccess) e = matrix_map(&e16, a, w.E, 2 * C, sh);
  constexpr uint32_t bytes = Lay<BWD>::BYTES;
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(scan_kernel<AB16, KD, BWD, SUM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return e;
  const int tiles = (a.V + VT - 1) / VT + (SUM ? 1 : 0), segs = SUM ? w.nseg - 1 : w.nseg;
  scan_kernel<AB16, KD, BWD, SUM>
      <<<(unsigned)((int64_t)a.n_seqs * a.HV * segs * tiles), Warps<BWD>::THREADS, bytes, a.stream>>>(q, k, v, o, st, e16, a, w);
  return cudaGetLastError();
}

template <int AB16, int KD>
cudaError_t pick(const GdrArgs& a, const Ws& w, ScanMode mode) {
  if (mode == SCAN_BWD) return launch<AB16, KD, true, false>(a, w);
  return mode == SCAN_SUM ? launch<AB16, KD, false, true>(a, w) : launch<AB16, KD, false, false>(a, w);
}

}  // namespace

cudaError_t scan(const GdrArgs& a, const Ws& w, ScanMode mode, int* launches) {
  ++*launches;
  const bool small = a.K <= 64;
  if (a.dtype == DT_BF16) return small ? pick<1, 64>(a, w, mode) : pick<1, 128>(a, w, mode);
  return small ? pick<0, 64>(a, w, mode) : pick<0, 128>(a, w, mode);
}

}  // namespace gdrtc
}  // namespace ccq
