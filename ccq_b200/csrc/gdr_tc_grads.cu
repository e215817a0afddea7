// Tensor-core path of the gated delta rule, gradients inside a chunk, per (chunk, key head):
//
//   dQ = scale Gam dO S0^T + W K                       W_ij = scale D_ij beta_j (dO E^T)_ij, j <= i
//   dK = -Gam dV S0^T + w beta E dS1^T + W^T Q + (N + N^T) K    N_ij = -D_ij beta_j (dV E^T)_ij, j < i
//   dbeta_j = sum_i scale D_ij (q_i.k_j) (dO E^T)_ij + w_j k_j.(E dS1^T)_j - sum_i D_ij (k_i.k_j) (dV E^T)_ij
//   dg_t = sum_{i >= t} (dO_i . O_i - V_i . dV_i) + <dS, S>, over the tokens up to the next anchor and there
//
// summed over the value heads of the key head in TMEM.  The chunks are independent: persistent blocks
// walk (chunk, key head) items, and an item's (value head, 64 columns of V) steps are loaded by TMA two
// ahead, across items.  The 64-token operands are stacked in pairs to fill the 128 lanes: rows 0-63 carry what
// leads to dK, rows 64-127 what leads to dQ:
//
//   X  = [dV ; dO] S0^T    [128 x K]      P = [dV ; dO] E^T   [128 x 64]     B = [K ; Q] K^T  [128 x 64]
//   X2 = E dS1^T           [64 x K] (its other 64 rows are not read)
//   F  = [-Gam X + w beta X2 ; scale Gam X] + [N ; W] K + [N^T ; 0] K + [W^T ; 0] Q
//
// X, X2, P and B are read by the epilogue warps (P and B first, which are committed before the last X and X2), which put the first term of F back into TMEM and [N ; W]
// into shared memory; the transposed products read the same bytes MN-major, with the other half's lanes
// masked.  60 MMAs an item at V = 128.  Operands are single 16-bit values but for W, and E in P (see
// gdr_tc.cuh).  An item moves 192 KB, which bounds the kernel: 8192 items take 302 us, 5.3 TB/s.  What is not on the
// path from one group of products to the next (statistics, dbeta and dg, waiting for the stores to leave) comes after
// the output, beside the next item's products; with it in front the same items took 368 us.  float16: 425 us, since N and
// W are written only when all of them are known, and so is their factor.
//
// Warps (576 threads): 0-7 epilogue A (P and B), 8-15 epilogue B (X and X2), all of them the output; 16 TMA,
// 17 MMA.
#include "gdr_tc.cuh"

namespace ccq {
namespace gdrtc {
namespace {
using namespace tc;

constexpr int THREADS = 576, EPI = 512;
constexpr uint32_t T_X = 0, T_X2 = 128, T_P = 256, T_B = 320, T_F = 384;
// one step: [dV ; dO] (two panels), E hi and lo, S0 and dS1 (two panels each)
constexpr uint32_t B_DV = 0, B_DO = PANEL, B_E = 2 * PANEL, B_S = 4 * PANEL, B_DS = 6 * PANEL, B_SIZE = 8 * PANEL;
constexpr uint32_t L_KQ = 0;                       // two buffers: K over Q in panels of 128 rows
constexpr uint32_t L_B = 8 * PANEL;                // two steps
constexpr uint32_t L_W = L_B + 2 * B_SIZE;         // N, W and what W's rounding leaves
constexpr uint32_t AX_BYTES = (AX_N * 4 + 127) & ~127u;
constexpr uint32_t L_AX = L_W + 3 * PANEL;            // four
constexpr int RING = 4;

// One value head of an item (float16: 128 of its columns of V, which have factors of their own), written by the TMA
// thread.  Four in a ring: the loads run at most two steps ahead of the products, those one record ahead of the epilogue.
struct Rec {
  int live, hv, h, row0, valid, first, last, qk, more, zero_first;
  int steps, head_first, head_last;  // 64 columns of V each; whether it begins and ends its value head
  int64_t sh, anchor, factors;
};
struct Small {
  uint64_t full[2], empty[2], qk_empty[2];
  uint64_t rec_full[RING];  // the record and its per-token factors
  uint64_t p_full, x_full, wn_ready, f_full, kz, done;
  Rec rec[RING];
  float top[8];  // float16: largest N or W of each warp of epilogue A
  int apart;     // float16: N and W have factors of their own
  float ke[2][C], db[4][C], dg[17];
  uint32_t tmem;
  int go, abort;
};
constexpr uint32_t L_SMALL = L_AX + RING * AX_BYTES;
constexpr uint32_t BYTES = L_SMALL + sizeof(Small) + 1024;
static_assert(BYTES <= 232448, "shared memory");

template <int AB16, int KD>
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
  constexpr int NP = KD / 64;
  const int group = a.HV / a.H, nvt = (a.V + 63) / 64, parts = AB16 ? 1 : (a.V + VT - 1) / VT;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S_.full[i], 1);
      mbar_init(&S_.empty[i], 1);
      mbar_init(&S_.qk_empty[i], 1);
    }
    for (int i = 0; i < RING; ++i) mbar_init(&S_.rec_full[i], 1);
    mbar_init(&S_.p_full, 1);
    mbar_init(&S_.x_full, 1);
    mbar_init(&S_.wn_ready, EPI / 32);
    mbar_init(&S_.f_full, 1);
    mbar_init(&S_.kz, EPI / 32);
    mbar_init(&S_.done, 1);
    S_.abort = 0;
    fence_barrier_init();
  }
  if (warp == 17) tmem_alloc(&S_.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tb = S_.tmem;
  volatile int* ab = &S_.abort;
  int* err = w.err;

  if (warp == 16) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      const int items = (int)(gdr_slots(a, C) * a.H);
      int step = 0, rec = 0, count = 0;
      bool ok = true;
      for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
        const int slot = item / a.H, h = item - slot * a.H;
        int n, c;
        Seq sq;
        if (!gdr_slot_find(a, slot, C, &n, &c, &sq)) continue;
        const int row = (int)(sq.bos + (int64_t)c * C), nch = (sq.len + C - 1) / C;
        for (int part = 0; part < group * parts && ok; ++part, ++rec) {
          const int g = part / parts, vt0 = part % parts * (VT / 64), hv = h * group + g, r = rec % RING;
          const int64_t sh = (int64_t)slot * a.HV + hv;
          const int vt1 = AB16 ? nvt : min(nvt, vt0 + VT / 64);
          for (int vt = vt0; vt < vt1; ++vt, ++step) {
            const int b = step & 1;
            const bool begin = part == 0 && vt == 0;
            if (step >= 2 && !pipe_wait(&S_.empty[b], ((step - 2) >> 1) & 1, ab, err, 1)) { ok = false; break; }
            if (begin && count >= 2 && !pipe_wait(&S_.qk_empty[count & 1], ((count - 2) >> 1) & 1, ab, err, 2)) {
              ok = false;
              break;
            }
            if (*ab) { ok = false; break; }
            uint64_t* bar = &S_.full[b];
            uint8_t* p = sm + L_B + b * B_SIZE;
            mbar_arrive_expect_tx(bar, 2 * NP * PANEL + 4 * PANEL + (begin ? 2 * NP * PANEL : 0));
            if (vt == vt0) {
              Rec& R = S_.rec[r];
              R.live = 1;
              R.hv = hv;
              R.h = h;
              R.row0 = row;
              R.valid = min(C, sq.len - c * C);
              R.first = part == 0;
              R.last = part == group * parts - 1;
              if (!AB16) {
                R.steps = vt1 - vt0;
                R.head_first = vt0 == 0;
                R.head_last = vt1 == nvt;
                R.factors = vt0 / (VT / 64) * gdr_slots(a, C) * a.HV + sh;
              }
              R.qk = count & 1;
              R.more = min(ANCHOR - 1 - c % ANCHOR, nch - 1 - c);
              R.zero_first = c == 0 && a.initial_state == nullptr;
              R.sh = sh;
              R.anchor = (gdr_slot0(a, n, sq, C * ANCHOR) + c / ANCHOR) * a.HV + hv;
              mbar_arrive_expect_tx(&S_.rec_full[r], AX_N * 4);
              bulk_load(sm + L_AX + r * AX_BYTES, w.aux + sh * AX_N, AX_N * 4, &S_.rec_full[r]);
              if (begin) {
                uint8_t* d = sm + L_KQ + (count & 1) * 4 * PANEL;
                for (int i = 0; i < NP; ++i) {
                  tma_load_3d(d + 2 * i * PANEL, &tmk, bar, 64 * i, h, row);
                  tma_load_3d(d + (2 * i + 1) * PANEL, &tmq, bar, 64 * i, h, row);
                }
              }
            }
            tma_load_3d(p + B_DV, &tmdv, bar, 64 * vt, hv, row);
            tma_load_3d(p + B_DO, &tmo, bar, 64 * vt, hv, row);
            tma_load_3d(p + B_E, &tme, bar, 0, 64 * vt, (int)sh);
            tma_load_3d(p + B_E + PANEL, &tme, bar, C, 64 * vt, (int)sh);
            for (int i = 0; i < NP; ++i) {
              tma_load_3d(p + B_S + i * PANEL, &tms, bar, 64 * i, 64 * vt, (int)sh);
              tma_load_3d(p + B_DS + i * PANEL, &tmds, bar, 64 * i, 64 * vt, (int)sh);
            }
          }
        }
        ++count;
      }
      // never leave the block with copies in flight; then the end, for the others
      for (int i = (step > 2 ? step - 2 : 0); i < step; ++i) own_copy_wait(&S_.full[i & 1], (i >> 1) & 1, ab, err, 4);
      for (int i = (rec > RING ? rec - RING : 0); i < rec; ++i)
        own_copy_wait(&S_.rec_full[i % RING], (i / RING) & 1, ab, err, 4);
      if (ok) {
        S_.rec[rec % RING].live = 0;
        mbar_arrive(&S_.rec_full[rec % RING]);
      }
    }
  } else if (warp == 17) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t id_x = idesc_f16(128, KD, AB16, 0, 1), id_x2 = idesc_f16(128, KD, AB16, 1, 1);
      const uint32_t id_p = idesc_f16(128, 64, AB16, 0, 1), id_b = idesc_f16(128, 64, AB16, 0, 0);
      const uint32_t W = sb + L_W;
      int step = 0, zeroed = 0;
      for (int rec = 0;; ++rec) {
        const int r = rec % RING;
        if (!spin_wait(&S_.rec_full[r], (rec / RING) & 1, ab, err, 8)) break;
        const Rec& R = S_.rec[r];
        if (!R.live) break;
        const uint32_t KQ = sb + L_KQ + R.qk * 4 * PANEL;
        bool ok = true;
        const int steps = AB16 ? nvt : R.steps;
        for (int vt = 0; vt < steps; ++vt, ++step) {
          const int b = step & 1;
          const uint32_t p = sb + L_B + b * B_SIZE;
          if (!spin_wait(&S_.full[b], (step >> 1) & 1, ab, err, 0x10)) { ok = false; break; }
          if (vt == 0 && R.first && R.valid < C) {
            if (!spin_wait(&S_.kz, zeroed & 1, ab, err, 0x20)) { ok = false; break; }
            ++zeroed;
          }
          tc_fence_after();
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              umma(tb + T_P, sdesc(p + B_DV + ks * 32, 16, 1024), sdesc(p + B_E + x * PANEL + ks * 2048, PANEL, 1024), id_p,
                   vt + x + ks > 0);
          if (vt == 0) {
#pragma unroll
            for (int ks = 0; ks < KD / 16; ++ks) {
              const uint64_t d = sdesc(KQ + (ks >> 2) * 2 * PANEL + (ks & 3) * 32, 16, 1024);
              umma(tb + T_B, d, d, id_b, ks > 0);
            }
          }
          if (vt == steps - 1) umma_commit(&S_.p_full);  // epilogue A starts on these, beside the products below
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma(tb + T_X, sdesc(p + B_DV + ks * 32, 16, 1024), sdesc(p + B_S + ks * 2048, PANEL, 1024), id_x, vt + ks > 0);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma(tb + T_X2, sdesc(p + B_E + ks * 2048, PANEL, 1024), sdesc(p + B_DS + ks * 2048, PANEL, 1024), id_x2, vt + ks > 0);
          umma_commit(&S_.empty[b]);
        }
        if (!ok) break;
        umma_commit(&S_.x_full);
        if (!spin_wait(&S_.wn_ready, rec & 1, ab, err, 0x40)) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          umma(tb + T_F, sdesc(W + ks * 32, 16, 1024), sdesc(KQ + ks * 2048, 2 * PANEL, 1024), id_x, 1);
        const bool apart = !AB16 && S_.apart;  // the third panel is W for the transposed product, else W's second part
#pragma unroll
        for (int ks = 0; ks < 4 && !apart; ++ks)
          umma_masked(tb + T_F, sdesc(W + PANEL + ks * 32, 16, 1024), sdesc(KQ + ks * 2048, 2 * PANEL, 1024), id_x, 1, ~0u, 0);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          umma_masked(tb + T_F, sdesc(W + ks * 2048, PANEL, 1024), sdesc(KQ + ks * 2048, 2 * PANEL, 1024), id_x2, 1, 0, ~0u);
#pragma unroll
        for (int x = 1; x < 3; ++x)
#pragma unroll
          for (int ks = 0; ks < 4 && !(apart && x == 1); ++ks)
            umma_masked(tb + T_F, sdesc(W + x * PANEL + ks * 2048, 0, 1024), sdesc(KQ + PANEL + ks * 2048, 2 * PANEL, 1024), id_x2, 1, 0,
                        ~0u);
        umma_commit(&S_.f_full);
      }
      umma_commit(&S_.done);  // TMEM is freed only after every issued MMA has completed
      mbar_wait(&S_.done, 0);
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const int quad = warp & 3;
    const bool kside = quad < 2;          // rows 0-63: what leads to dK
    const int i = (quad & 1) * 32 + lane; // token
    const uint32_t tl = tb + ((uint32_t)(quad * 32) << 16);
    int stored = -1;
    int first_step = 0, steps = 0;        // step of this record's first loads, and how many it has
    // float16: the factors of F's rows 0-63 (with N, and W for its transpose) and 64-127 (with W), and whether they
    // differ in this record; this token's dbeta from the columns before
    [[maybe_unused]] float sN = 1.f, sW = 1.f, head_db = 0.f;
    [[maybe_unused]] bool apart = false;
    for (int rec = 0;; ++rec, first_step += AB16 ? nvt : steps) {
      const int r = rec % RING;
      const Rec& R = S_.rec[r];
      // one decision for all warps, so that a wait that gave up cannot leave some of them at a barrier
      if (tid == 0) S_.go = pipe_wait(&S_.rec_full[r], (rec / RING) & 1, ab, err, 0x80) && R.live;
      bar_sync<1, EPI>();
      if (tid == 256 && stored >= 0) {  // the last item's output has left its buffer
        bulk_wait_read();
        mbar_arrive(&S_.qk_empty[stored]);
      }
      stored = -1;
      if (!S_.go) break;
      const int valid = R.valid;
      if (!AB16) steps = R.steps;
      const uint32_t KQ = sb + L_KQ + R.qk * 4 * PANEL;
      const float* ax = reinterpret_cast<const float*>(sm + L_AX + r * AX_BYTES);
      if (valid < C && R.first) {
        pipe_wait(&S_.full[first_step & 1], (first_step >> 1) & 1, ab, err, 0x100);
        // the rows past the document belong to another one: what a product sums over must be zero
        for (int p = 0; p < 2 * NP; ++p) zero_rows(KQ + p * PANEL, 1, valid, tid, EPI);
        fence_async_smem();
        warp_arrive(&S_.kz);
      }
      // float16: what undoes the factors of X's and X2's rows, and of P's columns (one a lane)
      [[maybe_unused]] float uX = 1.f, uX2 = 1.f, uP = 1.f, uRow = 1.f;
      if constexpr (!AB16) {
        const float* f = factors_of(a, w) + R.factors * FX_N;
        uRow = kside ? f[FX_DV + i] : 1.f;
        if (warp < 8) {
          uP = f[FX_E + 32 * (warp >> 2) + lane];
        } else {
          uX = uRow * f[FX_S];
          uX2 = f[FX_E + i] * f[FX_DS];
        }
      }
      // and, once the epilogue's first half has N and W, their factors: every warp passes here once a record.  They are one,
      // and W is hi + lo, unless N is 4096 times W or more.  Inside an item they only fall, so that what is in F already
      // stays in range.
      [[maybe_unused]] float turn = 1.f, sF = 1.f;
      [[maybe_unused]] auto factors = [&] {
        bar_sync<1, EPI>();
        const float n = fmaxf(fmaxf(S_.top[0], S_.top[1]), fmaxf(S_.top[4], S_.top[5]));
        const float t = fmaxf(fmaxf(S_.top[2], S_.top[3]), fmaxf(S_.top[6], S_.top[7]));
        const float before = kside ? sN : sW;
        sN = fminf(pow2_of(fmaxf(n, t)).s, R.first ? 0x1p40f : sN);
        sW = fminf(pow2_of(t).s, R.first ? 0x1p40f : sW);
        apart = sW > 4096.f * sN;
        if (!apart) sW = sN;
        if (tid == 0) S_.apart = apart;
        sF = kside ? sN : sW;
        turn = sF / before;
      };
      pipe_wait(warp < 8 ? &S_.p_full : &S_.x_full, rec & 1, ab, err, 0x200);
      tc_fence_after();
      float z[32];
      if (warp < 8) {
        // [N ; W] and the scores' part of dbeta, columns c0 .. c0 + 31
        const int c0 = 32 * (warp >> 2);
        const uint32_t row = sb + L_W + (kside ? 0 : PANEL);
        const bool above = c0 > (quad & 1) * 32;  // the block above the diagonal
        auto zero = [&] {
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) {
            sts128(row + sw128(i, c0 / 8 + cc), make_uint4(0, 0, 0, 0));
            if (!kside) sts128(row + PANEL + sw128(i, c0 / 8 + cc), make_uint4(0, 0, 0, 0));
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) z[e] = 0.f;
        };
        if constexpr (AB16) {
          if (above) {
            zero();
          } else {
            const float gh[2] = {ax[AX_GH + i], ax[AX_GH + i]}, gl[2] = {ax[AX_GL + i], ax[AX_GL + i]};
            const float sx[2] = {kside ? -1.f : a.scale, kside ? -1.f : a.scale}, m1[2] = {-1.f, -1.f};
            const int top = i < valid ? (kside ? i - 1 : i) : -1;  // last column of this row
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) {
              float x[8], y[8];
              tmem_ld8x2(tl + T_P + c0 + 8 * cc, tl + T_B + c0 + 8 * cc, x, y);
#pragma unroll
              for (int e = 0; e < 8; e += 2) {
                const int j = c0 + 8 * cc + e;
                float d[2], l[2];
                fma2(d, ax + AX_GH + j, m1, gh);
                fma2(l, ax + AX_GL + j, m1, gl);
                add2f(d, d, l);
                d[0] = ex2(d[0]);
                d[1] = ex2(d[1]);
                mul2f(x + e, x + e, sx);
                mul2f(d, d, x + e);
                d[0] = j <= top ? d[0] : 0.f;  // the masked places can hold anything
                d[1] = j < top ? d[1] : 0.f;
                mul2f(z + 8 * cc + e, d, y + e);
                mul2f(x + e, d, ax + AX_B + j);
              }
              uint32_t u[4], lo[4];
              split<AB16, 4>(x, u, lo);
              sts128(row + sw128(i, c0 / 8 + cc), make_uint4(u[0], u[1], u[2], u[3]));
              if (!kside) sts128(row + PANEL + sw128(i, c0 / 8 + cc), make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
          }
        } else {
          float m = 0.f;
          if (above) {
            zero();
          } else {
            const int top = i < valid ? (kside ? i - 1 : i) : -1;
            const float gh = ax[AX_GH + i], gl = ax[AX_GL + i], sx = kside ? -uRow : a.scale;
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) {
              float* d = z + 8 * cc;
              tmem_ld8(tl + T_P + c0 + 8 * cc, d);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int j = c0 + 8 * cc + e;
                d[e] *= ex2((gh - ax[AX_GH + j]) + (gl - ax[AX_GL + j])) * (sx * __shfl_sync(0xffffffffu, uP, 8 * cc + e));
                d[e] = j <= top ? d[e] : 0.f;  // the masked places can hold anything
                m = fmaxf(m, fabsf(d[e] * ax[AX_B + j]));
              }
            }
          }
          m = warp_max(m);
          if (lane == 0) S_.top[warp] = m;
          factors();
          if (!above) {
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) {
              float x[8], y[8];
              uint32_t u[4];
              tmem_ld8(tl + T_B + c0 + 8 * cc, y);
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = z[8 * cc + e] * ax[AX_B + c0 + 8 * cc + e];
#pragma unroll
              for (int e = 0; e < 8; ++e) z[8 * cc + e] *= y[e];
              uint32_t lo[4];
              float xs[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) xs[e] = x[e] * sF;
              split<AB16, 4>(xs, u, lo);
              sts128(row + sw128(i, c0 / 8 + cc), make_uint4(u[0], u[1], u[2], u[3]));
              if (!kside) {
                if (apart) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) lo[e] = pack2<AB16>(x[2 * e] * sN, x[2 * e + 1] * sN);
                }
                sts128(row + PANEL + sw128(i, c0 / 8 + cc), make_uint4(lo[0], lo[1], lo[2], lo[3]));
              }
            }
          }
        }
      } else {
        // the first term of F, half of its columns, and k_i . X2_i
        constexpr int KH = KD / 2;
        const int hf = (warp - 8) >> 2;
        float r0 = kside ? -ax[AX_G + i] : ax[AX_SG + i], r1 = ax[AX_WB + i];
        if constexpr (!AB16) {
          factors();
          r0 *= uX * sF;
          r1 *= uX2 * sF;
        }
        const float g0[2] = {r0, r0}, g1[2] = {r1, r1};
        float ke[2] = {0.f, 0.f};
#pragma unroll
        for (int k0 = 0; k0 < KH; k0 += 16) {
          const int k = KH * hf + k0;
          float x[16];
          if (kside) {
            float y[16];
            tmem_ld16x2(tl + T_X + k, tl + T_X2 + k, x, y);
            const uint32_t p = KQ + (k >> 6) * 2 * PANEL;
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              const uint4 kv = lds128(p + sw128(i, ((k & 63) >> 3) + cc));
              const uint32_t u[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2<AB16>(u[e]);
                const float f2[2] = {f.x, f.y};
                fma2(ke, f2, y + 8 * cc + 2 * e, ke);
              }
            }
#pragma unroll
            for (int e = 0; e < 16; e += 2) mul2f(y + e, y + e, g1);
#pragma unroll
            for (int e = 0; e < 16; e += 2) fma2(x + e, x + e, g0, y + e);
          } else {
            tmem_ld16(tl + T_X + k, x);
#pragma unroll
            for (int e = 0; e < 16; e += 2) mul2f(x + e, x + e, g0);
          }
          if (!R.first) {
            float y[16];
            tmem_ld16(tl + T_F + k, y);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = AB16 ? x[e] + y[e] : fmaf(y[e], turn, x[e]);
          }
          uint32_t u[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(x[e]);
          tmem_st8(tl + T_F + k, u);
          tmem_st8(tl + T_F + k + 8, u + 8);
        }
        if (kside) S_.ke[hf][i] = AB16 ? ke[0] + ke[1] : (ke[0] + ke[1]) * uX2;
        tmem_st_wait();
      }
      fence_async_smem();
      tc_fence_before();
      warp_arrive(&S_.wn_ready);
      // dO . O - V . dV: of this chunk's tokens in warps 0 and 1, of the chunks up to the next anchor in the
      // others; and <dS, S> there.  Asked for here, used after the output.
      const int64_t vs = gdr_slots(a, C) * a.HV, va = gdr_slots(a, C * ANCHOR) * a.HV;
      const int64_t at_dot = (R.sh + (int64_t)(tid >> 6) * a.HV) * C + (tid & 63), at_later = R.anchor * ANCHOR_PARTS + tid;
      const bool has_dot = (tid >> 6) <= R.more, has_later = tid < ANCHOR_PARTS;
      float dot = has_dot ? w.dotO[at_dot] : 0.f, dotV = has_dot ? w.dotV[at_dot] : 0.f, later = has_later ? w.anchor[at_later] : 0.f;
      if (warp < 8) {
        lane_sums<32>(z, lane);
        S_.db[quad][32 * (warp >> 2) + lane] = z[0];
      }
      pipe_wait(&S_.f_full, rec & 1, ab, err, 0x400);
      tc_fence_after();
      if (R.last) {
        // dK over the K rows and dQ over the Q rows, then out
        constexpr int KQTR = KD / 4;
        [[maybe_unused]] const float back = 1.f / sF;
        const int k0 = KQTR * (warp >> 2);
#pragma unroll
        for (int k = k0; k < k0 + KQTR; k += 16) {
          float x[16];
          tmem_ld16(tl + T_F + k, x);
          uint32_t u[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) u[e] = AB16 ? pack2<AB16>(x[2 * e], x[2 * e + 1]) : pack2<AB16>(x[2 * e] * back, x[2 * e + 1] * back);
          const uint32_t p = KQ + (k >> 6) * 2 * PANEL;
          sts128(p + sw128(quad * 32 + lane, (k & 63) >> 3), make_uint4(u[0], u[1], u[2], u[3]));
          sts128(p + sw128(quad * 32 + lane, ((k & 63) >> 3) + 1), make_uint4(u[4], u[5], u[6], u[7]));
        }
        fence_async_smem();
        bar_sync<1, EPI>();
        if (valid == C) {
          if (tid == 256) {
            for (int p = 0; p < NP; ++p)
              if (64 * p < a.K) {
                tma_store_3d(&tmdk, sm + (KQ - sb) + 2 * p * PANEL, 64 * p, R.h, R.row0);
                tma_store_3d(&tmdq, sm + (KQ - sb) + (2 * p + 1) * PANEL, 64 * p, R.h, R.row0);
              }
            bulk_commit();
          }
          stored = R.qk;
        } else {
          for (int e = tid; e < valid * 2 * NP * 8; e += EPI) {
            const int t = e / (2 * NP * 8), x = e % (2 * NP * 8), which = x & 1, ch = x >> 1;
            if (ch * 8 < a.K)
              *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(which ? a.dq : a.dk) +
                                        ((int64_t)(R.row0 + t) * a.H + R.h) * a.K + ch * 8) =
                  lds128(KQ + ((ch >> 3) * 2 + which) * PANEL + sw128(t, ch & 7));
          }
          bar_sync<1, EPI>();
          if (tid == 0) mbar_arrive(&S_.qk_empty[R.qk]);
        }
      }
      dot -= dotV;
      for (int v = 1; v < (a.V + VT - 1) / VT; ++v) {
        if (has_dot) dot += w.dotO[v * vs * C + at_dot] - w.dotV[v * vs * C + at_dot];
        if (has_later) later += w.anchor[v * va * ANCHOR_PARTS + at_later];
      }
      {
        const float x = warp_sum(warp < 2 ? later : dot + later);
        if (lane == 0) S_.dg[warp] = x;
      }
      bar_sync<1, EPI>();
      if (warp < 2) {
        const int j = tid;
        const int64_t at = (int64_t)(R.row0 + j) * a.HV + R.hv;
        float db = S_.db[0][j] + S_.db[1][j] + S_.db[2][j] + S_.db[3][j] + ax[AX_W + j] * (S_.ke[0][j] + S_.ke[1][j]);
        if constexpr (!AB16) {
          if (!R.head_first) db += head_db;
          head_db = db;
        }
        if (j < valid && (AB16 || R.head_last)) gate_store(a.dbeta, a.beta_dtype, at, db);
        // dg: reverse running sum; warp 1 holds tokens 32..63, whose sum warp 0 adds
        float x = dot;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float u = __shfl_down_sync(0xffffffffu, x, o);
          if (lane + o < 32) x += u;
        }
        if (lane == 0 && warp == 1) S_.dg[16] = x;
        bar_sync<2, 64>();
        float rest = S_.dg[lane & 15];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
        x += rest + (warp == 0 ? S_.dg[16] : 0.f);
        // nothing decays at the first token of a document that starts from a zero state
        if (j == 0 && R.zero_first) x = 0.f;
        if (j < valid && (AB16 || R.head_last)) gate_store(a.dg, a.g_dtype, at, x);
      }
    }
    if (tid == 256) bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 17) tmem_dealloc(tb, 512);
}

template <int AB16, int KD>
cudaError_t launch(const GdrArgs& a, const Ws& w) {
  const int64_t slots = gdr_slots(a, C), sh = slots * a.HV;
  CUtensorMap q, k, o, dv, e, s, ds, dq, dk;
  cudaError_t r = token_map(&q, a, a.q, a.H, a.K);
  if (r == cudaSuccess) r = token_map(&k, a, a.k, a.H, a.K);
  if (r == cudaSuccess) r = token_map(&o, a, a.d_o, a.HV, a.V);
  if (r == cudaSuccess) r = token_map(&dv, a, AB16 ? a.dv : scaled_dv_of(a, w), a.HV, a.V);
  if (r == cudaSuccess) r = matrix_map(&e, a, w.E, 2 * C, sh);
  if (r == cudaSuccess) r = matrix_map(&s, a, w.S0, a.K, sh);
  if (r == cudaSuccess) r = matrix_map(&ds, a, w.dS1, a.K, sh);
  if (r == cudaSuccess) r = token_map(&dq, a, a.dq, a.H, a.K);
  if (r == cudaSuccess) r = token_map(&dk, a, a.dk, a.H, a.K);
  if (r == cudaSuccess) r = cudaFuncSetAttribute(grads_kernel<AB16, KD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)BYTES);
  if (r != cudaSuccess) return r;
  const int64_t items = slots * a.H;
  const unsigned grid = (unsigned)(items < 148 ? items : 148);  // one persistent block per SM
  grads_kernel<AB16, KD><<<grid, THREADS, BYTES, a.stream>>>(q, k, o, dv, e, s, ds, dq, dk, a, w);
  return cudaGetLastError();
}

}  // namespace

cudaError_t grads(const GdrArgs& a, const Ws& w, int* launches) {
  ++*launches;
  const bool small = a.K <= 64;
  if (a.dtype == DT_BF16) return small ? launch<1, 64>(a, w) : launch<1, 128>(a, w);
  return small ? launch<0, 64>(a, w) : launch<0, 128>(a, w);
}

}  // namespace gdrtc
}  // namespace ccq
