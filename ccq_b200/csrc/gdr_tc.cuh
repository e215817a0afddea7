// Gated delta rule, tensor-core path: what its kernels share.  bf16 or fp16, K a multiple of 8 up to
// 128, V a multiple of 8, 16-byte aligned tensors; chunks of 64 tokens.  Formulas: gdr.h.
//
//   prep   (gdr_tc_prep.cu)   per (chunk, value head): T and P and the per-token factors, to the workspace
//   scan   (gdr_tc_scan.cu)   per (document, value head, 128 columns of V): the state, chunk by chunk
//   rscan  (gdr_tc_rscan.cu)  the same in reverse for the state's gradient
//   grads  (gdr_tc_grads.cu)  per (chunk, key head): dq, dk, dg, dbeta
//   join   (gdr_tc_seg.cu)    long documents of few heads, walked in segments side by side
//
// Precision.  The tensor cores multiply 16-bit operands.  What enters as an operand of the two scans and is
// not an input (S, E, T, P and their gradients' counterparts) is given as a sum of two 16-bit numbers,
// hi + lo, which keeps 2^-17 of it: the state and its gradient then stay at fp32 accuracy over any number
// of chunks (measured 4e-6 against 64 bits), as they would not with one rounding each (2.4e-3).  The
// products cost two or three MMAs instead of one; the scans are bound by the latency of one chunk's
// chain of three products, not by the MMA rate.  The gradient kernel, whose outputs are
// rounded to 16 bits next and feed no recurrence, uses single 16-bit operands but for E where it makes W
// and for W: each of these roundings alone left 1.6e-3 in dq and dk, as much as the outputs' own.
//
// Range.  bfloat16 has float's exponents; float16 ends at 65504 and its hi + lo loses bits below 2^-8, while states and
// gradients are fp32 of any size.  For float16 inputs, therefore:
//   * a product without an input (R T, E P beta, dE T) has bfloat16 operands;
//   * an operand that meets an input has to be float16.  It is multiplied by a power of two that puts its largest value,
//     or a bound on it, into [2^14, 2^15) (pow2_of; hi + lo then keeps 2^-22 of every value down to 2^-22 of the largest),
//     and the product's fp32 sums by the inverse.
//     "Its" means of a chunk and 128 columns of V, for the stored E and dV also of a token, for N and W of a chunk.
// Operands that share an accumulator would have to share the factor, so float16 forms R = V - Gam K S0 before the
// product with T, reads the two products of dS one after the other, and takes the gradient kernel's V in tiles of 128
// columns; W, the one operand of two sums there, takes N's factor with it, or where N is far larger one for each sum.
#pragma once

#include "gdr.h"

namespace ccq {
namespace gdrtc {

constexpr int C = 64;             // tokens per chunk
constexpr int VT = 128;           // columns of V per block of the scans (TMEM lanes)
constexpr uint32_t PANEL = 64 * 128;        // 64 rows of 128 bytes, 128-byte swizzle
constexpr uint32_t TILE = 2 * PANEL;        // 64 rows x 128 columns
constexpr uint32_t MATS = 4 * PANEL;        // T hi, T lo, P beta hi, P beta lo: 64 x 64 each, swizzled as in shared memory
// float16: these in bfloat16, then P beta hi, lo in float16 with a factor, for the product with dO
__host__ __device__ constexpr uint32_t mats_bytes(bool bf16) { return bf16 ? MATS : MATS + 2 * PANEL; }
// per (chunk, value head) floats, 64 tokens each: Gam, scale Gam, w beta, beta, w, G (hi and lo part); then Gam_C
constexpr int AX_G = 0, AX_SG = 64, AX_WB = 128, AX_B = 192, AX_W = 256, AX_GH = 320, AX_GL = 384, AX_GC = 448, AX_N = 456;
// float16 only: what undoes the factor of P beta; bounds on |k| and |q| of the chunk's tokens; the largest |scale| Gam
constexpr int AX_UP = 449, AX_KN = 450, AX_QN = 451, AX_SM = 452;
// float16 only, per (V tile, chunk, value head): what undoes the factors of E and dV, by token, and of S0 and dS1; the
// largest |dO|
constexpr int FX_E = 0, FX_DV = 64, FX_S = 128, FX_DS = 129, FX_DO = 130, FX_N = 132;

// <dS, S> at a chunk's end, which every dg of the chunk holds, is the sum of the later tokens' dO . O - V . dV
// plus its value at a later place.  Both dot products are kept to fp32, and every ANCHOR chunks <dS, S>
// itself is formed from fp32 states, so that neither the 16-bit copies of the states (which left 5e-3 in
// dg) nor a long document's sum of rounding errors gets into dg.
constexpr int ANCHOR = 8;

// Workspace regions; every kernel indexes them by sh = slot * HV + value head.
struct Ws {
  int* err;            // word 0: device error code of the scans
  const int* order;    // launch slot -> document of a packed batch, longest first; nullptr: as they come
  uint8_t* mats;       // [slots * HV][mats_bytes]
  float* aux;          // [slots * HV][AX_N]
  // Few heads, a long axis: documents are cut into nseg segments of seg_chunks chunks (a multiple of ANCHOR),
  // which run side by side once the states at their starts are known (gdr_tc_seg.cu).  Index s * heads + head,
  // heads = n_seqs * HV.
  int nseg, seg_chunks;
  float* Sin;          // [nseg][heads][K][V] state at a segment's start
  float* Bs;           // [nseg][heads][K][V] its end from a zero (first: the given) state; backwards: its start's gradient
  float* Ms;           // [nseg][heads][K][K] its end as a linear map of its start
  float* dSend;        // [nseg][heads][K][V] gradient of the state at a segment's end (backward)
  // backward only
  uint16_t* S0;        // [slots * HV][V][K] state before the chunk, transposed, 16-bit
  uint16_t* dS1;       // [slots * HV][V][K] gradient of the state after it
  uint16_t* E;         // [slots * HV][V][2 C] E transposed: hi part, then lo part; float16: then factors and dVs (below)
  float* dotO;         // [V tiles][slots * HV][C]: dO . O
  float* dotV;         // [V tiles][slots * HV][C]: V . dV
  float* Sf;           // [slots of 512 * HV][K][V] fp32 state after every ANCHOR chunks and after the last one
  float* anchor;       // [V tiles][slots of 512 * HV][16]: <dS, S> there, one part per chain warp
};

// float16 only: [V tiles][slots * HV][FX_N] behind E, and dV times its factors, as dv, behind that.  Not members of Ws:
// past 128 bytes of it the compiler keeps the arguments in fewer registers and the bfloat16 kernels lose 2 to 5 %.
__host__ __device__ inline float* factors_of(const GdrArgs& a, const Ws& w) {
  return reinterpret_cast<float*>(w.E + ((gdr_slots(a, C) * a.HV * 2 * C * a.V + 127) & ~int64_t(127)));
}
__host__ __device__ inline uint16_t* scaled_dv_of(const GdrArgs& a, const Ws& w) {
  const int64_t n = (a.V + VT - 1) / VT * gdr_slots(a, C) * a.HV * FX_N;
  return reinterpret_cast<uint16_t*>(factors_of(a, w) + ((n + 63) & ~int64_t(63)));
}

cudaError_t prep(const GdrArgs& a, const Ws& w, int* launches);
enum ScanMode { SCAN_FWD, SCAN_BWD, SCAN_SUM };  // output; for the backward; a segment's end state only
cudaError_t scan(const GdrArgs& a, const Ws& w, ScanMode mode, int* launches);
cudaError_t rscan(const GdrArgs& a, const Ws& w, bool sum, int* launches);
// the states at the segments' starts from their summaries; backwards, the gradients at their ends
cudaError_t join(const GdrArgs& a, const Ws& w, bool reverse, int* launches);
int plan_segments(const GdrArgs& a, int* seg_chunks);
cudaError_t grads(const GdrArgs& a, const Ws& w, int* launches);

}  // namespace gdrtc
}  // namespace ccq

#ifdef __CUDACC__
#include "tc_common.cuh"
#include "tma_host.h"

namespace ccq {
namespace gdrtc {

// 2^x by the hardware's approximation (2 ulp; below 2^-126 it is zero, as it may be for a decay)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ void fma2(float* d, const float* a, const float* b, const float* c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair(a[0], a[1])), "l"(pair(b[0], b[1])), "l"(pair(c[0], c[1])));
  unpair(r, d[0], d[1]);
}
__device__ __forceinline__ void add2f(float* d, const float* a, const float* b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair(a[0], a[1])), "l"(pair(b[0], b[1])));
  unpair(r, d[0], d[1]);
}
__device__ __forceinline__ void mul2f(float* d, const float* a, const float* b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair(a[0], a[1])), "l"(pair(b[0], b[1])));
  unpair(r, d[0], d[1]);
}

// 2 n values as n packed hi words and n packed lo words
template <int AB16, int N>
__device__ __forceinline__ void split(const float* x, uint32_t* hi, uint32_t* lo) {
  const float m1[2] = {-1.f, -1.f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    hi[i] = tc::pack2<AB16>(x[2 * i], x[2 * i + 1]);
    const float2 f = tc::unpack2<AB16>(hi[i]);
    const float h[2] = {f.x, f.y};
    float r[2];
    fma2(r, h, m1, x + 2 * i);
    lo[i] = tc::pack2<AB16>(r[0], r[1]);
  }
}

// 16 fp32 values of this thread's lane as 8 packed columns at hi and 8 at lo
template <int AB16>
__device__ __forceinline__ void st_split16(uint32_t hi_addr, uint32_t lo_addr, const float* x) {
  uint32_t hi[8], lo[8];
  split<AB16, 8>(x, hi, lo);
  tc::tmem_st8(hi_addr, hi);
  tc::tmem_st8(lo_addr, lo);
}

// 8 and 16 consecutive fp32 columns of this thread's lane
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float* v) {
  uint32_t r[8];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// a power of two that takes a largest value of m to [2^14, 2^15), and its inverse (m below 2^-60 counts as that, so
// that products of factors stay finite)
struct Pow2 {
  float s, u;
};
__device__ __forceinline__ Pow2 pow2_of(float m) {
  const int e = max((int)(__float_as_uint(m) >> 23) - 127, -60);
  return {__uint_as_float((uint32_t)(141 - e) << 23), __uint_as_float((uint32_t)(113 + e) << 23)};
}
template <int N>
__device__ __forceinline__ float abs_max(const float* x) {
  float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) m[i & 3] = fmaxf(m[i & 3], fabsf(x[i]));
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
// the largest m of a warp; m is not negative
__device__ __forceinline__ float warp_max(float m) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m))); }
// per token, the largest |x| of the 128 lanes of four warps, this one being `quad`: N (16 or 32) tokens from j0.  put
// before a barrier of these warps, get after it.  Only the exponent counts, so the upper halves of two tokens share a
// word; every step halves the words a lane keeps.  (A reduction instruction a token is several times slower.)
template <int N>
__device__ __forceinline__ void token_max_put(const float* x, float (*parts)[C], int j0, int quad, int lane) {
  uint32_t m[N / 2];
#pragma unroll
  for (int j = 0; j < N / 2; ++j)
    m[j] = __byte_perm(__float_as_uint(x[2 * j]), __float_as_uint(x[2 * j + 1]), 0x7632) & 0x7FFF7FFFu;
#pragma unroll
  for (int s = 0; s < 5; ++s) {
    const int o = 16 >> s, n = (N / 2) >> s;
    const bool up = (lane & o) != 0;
    if (n <= 1) {
      m[0] = tc::max2_bf16(m[0], __shfl_xor_sync(0xffffffffu, m[0], o));
    } else {
#pragma unroll
      for (int i = 0; i < n / 2; ++i) {
        const uint32_t send = up ? m[i] : m[i + n / 2], keep = up ? m[i + n / 2] : m[i];
        m[i] = tc::max2_bf16(keep, __shfl_xor_sync(0xffffffffu, send, o));
      }
    }
  }
  constexpr int LANES = 64 / N;  // that hold the same two tokens
  if (lane % LANES == 0)
    *reinterpret_cast<float2*>(&parts[quad][j0 + 2 * (lane / LANES)]) =
        make_float2(__uint_as_float(m[0] << 16), __uint_as_float(m[0] & 0xFFFF0000u));
}
__device__ __forceinline__ float token_max_get(const float (*parts)[C], int j) {
  return fmaxf(fmaxf(parts[0][j], parts[1][j]), fmaxf(parts[2][j], parts[3][j]));
}
// the largest m of W warps, this one being `w`; `parts` (16-byte aligned) is written again only after another barrier of
// these warps
template <int ID, int W>
__device__ __forceinline__ float warps_max(float m, float* parts, int w) {
  m = warp_max(m);
  if ((threadIdx.x & 31) == 0) parts[w] = m;
  tc::bar_sync<ID, 32 * W>();
  m = 0.f;
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(parts + i);
    m = fmaxf(fmaxf(m, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
  }
  return m;
}
// The factor of a state comes from a bound on it: what it was and 64 max |k| max |w beta E| a chunk, loose by a few powers
// of two, of which there are 20 to spare; every EXACT chunks it is taken anew.  (A largest value each time, over the
// chain's warps: 10 % of the scans' time.  w beta E and Gam dV have no such bound where a state decays inside a chunk.)
constexpr int EXACT = 8;

template <int AB16>
__device__ __forceinline__ float h2f(uint16_t x) {
  if (AB16) return __uint_as_float((uint32_t)x << 16);
  return __half2float(__ushort_as_half(x));
}
template <int AB16>
__device__ __forceinline__ uint16_t f2h(float x) {
  if (AB16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  return __half_as_ushort(__float2half_rn(x));
}

// The chunks [c0, c1) of its document that a block walks, as a document of its own.
struct Segment {
  Seq doc, sq;       // whole; this block's part
  int c0, c1, nch;   // nch: chunks of the whole document
  bool live;
  __device__ __forceinline__ Segment(const GdrArgs& a, const Ws& w, int n, int s) {
    doc = seq_of(n, a.T, a.cu_seqlens);
    nch = (doc.len + C - 1) / C;
    c0 = s * w.seg_chunks;
    c1 = w.nseg == 1 ? nch : min(nch, c0 + w.seg_chunks);
    live = s == 0 || c0 < nch;
    sq.bos = doc.bos + (int64_t)c0 * C;
    sq.len = min(doc.len - c0 * C, (c1 - c0) * C);
  }
  __device__ __forceinline__ bool last() const { return c1 == nch; }
};

// A [64 tokens x 128 columns] tile of two swizzled panels, read or written one column per thread:
// `col` 0..127 is the thread's column.
struct Column {
  uint32_t base, chunk, byte;
  __device__ __forceinline__ Column(uint32_t tile, int col)
      : base(tile + (uint32_t)(col >> 6) * PANEL), chunk((uint32_t)(col & 63) >> 3), byte((uint32_t)(col & 7) * 2) {}
  __device__ __forceinline__ uint32_t at(int row) const { return base + tc::sw128(row, chunk) + byte; }
};
__device__ __forceinline__ uint16_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
  return v;
}
// the same, free to run ahead of ordinary loads
__device__ __forceinline__ uint32_t lds16_early(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts16(uint32_t addr, uint16_t v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(v) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
// untiled bulk copy global -> shared; addresses and size are multiples of 16 bytes
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   tc::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
               : "memory");
}

// rows [from, 64) of a tile of `panels` panels set to zero by `count` threads, this one being `t`
__device__ __forceinline__ void zero_rows(uint32_t tile, int panels, int from, int t, int count) {
  for (int i = t; i < panels * (64 - from) * 8; i += count) {
    const int p = i / ((64 - from) * 8), r = i % ((64 - from) * 8);
    sts128(tile + p * PANEL + (from + (r >> 3)) * 128 + (r & 7) * 16, make_uint4(0, 0, 0, 0));
  }
}

// rows [0, valid) of a staged [64 x 128] tile to a [tokens, HV, V] tensor with plain stores; ANY: of whole elements
// where the tensor is off 16 bytes
template <bool ANY = false>
__device__ __forceinline__ void copy_rows(uint32_t tile, uint16_t* dst, int64_t row0, int HV, int hv, int V, int v0,
                                          int valid, int t, int count) {
  for (int i = t; i < valid * 16; i += count) {
    const int r = i >> 4, ch = i & 15;
    if (v0 + ch * 8 >= V) continue;
    uint16_t* to = dst + ((row0 + r) * HV + hv) * V + v0 + ch * 8;
    const uint32_t from = tile + (ch >> 3) * PANEL + tc::sw128(r, ch & 7);
    if (!ANY || ((uintptr_t)dst & 15) == 0) {
      *reinterpret_cast<uint4*>(to) = lds128(from);
    } else {
#pragma unroll 1
      for (int e = 0; e < 8; ++e) to[e] = lds16(from + 2 * e);
    }
  }
}

// Warps of a scan: OW for the output (a share of the tokens of one TMEM quadrant each), CW for the chain (a share
// of the tokens and of K each), then a warpgroup of which the first warp loads and the second issues MMAs.
// RC, RO, RX: registers of a thread by role, redistributed from an even share.
template <int CW, int OW, int RC, int RO, int RX>
struct ScanWarps {
  static constexpr int CHAIN = OW, TMA = OW + CW, MMA = TMA + 1, THREADS = 32 * (TMA + 4);
  static constexpr int CHAIN_WARPS = CW, OUT_WARPS = OW, CHAIN_THREADS = 32 * CW, OUT_THREADS = 32 * OW;
  static constexpr int CT = 256 / CW, OT = 256 / OW;  // tokens of a chain and of an output thread
  static constexpr int EVEN = 65536 / THREADS / 8 * 8;
  static_assert(32 * CW * RC + 32 * OW * RO + 128 * RX <= THREADS * EVEN, "registers");
  template <int R>
  static __device__ __forceinline__ void set_regs() {
    if (R > EVEN) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
    if (R < EVEN) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
  }
  static __device__ __forceinline__ void chain_regs() { set_regs<RC>(); }
  static __device__ __forceinline__ void out_regs() { set_regs<RO>(); }
  static __device__ __forceinline__ void rest_regs() { set_regs<RX>(); }
};
// Measured at B=8, T=4096, H=16, K=V=128, bf16 (prep and scan; whole backward): 8 and 4 warps 367 us and
// 1190 us, 16 and 8 warps 400 us and 1127 us.  The backward's scans also stage the states and form a dot
// product per token, which four output warps do not finish within a chunk.
using FwdWarps = ScanWarps<8, 4, 144, 128, 96>;
using BwdWarps = ScanWarps<16, 8, 72, 72, 72>;
constexpr int ANCHOR_PARTS = BwdWarps::CHAIN_WARPS;

// pipe_wait for the MMA thread: polls without suspending (a suspended try_wait wakes a few hundred cycles
// late, and this thread's waits are all on the chunk's critical path), bounded like the others.
__device__ __forceinline__ bool spin_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* err, int code) {
  if (tc::mbar_test(bar, parity)) return true;
  const long long t0 = clock64();
  while (!tc::mbar_test(bar, parity)) {
    if (*abort) return false;
    if (clock64() - t0 > (1ll << 31)) {
      *abort = 1;
      atomicOr(err, code);
      return false;
    }
  }
  return true;
}

// sum over the 32 lanes of 2^k values a thread, in place: afterwards lane l holds in x[0 .. n/32) (n >= 32)
// the sums of values l * n / 32 + ...; each step halves what a thread keeps
template <int N>
__device__ __forceinline__ void lane_sums(float* x, int lane) {
#pragma unroll
  for (int o = 16, n = N; o > 0; o >>= 1, n >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float send = up ? x[i] : x[i + n / 2], keep = up ? x[i + n / 2] : x[i];
      x[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
}

// a swizzled panel of 128 rows to a [V][width] matrix of (chunk, value head) sh, columns from x, by one thread
__device__ __forceinline__ void store_panel(const CUtensorMap* m, const uint8_t* panel, int x, int v0, int V, int64_t sh) {
  tc::tma_store_3d(m, panel, x, v0, (int)sh);
  if (v0 + 64 < V) tc::tma_store_3d(m, panel + PANEL, x, v0 + 64, (int)sh);
  tc::bulk_commit();
}

// [n][V][width] matrices (the saved states and E), box 64 of width x 64 of V
inline cudaError_t matrix_map(CUtensorMap* m, const GdrArgs& a, const void* p, int width, int64_t n) {
  auto fn = tc::encode_fn();
  if (fn == nullptr) return cudaErrorNotSupported;
  cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)a.V, (cuuint64_t)n};
  cuuint64_t strides[2] = {(cuuint64_t)width * 2, (cuuint64_t)width * a.V * 2};
  cuuint32_t box[3] = {64, 64, 1};
  cuuint32_t es[3] = {1, 1, 1};
  CUresult r = fn(m, a.dtype == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                  const_cast<void*>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

inline cudaError_t token_map(CUtensorMap* m, const GdrArgs& a, const void* p, int heads, int width) {
  return tc::make_token_map(m, p, (int64_t)a.B * a.T, heads, width, C, a.dtype == DT_BF16);
}

}  // namespace gdrtc
}  // namespace ccq
#endif
