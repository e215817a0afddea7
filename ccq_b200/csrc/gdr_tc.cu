// Tensor-core path of the gated delta rule: when it applies, its workspace and its launches.
#include <stdlib.h>
#include <string.h>

#include "gdr_tc.cuh"

namespace ccq {
namespace {

using namespace gdrtc;

size_t carve(const GdrArgs& a, bool bwd, Ws* w) {
  const size_t sh = (size_t)gdr_slots(a, C) * a.HV;
  uint8_t* base = reinterpret_cast<uint8_t*>(a.workspace);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    uint8_t* p = base ? base + off : nullptr;
    off += ws_align(bytes);
    return p;
  };
  const size_t nvt = (a.V + VT - 1) / VT;
  Ws t;
  memset(&t, 0, sizeof(t));
  t.err = reinterpret_cast<int*>(take(256));
  // what the forward leaves for the backward: in its workspace, here if that is not given
  uint8_t* here = base;
  const size_t at = off;
  if (a.fwd_workspace != nullptr) {
    base = reinterpret_cast<uint8_t*>(const_cast<void*>(a.fwd_workspace));
    off = ws_align(256);
  }
  const size_t order = lpt_order_bytes(a.n_seqs, a.cu_seqlens != nullptr);
  const size_t heads = (size_t)a.n_seqs * a.HV, states = heads * a.K * a.V * 4;
  t.nseg = plan_segments(a, &t.seg_chunks);
  t.order = order ? reinterpret_cast<int*>(take(order)) : nullptr;
  t.mats = take(sh * mats_bytes(a.dtype == DT_BF16));
  t.aux = reinterpret_cast<float*>(take(sh * AX_N * 4));
  if (t.nseg > 1) {
    t.Sin = reinterpret_cast<float*>(take(t.nseg * states));
    t.Ms = reinterpret_cast<float*>(take(t.nseg * heads * a.K * a.K * 4));
  }
  if (a.fwd_workspace != nullptr) {
    base = here;
    off = at;
  }
  if (t.nseg > 1) t.Bs = reinterpret_cast<float*>(take(t.nseg * states));
  if (t.nseg > 1 && bwd) t.dSend = reinterpret_cast<float*>(take(t.nseg * states));
  if (bwd) {
    t.S0 = reinterpret_cast<uint16_t*>(take(sh * a.K * a.V * 2));
    t.dS1 = reinterpret_cast<uint16_t*>(take(sh * a.K * a.V * 2));
    t.E = reinterpret_cast<uint16_t*>(take(sh * 2 * C * a.V * 2));
    if (a.dtype == DT_F16) {
      take(nvt * sh * FX_N * 4);
      take((size_t)a.B * a.T * a.HV * a.V * 2);
    }
    t.dotO = reinterpret_cast<float*>(take(nvt * sh * C * 4));
    t.dotV = reinterpret_cast<float*>(take(nvt * sh * C * 4));
    const size_t ah = (size_t)gdr_slots(a, C * ANCHOR) * a.HV;
    t.Sf = reinterpret_cast<float*>(take(ah * a.K * a.V * 4));
    t.anchor = reinterpret_cast<float*>(take(nvt * ah * ANCHOR_PARTS * 4));
  }
  if (w) *w = t;
  return off;
}

// What the scans start from: the launch order of packed documents, the chunks' inverses, scores and factors, the
// states at the starts of segments.
cudaError_t start(const GdrArgs& a, const Ws& w, int* launches) {
  cudaError_t e = cudaSuccess;
  if (w.order) {
    CleanArgs c;
    memset(&c, 0, sizeof(c));
    c.T = a.T;
    c.n_seqs = a.n_seqs;
    c.cu_seqlens = a.cu_seqlens;
    c.stream = a.stream;
    e = lpt_order(c, const_cast<int*>(w.order), launches);
  }
  if (e == cudaSuccess) e = prep(a, w, launches);
  if (e == cudaSuccess && w.nseg > 1) e = scan(a, w, SCAN_SUM, launches);
  if (e == cudaSuccess && w.nseg > 1) e = join(a, w, false, launches);
  return e;
}

}  // namespace

// The backward takes the forward's workspace without asking who wrote it, so what decides here has to be the same
// in both calls: the environment is read once, and o, which the backward does not have, is left out (an o off
// 16 bytes is stored without TMA).  The backward's own tensors only ever add reasons for the exact path, which
// does not read the forward's workspace.
bool gdr_tc_supported(const GdrArgs& a) {
  static const bool forced = [] {
    const char* env = getenv("CCQ_B200_FORCE_SIMT");
    return env && env[0] == '1';
  }();
  if (forced) return false;
  if (a.dtype != DT_BF16 && a.dtype != DT_F16) return false;
  if (a.T < 1 || a.K > 128 || a.K % 8 != 0 || a.V % 8 != 0) return false;
  if (gdr_slots(a, C) * a.HV >= (1ll << 31)) return false;  // the kernels count (chunk, head) pairs in 32 bits
  const uintptr_t p = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.d_o | (uintptr_t)a.dq |
                      (uintptr_t)a.dk | (uintptr_t)a.dv;
  return (p & 15) == 0;
}

size_t gdr_tc_workspace(const GdrArgs& a, bool bwd) {
  GdrArgs b = a;
  b.workspace = nullptr;
  return carve(b, bwd, nullptr);
}

cudaError_t gdr_tc_fwd(const GdrArgs& a, int* launches) {
  Ws w;
  carve(a, false, &w);
  cudaError_t e = cudaMemsetAsync(w.err, 0, 8, a.stream);
  if (e == cudaSuccess) e = start(a, w, launches);
  if (e == cudaSuccess) e = scan(a, w, SCAN_FWD, launches);
  return e;
}

cudaError_t gdr_tc_bwd(const GdrArgs& a, int* launches) {
  Ws w;
  carve(a, true, &w);
  cudaError_t e = cudaMemsetAsync(w.err, 0, 8, a.stream);
  if (e == cudaSuccess && a.fwd_workspace == nullptr) e = start(a, w, launches);
  if (e == cudaSuccess) e = scan(a, w, SCAN_BWD, launches);
  if (e == cudaSuccess && w.nseg > 1) e = rscan(a, w, true, launches);
  if (e == cudaSuccess && w.nseg > 1) e = join(a, w, true, launches);
  if (e == cudaSuccess) e = rscan(a, w, false, launches);
  if (e == cudaSuccess) e = grads(a, w, launches);
  return e;
}

}  // namespace ccq
