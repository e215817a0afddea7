// Tensor-core path of the gated delta rule: documents in segments, for few heads and a long axis.
//
// A segment's end state is a linear map of its start, S_end = M S_start + B: B is the walk from a zero state, M
// the walk from the identity without V, both with the scan's own kernel (SCAN_SUM).  All segments are
// summarised side by side, the starts follow from S_{s+1} = M_s S_s + B_s (fp32, this file), and then every
// segment is walked from its start at once.  Backwards the gradient at a segment's start is M^T dS_end + D
// with the same M, D being the reverse walk from a zero gradient.
//
// A document's chunks cost one walk instead of three, so this pays where the heads leave SMs idle: 16 heads of
// 16384 tokens (K = V = 128) take 8 segments of 32 chunks and 464 us, 887 us in one piece.
#include "gdr_tc.cuh"

namespace ccq {
namespace gdrtc {
namespace {

constexpr int COLS = 16, THREADS = 256;

// S_next [K][COLS] = M S + B over the segments of one (document, value head), or backwards with M^T
template <bool REV>
__global__ void __launch_bounds__(THREADS) join_kernel(GdrArgs a, Ws w) {
  extern __shared__ float4 smem4[];
  const int K = a.K, ld = K + 4;
  float* M = reinterpret_cast<float*>(smem4);  // [K][ld]
  float* S = M + K * ld;                       // [K][COLS]
  const int64_t heads = (int64_t)a.n_seqs * a.HV, nh = blockIdx.x;
  const int c = threadIdx.x & (COLS - 1), r0 = threadIdx.x / COLS, v = blockIdx.y * COLS + c;
  const bool in = v < a.V;
  const Seq doc = seq_of((int)(nh / a.HV), a.T, a.cu_seqlens);
  const int nch = (doc.len + C - 1) / C, segs = (nch + w.seg_chunks - 1) / w.seg_chunks;  // those it has
  if (segs < 2) return;
  constexpr int ROWS = 128 * COLS / THREADS;
  for (int step = 0; step < segs - 1; ++step) {
    const int s = REV ? segs - 1 - step : step;  // the segment stepped over
    float x[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int k = r0 + i * (THREADS / COLS);
      x[i] = k < K && in ? w.Bs[((s * heads + nh) * K + k) * a.V + v] : 0.f;
    }
    if (step > 0) {
      const float* m = w.Ms + (s * heads + nh) * K * K;
      for (int i = threadIdx.x; i < K * K / 4; i += THREADS) {
        const int row = i * 4 / K, col = i * 4 % K;
        *reinterpret_cast<float4*>(M + row * ld + col) = reinterpret_cast<const float4*>(m)[i];
      }
      __syncthreads();
      for (int j = 0; j < K; ++j) {
        const float sj = S[j * COLS + c];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const int k = r0 + i * (THREADS / COLS);
          if (k < K) x[i] = fmaf(REV ? M[j * ld + k] : M[k * ld + j], sj, x[i]);
        }
      }
      __syncthreads();
    }
    float* out = REV ? w.dSend + ((s - 1) * heads + nh) * K * a.V : w.Sin + ((s + 1) * heads + nh) * K * a.V;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int k = r0 + i * (THREADS / COLS);
      if (k < K) {
        S[k * COLS + c] = x[i];
        if (in) out[(int64_t)k * a.V + v] = x[i];
      }
    }
  }
}

}  // namespace

// Segments of a document: the count that minimises the waves of blocks over 148 SMs, in chunks walked one
// after another (a summary walks a chunk in about 0.85 of the time; the launches and the joining cost about 12
// chunks), if it saves a quarter at least.
int plan_segments(const GdrArgs& a, int* seg_chunks) {
  const int chunks = (a.T + C - 1) / C, nvt = (a.V + VT - 1) / VT;
  const int64_t heads = (int64_t)a.n_seqs * a.HV;
  auto waves = [](int64_t blocks) { return (double)((blocks + 147) / 148); };
  int best = 1, best_len = chunks;
  double cost = 0.75 * waves(heads * nvt) * chunks;
  for (int n = 2; n <= 16; ++n) {
    const int len = ((chunks + n - 1) / n + ANCHOR - 1) / ANCHOR * ANCHOR, segs = (chunks + len - 1) / len;
    if (segs < 2) break;
    const double t = 0.85 * waves(heads * ((segs - 1) * nvt + segs - 2)) * len + waves(heads * nvt * segs) * len + 12;
    if (t < cost) {
      cost = t;
      best = segs;
      best_len = len;
    }
  }
  *seg_chunks = best_len;
  return best;
}

cudaError_t join(const GdrArgs& a, const Ws& w, bool reverse, int* launches) {
  ++*launches;
  const size_t bytes = sizeof(float) * ((size_t)a.K * (a.K + 4) + a.K * COLS);
  const dim3 grid((unsigned)(a.n_seqs * a.HV), (a.V + COLS - 1) / COLS);
  cudaError_t e = reverse ? cudaFuncSetAttribute(join_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes)
                          : cudaFuncSetAttribute(join_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return e;
  if (reverse) join_kernel<true><<<grid, THREADS, bytes, a.stream>>>(a, w);
  else join_kernel<false><<<grid, THREADS, bytes, a.stream>>>(a, w);
  return cudaGetLastError();
}

}  // namespace gdrtc
}  // namespace ccq
