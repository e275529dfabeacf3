// Rows of logits: how a block's threads share one, for the kernels that go through
// long rows once (csrc/select.cu, csrc/distill.cu).
#pragma once

#include "common.cuh"

namespace wxx_rows {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A row split over THREADS threads: 16-byte groups in the aligned middle, thread
// t taking groups t, t + THREADS, ..., and up to six single entries at its ends,
// one each for the first threads.
struct Row {
  const float* p;
  const float4* mid;
  int V, head, groups, single;        // single: this thread's single entry, -1 for none
  __device__ Row(const float* row, int n) : p(row), V(n) {
    head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / 4);
    groups = (n - head) / 4;
    mid = reinterpret_cast<const float4*>(row + head);
    const int tail = n - head - 4 * groups, t = threadIdx.x;
    single = t < head ? t : t < head + tail ? n - tail + (t - head) : -1;
  }
  template <int THREADS, class F>
  __device__ __forceinline__ void each(F f) const {
    if (single >= 0) f(p[single], single);
    constexpr int kAhead = 4;         // loads in flight: they come from L2
    for (int i = threadIdx.x; i < groups; i += kAhead * THREADS) {
      float4 v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (i + k * THREADS < groups) v[k] = mid[i + k * THREADS];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (i + k * THREADS >= groups) break;
        const int at = head + 4 * (i + k * THREADS);
        f(v[k].x, at);
        f(v[k].y, at + 1);
        f(v[k].z, at + 2);
        f(v[k].w, at + 3);
      }
    }
  }
};

}  // namespace wxx_rows
