// Distillation from a teacher's top logits.  Row n has the student's logits
// z (V) and the teacher's K stored logits t_k with their ids i_k:
//
//   p = softmax(t / tau) over the K stored entries, q = softmax(z / tau) over V
//   loss = tau^2 sum_k p_k (log p_k - log q_{i_k})
//   dz_j = g tau (q_j - sum_{k: i_k = j} p_k)
//
// An entry whose teacher logit is -inf is not there (rows may have fewer than
// K), and a row with none has loss 0 and gradient 0.  An id outside the
// vocabulary raises WXX_DEV_ERR_BAD_INDEX and its entry counts as not there.

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace {

constexpr int kT = 256;
constexpr int kMaxK = 1024;

template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) v += red[w];
  __syncthreads();
  return v;
}

// The maximum, NaN if there is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

template <int THREADS>
__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 32; ++w) v = max_nan(v, red[w]);
  __syncthreads();
  return v;
}

// The teacher's side of a row: s_t[k] = (t_k - max) / tau, s_p[k] = p_k; returns
// whether the row has an entry, and log of the sum in log_sum.
template <int THREADS>
__device__ bool teacher_row(const float* __restrict__ top, const uint32_t* __restrict__ ids, int K,
                            uint32_t V, float inv_tau, float* s_t, float* s_p, float* red,
                            float& log_sum, int* err) {
  float m = -INFINITY;
  for (int k = threadIdx.x; k < K; k += THREADS) {
    float t = top[k];
    if (t != -INFINITY && ids[k] >= V) {
      wxx_device_fail(err, WXX_DEV_ERR_BAD_INDEX);
      t = -INFINITY;
    }
    s_t[k] = t;
    m = max_nan(m, t);
  }
  m = block_max<THREADS>(m, red);
  const bool some = m != -INFINITY;
  float s = 0.f;
  for (int k = threadIdx.x; k < K; k += THREADS) {
    const float t = some ? (s_t[k] - m) * inv_tau : 0.f;
    const float e = some ? expf(t) : 0.f;
    s_t[k] = t;
    s_p[k] = e;
    s += e;
  }
  s = block_sum<THREADS>(s, red);
  log_sum = some ? logf(s) : 0.f;
  const float inv = some ? 1.0f / s : 0.f;
  for (int k = threadIdx.x; k < K; k += THREADS) s_p[k] *= inv;
  __syncthreads();
  return some;
}

__global__ void __launch_bounds__(kT)
    distill_forward_kernel(float* __restrict__ loss, float* __restrict__ stats,
                           const float* __restrict__ logits, int64_t ld,
                           const float* __restrict__ top, const uint32_t* __restrict__ ids, int V,
                           int K, float inv_tau, float tau2, int* err) {
  __shared__ float s_t[kMaxK], s_p[kMaxK], red[kT / 32];
  const int64_t row = blockIdx.x;
  const float* z = logits + row * ld;
  float log_sum;
  const bool some = teacher_row<kT>(top + row * K, ids + row * K, K, V, inv_tau, s_t, s_p, red,
                                    log_sum, err);
  float m = -INFINITY;
  for (int c = threadIdx.x; c < V; c += kT) m = max_nan(m, z[c]);
  m = block_max<kT>(m, red);
  float s = 0.f;
  for (int c = threadIdx.x; c < V; c += kT) s += expf((z[c] - m) * inv_tau);
  s = block_sum<kT>(s, red);
  const float log_s = logf(s);
  float part = 0.f;
  for (int k = threadIdx.x; k < K; k += kT) {
    const float p = s_p[k];
    if (!(p == 0.f))
      part += p * ((s_t[k] - log_sum) - ((z[ids[row * K + k]] - m) * inv_tau - log_s));
  }
  part = block_sum<kT>(part, red);
  if (threadIdx.x == 0) {
    loss[row] = some ? tau2 * part : 0.f;
    stats[2 * row] = m;
    stats[2 * row + 1] = s;
  }
}

__global__ void __launch_bounds__(kT)
    distill_backward_kernel(float* __restrict__ dz, const float* __restrict__ grad,
                            const float* __restrict__ logits, int64_t ld,
                            const float* __restrict__ top, const uint32_t* __restrict__ ids,
                            const float* __restrict__ stats, int V, int K, float tau,
                            float inv_tau, int* err) {
  __shared__ float s_t[kMaxK], s_p[kMaxK], red[kT / 32];
  const int64_t row = blockIdx.x;
  const float* z = logits + row * ld;
  const uint32_t* id = ids + row * K;
  float* out = dz + row * V;
  float log_sum;
  const bool some = teacher_row<kT>(top + row * K, id, K, V, inv_tau, s_t, s_p, red, log_sum, err);
  const float m = stats[2 * row], inv = 1.0f / stats[2 * row + 1], g = grad[row] * tau;
  for (int c = threadIdx.x; c < V; c += kT)
    out[c] = some ? g * (expf((z[c] - m) * inv_tau) * inv) : 0.f;
  __syncthreads();
  // the first entry of an id takes all that have it
  for (int k = threadIdx.x; k < K; k += kT) {
    if (s_p[k] == 0.f || !some) continue;
    const uint32_t c = id[k];
    float p = s_p[k];
    bool first = true;
    for (int j = 0; j < k; ++j) first = first && !(id[j] == c && s_p[j] != 0.f);
    if (!first) continue;
    for (int j = k + 1; j < K; ++j)
      if (id[j] == c) p += s_p[j];
    out[c] = g * (expf((z[c] - m) * inv_tau) * inv - p);
  }
}

}  // namespace

// loss (N) and the row statistics stats (N, 2: the largest logit and the sum of
// exp((z - largest) / tau)) that wxx_distill_backward takes; logits (N, V) with
// row stride ld, top and ids (N, K).
WXX_EXPORT int wxx_distill_loss(float* loss, float* stats, const float* logits, int64_t ld,
                                const float* top, const uint32_t* ids, int64_t N, int64_t V, int K,
                                float tau) {
  WXX_REQUIRE_INIT();
  WXX_REQUIRE(N >= 0 && N < (int64_t(1) << 31) && V >= 1 && V < (int64_t(1) << 31),
              "wxx_distill_loss: bad sizes");
  WXX_REQUIRE(K >= 1 && K <= kMaxK, "wxx_distill_loss: %d stored logits outside [1, %d]", K, kMaxK);
  WXX_REQUIRE(tau > 0.f && tau < INFINITY, "wxx_distill_loss: the temperature must be positive");
  if (N == 0) return WXX_OK;
  distill_forward_kernel<<<(unsigned)N, kT, 0, wxx::stream()>>>(
      loss, stats, logits, ld, top, ids, (int)V, K, 1.0f / tau, tau * tau,
      wxx::device_error_word());
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}

// dz (N, V) from the gradient of the losses grad (N).
WXX_EXPORT int wxx_distill_backward(float* dz, const float* grad, const float* logits, int64_t ld,
                                    const float* top, const uint32_t* ids, const float* stats,
                                    int64_t N, int64_t V, int K, float tau) {
  WXX_REQUIRE_INIT();
  WXX_REQUIRE(N >= 0 && N < (int64_t(1) << 31) && V >= 1 && V < (int64_t(1) << 31),
              "wxx_distill_backward: bad sizes");
  WXX_REQUIRE(K >= 1 && K <= kMaxK, "wxx_distill_backward: %d stored logits outside [1, %d]", K,
              kMaxK);
  WXX_REQUIRE(tau > 0.f && tau < INFINITY,
              "wxx_distill_backward: the temperature must be positive");
  if (N == 0) return WXX_OK;
  distill_backward_kernel<<<(unsigned)N, kT, 0, wxx::stream()>>>(
      dz, grad, logits, ld, top, ids, stats, (int)V, K, tau, 1.0f / tau, wxx::device_error_word());
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}
