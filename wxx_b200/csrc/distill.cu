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
#include <cooperative_groups.h>
#include <stdint.h>

#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "rows.cuh"

namespace {

using wxx_rows::Row;
using wxx_rows::warp_sum;

constexpr int kT = 256;
constexpr int kWarps = kT / 32;
constexpr int kMaxK = 1024;
constexpr int kMaxParts = 8;          // blocks that share a row, at most
constexpr int kStats = 4;             // largest logit, sum of exp; the teacher's two

// The maximum, NaN if there is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// Over the block, in an order that depends on nothing but the values' places.
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();                    // red has been read
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) v += red[w];
  return v;
}
__device__ __forceinline__ float block_max_nan(float v, float* red) {
  v = warp_max_nan(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) v = max_nan(v, red[w]);
  return v;
}

// log2(e) / tau: rounded, and what is left of it.
struct Scale {
  float c, low;
  static Scale of(float tau) {
    const double c = 1.4426950408889634 / (double)tau;
    return {(float)c, (float)(c - (double)(float)c)};
  }
};
// exp of a logit's distance over tau as a term of a row's sum: 2^y with y = (v - m) c
// rounded, which costs it y half ulps -- but a term weighs q, and the mean of y over q is
// log2 V at most, so the sum loses less than by being added up.  (With scaled_exp2's
// terms the forward over 4096 x 50304 took 138 us, 131 with these.)
__device__ __forceinline__ float term_exp(float v, float m, Scale s) {
  return fast_exp2((v - m) * s.c);
}
// The same to a few ulp however far the logits are apart, for a q by itself: 2^y 2^r with
// r what the product and c lost, so little (where 2^y is not 0) that 2^r is 1 + r log 2.
// Without r q is 60 half ulps off at a distance of 80 tau.  Logits of -inf have y = -inf
// and an r that is no number, which any 2^r serves.
__device__ __forceinline__ float2 scaled_exp2(float v0, float v1, float m, Scale s) {
  float d0, d1, y0, y1, r0, r1, e0, e1;
  sub2(d0, d1, v0, v1, m, m);
  mul2(y0, y1, d0, d1, s.c, s.c);
  fma2(r0, r1, d0, d1, s.c, s.c, -y0, -y1);
  fma2(r0, r1, d0, d1, s.low, s.low, r0, r1);
  fma2(r0, r1, fminf(r0, 1.0f), fminf(r1, 1.0f), 0.6931471805599453f, 0.6931471805599453f, 1.0f,
       1.0f);
  mul2(e0, e1, fast_exp2(y0), fast_exp2(y1), r0, r1);
  return make_float2(e0, e1);
}
__device__ __forceinline__ float scaled_exp(float v, float m, Scale s) {
  return scaled_exp2(v, v, m, s).x;
}

// A stored teacher logit, -inf where the entry is not there.
__device__ __forceinline__ float stored(float t, uint32_t id, uint32_t V, int* err) {
  if (t == -INFINITY || id < V) return t;
  wxx_device_fail(err, WXX_DEV_ERR_BAD_INDEX);
  return -INFINITY;
}

struct Sum {
  float top, sum;                     // the largest so far, the sum of exp(v - top)
};
__device__ __forceinline__ Sum plus(Sum a, Sum b, Scale c) {
  const float top = max_nan(a.top, b.top);
  return {top, (a.top == top ? a.sum : a.sum * term_exp(a.top, top, c)) +
                   (b.top == top ? b.sum : b.sum * term_exp(b.top, top, c))};
}

// One pass over a row's piece: 16 logits at a time, their largest against the
// thread's so far, one rescaling of its sum where they exceed it.  4 bytes and
// one exponential a logit; the loads are what bounds it: 4096 x 50304 logits in 131
// us, 6.3 TB/s, eight blocks of 256 threads on an SM with 16 KB each on their way.
__device__ Sum piece_sum(const Row& row, Scale c, Sum* red) {
  Sum s{-INFINITY, 0.f};
  auto add = [&](float v) {
    if (v != -INFINITY) s = plus(s, {v, 1.0f}, c);
  };
  if (row.single >= 0) add(row.p[row.single]);
  constexpr int kAhead = 4;
  int i = threadIdx.x;
  for (; i + (kAhead - 1) * kT < row.groups; i += kAhead * kT) {
    float4 v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) v[k] = row.mid[i + k * kT];
    float n = s.top;
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      n = max_nan(max_nan(n, max_nan(v[k].x, v[k].y)), max_nan(v[k].z, v[k].w));
    if (n == -INFINITY) continue;
    float e = s.top == n ? s.sum : s.sum * term_exp(s.top, n, c);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      e += (term_exp(v[k].x, n, c) + term_exp(v[k].y, n, c)) +
           (term_exp(v[k].z, n, c) + term_exp(v[k].w, n, c));
    s = {n, e};
  }
  for (; i < row.groups; i += kT) {
    const float4 v = row.mid[i];
    const float n = max_nan(max_nan(s.top, max_nan(v.x, v.y)), max_nan(v.z, v.w));
    if (n == -INFINITY) continue;
    s = {n, (s.top == n ? s.sum : s.sum * term_exp(s.top, n, c)) +
                ((term_exp(v.x, n, c) + term_exp(v.y, n, c)) +
                 (term_exp(v.z, n, c) + term_exp(v.w, n, c)))};
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    s = plus(s, {__shfl_xor_sync(0xffffffffu, s.top, o), __shfl_xor_sync(0xffffffffu, s.sum, o)}, c);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = red[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) s = plus(s, red[w], c);
  return s;
}

// A row's blocks (a cluster where there are several) each take a piece of it; the
// first has the teacher's entries meanwhile, then joins the pieces' sums.
__global__ void __launch_bounds__(kT)
    distill_forward_kernel(float* __restrict__ loss, float* __restrict__ stats,
                           const float* __restrict__ logits, int64_t ld,
                           const float* __restrict__ top, const uint32_t* __restrict__ ids, int V,
                           int K, int parts, int length, float inv_tau, Scale c, float tau2,
                           int* err) {
  namespace cg = cooperative_groups;
  __shared__ float s_t[kMaxK], red[kWarps];
  __shared__ Sum s_red[kWarps], s_part[kMaxParts];
  const int part = blockIdx.x % parts;
  const int64_t at = blockIdx.x / parts;
  const float* z = logits + at * ld;
  if (parts > 1) cg::this_cluster().barrier_arrive();
  float t_top = -INFINITY, t_sum = 0.f;
  if (part == 0) {
    for (int k = threadIdx.x; k < K; k += kT) {
      const float t = stored(top[at * K + k], ids[at * K + k], V, err);
      s_t[k] = t;
      t_top = max_nan(t_top, t);
    }
    t_top = block_max_nan(t_top, red);
    for (int k = threadIdx.x; k < K; k += kT)
      if (t_top != -INFINITY) t_sum += expf((s_t[k] - t_top) * inv_tau);
    t_sum = block_sum(t_sum, red);
  }
  const int from = part * length;
  Sum s = piece_sum(Row(z + from, min(length, V - from)), c, s_red);
  if (parts > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.barrier_wait();          // the first block is there
    if (threadIdx.x == 0) *cluster.map_shared_rank(&s_part[part], 0) = s;
    cluster.sync();
    if (part != 0) return;
    s = s_part[0];
    for (int k = 1; k < parts; ++k) s = plus(s, s_part[k], c);
  }
  const bool some = t_top != -INFINITY;
  const float log_s = logf(s.sum), log_t = logf(t_sum), inv = 1.0f / t_sum;
  float sum = 0.f;
  if (some)
    for (int k = threadIdx.x; k < K; k += kT) {
      const float t = (s_t[k] - t_top) * inv_tau, p = expf(t) * inv;
      // an entry that is not there may have any id, and a p of NaN from one that is
      if (s_t[k] != -INFINITY && !(p == 0.f))
        sum += p * ((t - log_t) - ((z[ids[at * K + k]] - s.top) * inv_tau - log_s));
    }
  sum = block_sum(sum, red);
  if (threadIdx.x == 0) {
    loss[at] = some ? tau2 * sum : 0.f;
    float* o = stats + at * kStats;
    o[0] = s.top;
    o[1] = s.sum;
    o[2] = t_top;
    o[3] = t_sum;
  }
}

// Whether entry k is the first with its id; p, its own, becomes the sum over all that
// have the id.  (id is 16-byte aligned and filled to a multiple of four.)
__device__ __forceinline__ bool first_of_its_id(const uint32_t* id, const float* ps, int K, int k,
                                                float& p) {
  const uint32_t j = id[k];
  int same = 0;
#pragma unroll 4
  for (int o = 0; o < K; o += 4) {
    const uint4 four = *reinterpret_cast<const uint4*>(id + o);
    same += (four.x == j) + (four.y == j) + (four.z == j) + (four.w == j);
  }
  if (same == 1) return true;
  p = 0.f;
  bool first = true;
  for (int o = 0; o < K; ++o) {
    if (id[o] != j) continue;
    first = first && o >= k;
    p += ps[o];
  }
  return first;
}

// dz over a piece of a row: g tau q everywhere, then the stored entries that lie in
// it.  8 bytes a logit: 4096 x 50304 in 279 us, 5.9 TB/s, the rate of reading and
// writing at once.  (Cache hints for streaming did not help: 279 us on the stores,
// 300 us on the loads too.)  kAligned: logits and dz have the same place in their 16
// bytes, so both go four at a time.
template <bool kAligned>
__global__ void __launch_bounds__(kT)
    distill_backward_kernel(float* __restrict__ dz, const float* __restrict__ grad,
                            const float* __restrict__ logits, int64_t ld,
                            const float* __restrict__ top, const uint32_t* __restrict__ ids,
                            const float* __restrict__ stats, int V, int K, int parts, int length,
                            float tau, float inv_tau, Scale c, int* err) {
  __shared__ float s_p[kMaxK];
  __shared__ __align__(16) uint32_t s_id[kMaxK];
  const int part = blockIdx.x % parts;
  const int64_t at = blockIdx.x / parts;
  const int from = part * length, n = min(length, V - from);
  const float* z = logits + at * ld + from;
  float* out = dz + at * V + from;
  const float4 st = *reinterpret_cast<const float4*>(stats + at * kStats);
  const bool some = st.w != 0.f;     // the teacher's sum: 0 without entries
  const float m = st.x, inv = 1.0f / st.y, g = grad[at] * tau;
  if (some) {
    const float inv_t = 1.0f / st.w;
    if (threadIdx.x < 4 && K + threadIdx.x < kMaxK) s_id[K + threadIdx.x] = 0xffffffffu;
    for (int k = threadIdx.x; k < K; k += kT) {
      const uint32_t j = ids[at * K + k];
      const float t = stored(top[at * K + k], j, V, part == 0 ? err : nullptr);
      s_id[k] = j;
      s_p[k] = t == -INFINITY ? 0.f : expf((t - st.z) * inv_tau) * inv_t;
    }
  }
  auto value = [&](float v) { return some ? g * (scaled_exp(v, m, c) * inv) : 0.f; };
  auto values = [&](float4 v) {
    const float2 a = scaled_exp2(v.x, v.y, m, c), b = scaled_exp2(v.z, v.w, m, c);
    return some ? make_float4(g * (a.x * inv), g * (a.y * inv), g * (b.x * inv), g * (b.y * inv))
                : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  if (kAligned) {
    const Row row(z, n);
    if (row.single >= 0) out[row.single] = value(z[row.single]);
    float4* to = reinterpret_cast<float4*>(out + row.head);
    constexpr int kAhead = 4;
    int i = threadIdx.x;
    for (; i + (kAhead - 1) * kT < row.groups; i += kAhead * kT) {
      float4 v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) v[k] = row.mid[i + k * kT];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) to[i + k * kT] = values(v[k]);
    }
    for (; i < row.groups; i += kT) to[i] = values(row.mid[i]);
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += kT) out[i] = value(z[i]);
  }
  if (!some) return;
  __syncthreads();                   // the stored entries overwrite what is there
  for (int k = threadIdx.x; k < K; k += kT) {
    const uint32_t j = s_id[k];
    if (j < (uint32_t)from || j - (uint32_t)from >= (uint32_t)n) continue;
    const float q = scaled_exp(z[j - from], m, c) * inv;
    float p = s_p[k];
    if (first_of_its_id(s_id, s_p, K, k, p)) out[j - from] = g * (q - p);
  }
}

// Short rows: a warp a row, its logits in registers (entry 32 j + lane in v[j]) and a few
// stored entries a lane, so there is no barrier and one exponential a logit.  Bound by
// instructions and, with few rows, latencies: 4096 x 1021 logits with 64 stored take 6
// us forward (a block a row 23) and 12 backward (14), 4096 x 200 6 and 8 us (21 and 12).
// Backward, a warp is longer at comparing the stored ids with one another.  A warp and a
// block a row, 64 of 1021 stored: 128 rows 3.3 and 3.1 us, 512 rows 3.5 both, 768 rows 4.0
// both, 1023 rows 4.0 and 4.4, 2048 rows 5.4 and 7.3; 17 stored: 128 rows 2.6 and 2.8, 1023
// rows 3.0 and 4.0.  4096 rows with 128 stored took 21 and 19 us.  So it has 512 rows and
// more, and at most 64 stored entries.  (Backward: one call after the other over the same
// rows.)
constexpr int kRowWarps = 4;
constexpr int kForwardEntries = 4, kBackwardEntries = 2;       // of a lane
constexpr int kForwardV = 2048, kBackwardV = 1024, kBackwardN = 512;

template <int ITEMS>
__global__ void __launch_bounds__(kRowWarps * 32)
    distill_forward_rows_kernel(float* __restrict__ loss, float* __restrict__ stats,
                                const float* __restrict__ logits, int64_t ld,
                                const float* __restrict__ top, const uint32_t* __restrict__ ids,
                                int64_t N, int V, int K, float inv_tau, Scale c, float tau2,
                                int* err) {
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  if (at >= N) return;
  const float* z = logits + at * ld;
  float v[ITEMS], t[kForwardEntries];
  uint32_t id[kForwardEntries];          // V: not there
#pragma unroll
  for (int i = 0; i < kForwardEntries; ++i) {
    const int k = 32 * i + lane;
    id[i] = k < K ? ids[at * K + k] : 0u;
    t[i] = k < K ? top[at * K + k] : -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) v[j] = 32 * j + lane < V ? z[32 * j + lane] : -INFINITY;
  float m = -INFINITY, t_top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kForwardEntries; ++i) {
    t[i] = stored(t[i], id[i], V, err);
    if (t[i] == -INFINITY) id[i] = V;
    t_top = max_nan(t_top, t[i]);
  }
  t_top = warp_max_nan(t_top);
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) m = max_nan(m, v[j]);
  m = warp_max_nan(m);
  float s = 0.f, t_sum = 0.f;
  if (m != -INFINITY) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) s += term_exp(v[j], m, c);
  }
  s = warp_sum(s);
  const bool some = t_top != -INFINITY;
  float p[kForwardEntries];
#pragma unroll
  for (int i = 0; i < kForwardEntries; ++i) {
    t[i] = some ? (t[i] - t_top) * inv_tau : -INFINITY;
    t_sum += p[i] = expf(t[i]);
  }
  t_sum = warp_sum(t_sum);
  const float log_s = logf(s), log_t = logf(t_sum), inv = 1.0f / t_sum;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kForwardEntries; ++i) {
    if (id[i] >= (uint32_t)V || p[i] * inv == 0.f) continue;
    sum += p[i] * inv * ((t[i] - log_t) - ((z[id[i]] - m) * inv_tau - log_s));
  }
  sum = warp_sum(sum);
  if (lane == 0) {
    loss[at] = some ? tau2 * sum : 0.f;
    *reinterpret_cast<float4*>(stats + at * kStats) = make_float4(m, s, t_top, t_sum);
  }
}

template <int ITEMS>
__global__ void __launch_bounds__(kRowWarps * 32)
    distill_backward_rows_kernel(float* __restrict__ dz, const float* __restrict__ grad,
                                 const float* __restrict__ logits, int64_t ld,
                                 const float* __restrict__ top, const uint32_t* __restrict__ ids,
                                 const float* __restrict__ stats, int64_t N, int V, int K,
                                 float tau, float inv_tau, Scale c, int* err) {
  __shared__ __align__(16) uint32_t s_id[kRowWarps][32 * kBackwardEntries];
  __shared__ float s_p[kRowWarps][32 * kBackwardEntries];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t at = (int64_t)blockIdx.x * kRowWarps + warp;
  if (at >= N) return;
  const float* z = logits + at * ld;
  float* out = dz + at * V;
  const float4 st = *reinterpret_cast<const float4*>(stats + at * kStats);
  const bool some = st.w != 0.f;     // the teacher's sum: 0 without entries
  const float m = st.x, inv = 1.0f / st.y, inv_t = 1.0f / st.w, g = grad[at] * tau;
  float v[ITEMS];
  uint32_t id[kBackwardEntries];          // V: not there
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) v[j] = 32 * j + lane < V ? z[32 * j + lane] : 0.f;
#pragma unroll
  for (int i = 0; i < kBackwardEntries; ++i) {
    const int k = 32 * i + lane;
    id[i] = k < K ? ids[at * K + k] : 0u;
    const float t = k < K ? stored(top[at * K + k], id[i], V, err) : -INFINITY;
    if (t == -INFINITY) id[i] = V;
    s_id[warp][k] = id[i];
    s_p[warp][k] = t == -INFINITY ? 0.f : expf((t - st.z) * inv_tau) * inv_t;
  }
#pragma unroll
  for (int j = 0; j < ITEMS; j += 2) {
    const float2 e = scaled_exp2(v[j], v[j + 1], m, c);
    if (32 * j + lane < V) out[32 * j + lane] = some ? g * (e.x * inv) : 0.f;
    if (32 * j + 32 + lane < V) out[32 * j + 32 + lane] = some ? g * (e.y * inv) : 0.f;
  }
  if (!some) return;
  __syncwarp();                      // the stored entries overwrite what is there
#pragma unroll
  for (int i = 0; i < kBackwardEntries; ++i) {
    if (32 * i >= K) break;
    if (id[i] >= (uint32_t)V) continue;
    const float q = scaled_exp(z[id[i]], m, c) * inv;
    float p = s_p[warp][32 * i + lane];
    if (first_of_its_id(s_id[warp], s_p[warp], K, 32 * i + lane, p)) out[id[i]] = g * (q - p);
  }
}

// The kernel of a row length.
template <int MOST, class F>
int by_length(int64_t V, F launch) {
  using std::integral_constant;
  if (V <= 256) return launch(integral_constant<int, 8>{});
  if (V <= 512) return launch(integral_constant<int, 16>{});
  if constexpr (MOST > 1024)
    if (V > 1024) return launch(integral_constant<int, MOST / 32>{});
  return launch(integral_constant<int, 32>{});
}

int check_sizes(const char* what, int64_t N, int64_t V, int K, float tau) {
  WXX_REQUIRE(N >= 0 && N < (int64_t(1) << 28) && V >= 1 && V < (int64_t(1) << 31) - 4 * kT,
              "%s: bad sizes", what);
  WXX_REQUIRE(K >= 1 && K <= kMaxK, "%s: %d stored logits outside [1, %d]", what, K, kMaxK);
  WXX_REQUIRE(tau > 0.f && tau < INFINITY, "%s: the temperature must be positive", what);
  return WXX_OK;
}

// Pieces of a row, so that few long rows still give every SM two blocks; a piece is
// a multiple of 4 logits, about 4096 or more.  Forward and backward in pieces and whole:
// 1 row of 50304 6 + 4 and 10 + 10 us, 48 rows 8 + 6 and 10 + 10 us; 64 rows of 4096 (in
// pieces of 2048) 6 + 4 and 4 + 4 us.
void split_row(int64_t N, int64_t V, int& parts, int& length) {
  const int64_t wanted = (2 * wxx::num_sms() + N - 1) / N, most = (V + 4095) / 4096;
  int64_t n = wanted < most ? wanted : most;
  n = n < kMaxParts ? n : kMaxParts;
  length = (int)(((V + n - 1) / n + 3) / 4 * 4);
  parts = (int)((V + length - 1) / length);
}

}  // namespace

// loss (N) and the row statistics stats (N, 4: the largest logit and the sum of
// exp((z - largest) / tau), the same two of the teacher's entries) that
// wxx_distill_backward takes; logits (N, V) with row stride ld, top and ids (N, K).
WXX_EXPORT int wxx_distill_loss(float* loss, float* stats, const float* logits, int64_t ld,
                                const float* top, const uint32_t* ids, int64_t N, int64_t V, int K,
                                float tau) {
  WXX_REQUIRE_INIT();
  if (int st = check_sizes("wxx_distill_loss", N, V, K, tau)) return st;
  if (N == 0) return WXX_OK;
  const float inv_tau = 1.0f / tau;
  const Scale c = Scale::of(tau);
  const bool wide = (reinterpret_cast<uintptr_t>(stats) & 15) == 0;
  if (V <= kForwardV && K <= 32 * kForwardEntries && wide)
    return by_length<kForwardV>(V, [&](auto items) {
      distill_forward_rows_kernel<items.value>
          <<<(unsigned)((N + kRowWarps - 1) / kRowWarps), kRowWarps * 32, 0, wxx::stream()>>>(
              loss, stats, logits, ld, top, ids, N, (int)V, K, inv_tau, c, tau * tau,
              wxx::device_error_word());
      return wxx::after_launch(__FILE__, __LINE__);
    });
  int parts, length;
  split_row(N, V, parts, length);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(N * parts));
  cfg.blockDim = dim3(kT);
  cfg.stream = wxx::stream();
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {(unsigned)parts, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  WXX_CUDA_CHECK(cudaLaunchKernelEx(&cfg, distill_forward_kernel, loss, stats, logits, ld, top, ids,
                                    (int)V, K, parts, length, inv_tau, c, tau * tau,
                                    wxx::device_error_word()));
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}

// dz (N, V) from the gradient of the losses grad (N).
WXX_EXPORT int wxx_distill_backward(float* dz, const float* grad, const float* logits, int64_t ld,
                                    const float* top, const uint32_t* ids, const float* stats,
                                    int64_t N, int64_t V, int K, float tau) {
  WXX_REQUIRE_INIT();
  if (int st = check_sizes("wxx_distill_backward", N, V, K, tau)) return st;
  if (N == 0) return WXX_OK;
  WXX_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 15) == 0,
              "wxx_distill_backward: the statistics must be 16-byte aligned");
  const float inv_tau = 1.0f / tau;
  const Scale c = Scale::of(tau);
  if (V <= kBackwardV && K <= 32 * kBackwardEntries && N >= kBackwardN)
    return by_length<kBackwardV>(V, [&](auto items) {
      distill_backward_rows_kernel<items.value>
          <<<(unsigned)((N + kRowWarps - 1) / kRowWarps), kRowWarps * 32, 0, wxx::stream()>>>(
              dz, grad, logits, ld, top, ids, stats, N, (int)V, K, tau, inv_tau, c,
              wxx::device_error_word());
      return wxx::after_launch(__FILE__, __LINE__);
    });
  int parts, length;
  split_row(N, V, parts, length);
  const bool aligned = ((reinterpret_cast<uintptr_t>(dz) - reinterpret_cast<uintptr_t>(logits)) &
                        15) == 0 && (ld - V) % 4 == 0;
  auto kernel = aligned ? distill_backward_kernel<true> : distill_backward_kernel<false>;
  kernel<<<(unsigned)(N * parts), kT, 0, wxx::stream()>>>(
      dz, grad, logits, ld, top, ids, stats, (int)V, K, parts, length, tau, inv_tau, c,
      wxx::device_error_word());
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}
