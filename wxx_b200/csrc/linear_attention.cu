// Linear attention with a decay for each head:
//
//   S_t = l S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t,   l = exp(log_decay of the head)
//
// over q, k (B, T, H dk) and v (B, T, H dv), the state S (dk, dv) of a sequence's head
// starting from h0 or zero and taken as zero where reset (B, T) marks a new document.
// Backward, with R_t the gradient of S_t:
//
//   R_t = scale q_t do_t^T + l R_{t+1}  (R_{T-1} also takes dlast; cut at a reset of t + 1)
//   dq_t = scale S_t do_t,   dk_t = R_t v_t,   dv_t = R_t^T k_t,   dh0 = l R_0
//
// All of them are one operator, out_t = X_t^T x_t with X_t the decayed sum of y z^T, over
// (x, y, z) = (q, k, v) for o; (do, v, k) for dq; and backwards in time (k, q, do) for dv
// and (v, do, q) for dk: see Pass.

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace {

struct Operand {            // (B, T, heads * width) with unit stride inside
  const float* p;
  int64_t bs, ts;
};

// One sweep: out_t = out_scale X_t^T x_t over X_t = l X_{t-1} + y_scale y_t z_t^T, or with
// `back` over the positions from the last to the first, where l is applied after a
// position instead of before it.  x, y have p channels a head, z and out r.
struct Pass {
  Operand x, y, z;
  float* out;               // (B, T, H r)
  const float* from;        // X before the first position, NULL: zero
  float* last;              // X after the last one, NULL: not wanted
  int64_t p_stride, r_stride;   // of from and last within a head's p * r numbers
  int p, r;
  float y_scale, out_scale;
  int back;
};

struct Shape {
  const float* log_decay;   // (H)
  const uint32_t* reset;    // (B, T) or NULL
  int T, H;
};

constexpr int kT = 256;

// One position's decay of a state, l X.  A decay near 1 is applied as X + (l - 1) X: l alone
// is rounded to 2^-25, which n positions in a row make n 2^-25.
struct Decay {
  float less, whole;
  __device__ explicit Decay(float log_decay)
      : less(log_decay > -0.5f ? expm1f(log_decay) : expf(log_decay)),
        whole(log_decay > -0.5f ? 1.f : 0.f) {}
  __device__ __forceinline__ float operator()(float X) const { return fmaf(less, X, whole * X); }
};

// A block per sequence, head and 32 columns of X: lane = column, warp = every 8th row,
// K rows a thread.  One position after the other.
template <int K>
__global__ void __launch_bounds__(kT) sweep_kernel(const Pass a, const Shape s) {
  constexpr int kTile = K > 16 ? 8 : 16;      // positions of a tile
  __shared__ float sx[kTile][8 * K], sy[kTile][8 * K], sz[kTile][32], part[8][kTile][32];
  __shared__ int cut[kTile];
  const int slices = (a.r + 31) / 32;
  const int slice = blockIdx.x % slices, h = blockIdx.x / slices % s.H;
  const int64_t b = blockIdx.x / slices / s.H;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = slice * 32 + lane;
  const Decay l(s.log_decay[h]);
  const int64_t state = (b * s.H + h) * a.p * a.r;
  float X[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int p = warp + 8 * k;
    X[k] = a.from && p < a.p && c < a.r ? a.from[state + p * a.p_stride + c * a.r_stride] : 0.f;
  }
  const int tiles = (s.T + kTile - 1) / kTile;
  for (int i = 0; i < tiles; ++i) {
    const int t0 = (a.back ? tiles - 1 - i : i) * kTile, n = min(kTile, s.T - t0);
    __syncthreads();
    for (int e = threadIdx.x; e < kTile * 8 * K; e += kT) {
      const int t = e / (8 * K), p = e % (8 * K);
      const bool in = t < n && p < a.p;
      const int64_t at = (int64_t)h * a.p + p;
      sx[t][p] = in ? a.x.p[b * a.x.bs + (t0 + t) * a.x.ts + at] : 0.f;
      sy[t][p] = in ? a.y_scale * a.y.p[b * a.y.bs + (t0 + t) * a.y.ts + at] : 0.f;
    }
    for (int e = threadIdx.x; e < kTile * 32; e += kT) {
      const int t = e / 32, r = slice * 32 + e % 32;
      sz[t][e % 32] = t < n && r < a.r
                          ? a.z.p[b * a.z.bs + (t0 + t) * a.z.ts + (int64_t)h * a.r + r] : 0.f;
    }
    if (threadIdx.x < n) cut[threadIdx.x] = s.reset && s.reset[b * s.T + t0 + threadIdx.x] != 0;
    __syncthreads();
    for (int j = 0; j < n; ++j) {
      const int t = a.back ? n - 1 - j : j;
      const float z = sz[t][lane];
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!a.back) X[k] = cut[t] ? 0.f : l(X[k]);
        X[k] = fmaf(sy[t][warp + 8 * k], z, X[k]);
        sum = fmaf(sx[t][warp + 8 * k], X[k], sum);
        if (a.back) X[k] = cut[t] ? 0.f : l(X[k]);
      }
      part[warp][t][lane] = sum;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n * 32; e += kT) {
      const int t = e / 32, r = e % 32;
      float sum = 0.f;
      for (int w = 0; w < 8; ++w) sum += part[w][t][r];
      if (slice * 32 + r < a.r)
        a.out[((b * s.T + t0 + t) * s.H + h) * a.r + slice * 32 + r] = a.out_scale * sum;
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int p = warp + 8 * k;
    if (a.last && p < a.p && c < a.r) a.last[state + p * a.p_stride + c * a.r_stride] = X[k];
  }
}

// One position a sequence: a block per sequence, head and 32 columns of the state.
__global__ void __launch_bounds__(kT)
    step_kernel(float* __restrict__ o, float* __restrict__ state, const float* __restrict__ q,
                int64_t q_ld, const float* __restrict__ k, int64_t k_ld,
                const float* __restrict__ v, int64_t v_ld, const float* __restrict__ log_decay,
                int H, int dk, int dv, float scale) {
  __shared__ float part[8][32];
  const int slices = (dv + 31) / 32;
  const int slice = blockIdx.x % slices, h = blockIdx.x / slices % H;
  const int64_t b = blockIdx.x / slices / H;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = slice * 32 + lane;
  const Decay l(log_decay[h]);
  float* S = state + (b * H + h) * dk * dv;
  float sum = 0.f;
  if (c < dv) {
    const float z = v[b * v_ld + h * dv + c];
    for (int p = warp; p < dk; p += 8) {
      const float now = fmaf(k[b * k_ld + h * dk + p], z, l(S[(int64_t)p * dv + c]));
      S[(int64_t)p * dv + c] = now;
      sum = fmaf(q[b * q_ld + h * dk + p], now, sum);
    }
  }
  part[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && c < dv) {
    for (int w = 1; w < 8; ++w) sum += part[w][lane];
    o[(b * H + h) * dv + c] = scale * sum;
  }
}

int check_sizes(const char* what, int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv) {
  WXX_REQUIRE(B >= 0 && T >= 0 && H >= 0 && dk >= 0 && dv >= 0, "%s: negative size", what);
  WXX_REQUIRE(dk <= 256 && dv <= 256, "%s: heads of %lld and %lld channels (256 at most)", what,
              (long long)dk, (long long)dv);
  WXX_REQUIRE(T < (int64_t(1) << 31) - 256 && H < (int64_t(1) << 22) &&
                  B * H * 8 < (int64_t(1) << 31),
              "%s: too many positions, sequences or heads", what);
  return WXX_OK;
}

int sweep(const Pass& a, const Shape& s, int64_t B) {
  const unsigned grid = (unsigned)(B * s.H * ((a.r + 31) / 32));
  if (a.p <= 32)
    sweep_kernel<4><<<grid, kT, 0, wxx::stream()>>>(a, s);
  else if (a.p <= 64)
    sweep_kernel<8><<<grid, kT, 0, wxx::stream()>>>(a, s);
  else if (a.p <= 128)
    sweep_kernel<16><<<grid, kT, 0, wxx::stream()>>>(a, s);
  else
    sweep_kernel<32><<<grid, kT, 0, wxx::stream()>>>(a, s);
  return wxx::after_launch(__FILE__, __LINE__);
}

int copy_state(float* to, const float* from, int64_t n) {
  if (from)
    WXX_CUDA_CHECK(cudaMemcpyAsync(to, from, (size_t)n * sizeof(float), cudaMemcpyDeviceToDevice,
                                   wxx::stream()));
  else
    WXX_CUDA_CHECK(cudaMemsetAsync(to, 0, (size_t)n * sizeof(float), wxx::stream()));
  return WXX_OK;
}

int zero(float* to, int64_t n) { return n > 0 ? copy_state(to, nullptr, n) : WXX_OK; }

}  // namespace

// o (B, T, H dv) and last (B, H, dk, dv), the state after the last position; q, k, v with
// unit stride inside and the given batch and time strides; h0 (B, H, dk, dv) and reset
// (B, T) may be NULL.
WXX_EXPORT int wxx_linear_attention(float* o, float* last, const float* q, int64_t q_bs,
                                    int64_t q_ts, const float* k, int64_t k_bs, int64_t k_ts,
                                    const float* v, int64_t v_bs, int64_t v_ts,
                                    const float* log_decay, const float* h0,
                                    const uint32_t* reset, int64_t B, int64_t T, int64_t H,
                                    int64_t dk, int64_t dv, float scale) {
  WXX_REQUIRE_INIT();
  if (int st = check_sizes("wxx_linear_attention", B, T, H, dk, dv)) return st;
  if (B * H * dv == 0) return WXX_OK;
  if (dk == 0) return zero(o, B * T * H * dv);
  if (T == 0) return copy_state(last, h0, B * H * dk * dv);
  const Shape s{log_decay, reset, (int)T, (int)H};
  const Pass a{{q, q_bs, q_ts}, {k, k_bs, k_ts}, {v, v_bs, v_ts}, o, h0, last, dv, 1,
               (int)dk, (int)dv, 1.f, scale, 0};
  return sweep(a, s, B);
}

// dq, dk_out, dv_out (like q, k, v, dense) and dh0 (NULL: not wanted) from d_o, the
// gradient of the last state dlast (NULL: zero) and the forward's inputs.
WXX_EXPORT int wxx_linear_attention_backward(
    float* dq, float* dk_out, float* dv_out, float* dh0, const float* d_o, const float* dlast,
    const float* q, int64_t q_bs, int64_t q_ts, const float* k, int64_t k_bs, int64_t k_ts,
    const float* v, int64_t v_bs, int64_t v_ts, const float* log_decay, const float* h0,
    const uint32_t* reset, int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv, float scale) {
  WXX_REQUIRE_INIT();
  if (int st = check_sizes("wxx_linear_attention_backward", B, T, H, dk, dv)) return st;
  if (B * H * (dk + dv) == 0) return WXX_OK;
  if (dk == 0) return zero(dv_out, B * T * H * dv);
  if (dv == 0) {
    if (int st = zero(dq, B * T * H * dk)) return st;
    return zero(dk_out, B * T * H * dk);
  }
  if (T == 0) return dh0 ? copy_state(dh0, dlast, B * H * dk * dv) : WXX_OK;
  const Shape s{log_decay, reset, (int)T, (int)H};
  const Operand oq{q, q_bs, q_ts}, ok{k, k_bs, k_ts}, ov{v, v_bs, v_ts},
      od{d_o, T * H * dv, H * dv};
  const int K = (int)dk, V = (int)dv;
  const Pass passes[3] = {
      {od, ov, ok, dq, h0, nullptr, 1, dv, V, K, 1.f, scale, 0},
      {ok, oq, od, dv_out, dlast, dh0, dv, 1, K, V, scale, 1.f, 1},
      {ov, od, oq, dk_out, dlast, nullptr, 1, dv, V, K, scale, 1.f, 1}};
  for (const Pass& a : passes)
    if (int st = sweep(a, s, B)) return st;
  return WXX_OK;
}

// One position a sequence, in place: state (B, H, dk, dv) <- l state + k v^T, o (B, H dv) =
// scale state^T q; q, k, v with the given row strides.
WXX_EXPORT int wxx_linear_attention_step(float* o, float* state, const float* q, int64_t q_ld,
                                         const float* k, int64_t k_ld, const float* v,
                                         int64_t v_ld, const float* log_decay, int64_t B,
                                         int64_t H, int64_t dk, int64_t dv, float scale) {
  WXX_REQUIRE_INIT();
  if (int st = check_sizes("wxx_linear_attention_step", B, 1, H, dk, dv)) return st;
  if (B * H * dv == 0) return WXX_OK;
  step_kernel<<<(unsigned)(B * H * ((dv + 31) / 32)), kT, 0, wxx::stream()>>>(
      o, state, q, q_ld, k, k_ld, v, v_ld, log_decay, (int)H, (int)dk, (int)dv, scale);
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}
