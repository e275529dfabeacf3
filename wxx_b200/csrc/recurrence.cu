// Gated linear recurrence over time, per channel:
//
//   a_t = sigmoid(g_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t
//
// over x (B, T, D), with the gate logits g (B, T, H): head i's gate serves the
// D / H channels i D/H .. (i + 1) D/H - 1 (H = D: a gate per channel).  The
// state before position 0 is h0 (B, D) or zero, and where reset (B, T) is not
// zero a new document starts: the state before that position is zero.
//
// Backward, with G_t the total gradient of h_t and r_t = 0 at a reset, else 1:
//   G_t = dh_t + a_{t+1} r_{t+1} G_{t+1}          (G_{T-1} also takes dh_last)
//   dx_t = (1 - a_t) G_t
//   dg_t = sum over the head's channels of G_t (r_t h_{t-1} - x_t) a_t (1 - a_t)
//   dh0 = a_0 r_0 G_0

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

WXX_EXPORT int wxx_malloc(void** out, uint64_t nbytes);
WXX_EXPORT int wxx_free(void* p);
WXX_EXPORT int wxx_reduce(float* out, const float* x, int64_t outer, int64_t reduce, int64_t inner,
                          int mode);

namespace {

constexpr int kT = 256;

// a = sigmoid(g) and z = 1 - a = sigmoid(-g), each to a few ulp of itself:
// e = exp(-|g|) <= 1, the larger of the two is 1 / (1 + e), the other e times it.
__device__ __forceinline__ void gate_pair(float g, float& a, float& z) {
  const float e = expf(-fabsf(g));
  const float big = 1.0f / (1.0f + e), small = e * big;
  a = g >= 0.f ? big : small;
  z = g >= 0.f ? small : big;
  if (g != g) a = z = g;
}

// a h + z x as the larger-weighted of the two plus the smaller weight (<= 1/2)
// times their difference: a constant gate's fixed point stays where it is
// (a and z, each rounded, do not add up to 1: at z = 1e-3 their sum's error is
// multiplied by 1000), and a saturated gate keeps or replaces h exactly.
__device__ __forceinline__ float mix(float a, float z, float h, float x) {
  const bool keep = z <= a;
  const float base = keep ? h : x, other = keep ? x : h;
  return fmaf(keep ? z : a, other - base, base);
}

struct Operand {            // (B, T, ...) with unit stride inside
  const float* p;
  int64_t bs, ts;
};

// One thread per channel, position after position.
__global__ void recurrence_forward_kernel(float* __restrict__ h, float* __restrict__ h_last,
                                          Operand x, Operand g, const float* __restrict__ h0,
                                          const uint32_t* __restrict__ reset, int64_t B, int64_t T,
                                          int64_t D, int64_t per) {
  const int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x;
  if (i >= B * D) return;
  const int64_t b = i / D, d = i - b * D;
  float s = h0 ? h0[i] : 0.f;
  for (int64_t t = 0; t < T; ++t) {
    float a, z;
    gate_pair(g.p[b * g.bs + t * g.ts + d / per], a, z);
    if (reset && reset[b * T + t]) s = 0.f;
    s = mix(a, z, s, x.p[b * x.bs + t * x.ts + d]);
    h[(b * T + t) * D + d] = s;
  }
  h_last[i] = s;
}

__global__ void recurrence_backward_kernel(float* __restrict__ dx, float* __restrict__ dg,
                                           float* __restrict__ dh0, const float* __restrict__ dh,
                                           const float* __restrict__ dlast, Operand x, Operand g,
                                           const float* __restrict__ h,
                                           const float* __restrict__ h0,
                                           const uint32_t* __restrict__ reset, int64_t B,
                                           int64_t T, int64_t D, int64_t per) {
  const int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x;
  if (i >= B * D) return;
  const int64_t b = i / D, d = i - b * D;
  float carry = dlast ? dlast[i] : 0.f;
  for (int64_t t = T - 1; t >= 0; --t) {
    float a, z;
    gate_pair(g.p[b * g.bs + t * g.ts + d / per], a, z);
    const bool cut = reset && reset[b * T + t];
    const float before = cut ? 0.f : t > 0 ? h[(b * T + t - 1) * D + d] : h0 ? h0[i] : 0.f;
    const int64_t at = (b * T + t) * D + d;
    const float G = dh[at] + carry;
    dx[at] = z * G;
    dg[at] = G * (before - x.p[b * x.bs + t * x.ts + d]) * (a * z);
    carry = cut ? 0.f : a * G;
  }
  if (dh0) dh0[i] = carry;
}

__global__ void recurrence_step_kernel(float* __restrict__ state, const float* __restrict__ x,
                                       int64_t x_ld, const float* __restrict__ g, int64_t g_ld,
                                       int64_t n, int64_t D, int64_t per) {
  for (int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * kT) {
    const int64_t b = i / D, d = i - b * D;
    float a, z;
    gate_pair(g[b * g_ld + d / per], a, z);
    state[i] = mix(a, z, state[i], x[b * x_ld + d]);
  }
}

int check_sizes(const char* what, int64_t B, int64_t T, int64_t D, int64_t H) {
  WXX_REQUIRE(B >= 0 && T >= 0 && D >= 0 && H >= 0, "%s: negative size", what);
  WXX_REQUIRE(D == 0 || (H > 0 && D % H == 0), "%s: %lld channels are not a multiple of %lld heads",
              what, (long long)D, (long long)H);
  WXX_REQUIRE(B < (int64_t(1) << 31) && T < (int64_t(1) << 31) && D < (int64_t(1) << 31),
              "%s: a size is 2^31 or more", what);
  return WXX_OK;
}

}  // namespace

// h (B, T, D) and the state after the last position, h_last (B, D); x (B, T, D)
// and gate (B, T, H) have unit stride inside and the given batch and time
// strides; h0 (B, D) and reset (B, T) may be NULL.
WXX_EXPORT int wxx_gated_recurrence(float* h, float* h_last, const float* x, int64_t x_bs,
                                    int64_t x_ts, const float* gate, int64_t g_bs, int64_t g_ts,
                                    const float* h0, const uint32_t* reset, int64_t B, int64_t T,
                                    int64_t D, int64_t H) {
  WXX_REQUIRE_INIT();
  if (int st = check_sizes("wxx_gated_recurrence", B, T, D, H)) return st;
  if (B * D == 0) return WXX_OK;
  const int64_t blocks = (B * D + kT - 1) / kT;
  recurrence_forward_kernel<<<(unsigned)blocks, kT, 0, wxx::stream()>>>(
      h, h_last, Operand{x, x_bs, x_ts}, Operand{gate, g_bs, g_ts}, h0, reset, B, T, D, D / H);
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}

// Gradients of wxx_gated_recurrence: dx (B, T, D), dgate (B, T, H) and dh0
// (B, D; NULL: not wanted) from dh (B, T, D), dlast (B, D; NULL: zero), the
// forward's inputs and its h.
WXX_EXPORT int wxx_gated_recurrence_backward(float* dx, float* dgate, float* dh0, const float* dh,
                                             const float* dlast, const float* x, int64_t x_bs,
                                             int64_t x_ts, const float* gate, int64_t g_bs,
                                             int64_t g_ts, const float* h, const float* h0,
                                             const uint32_t* reset, int64_t B, int64_t T, int64_t D,
                                             int64_t H) {
  WXX_REQUIRE_INIT();
  if (int st = check_sizes("wxx_gated_recurrence_backward", B, T, D, H)) return st;
  if (B * D == 0) return WXX_OK;
  float* wide = dgate;
  void* scratch = nullptr;
  if (H != D && T > 0) {
    if (int st = wxx_malloc(&scratch, (uint64_t)(B * T * D) * sizeof(float))) return st;
    wide = static_cast<float*>(scratch);
  }
  const int64_t blocks = (B * D + kT - 1) / kT;
  recurrence_backward_kernel<<<(unsigned)blocks, kT, 0, wxx::stream()>>>(
      dx, wide, dh0, dh, dlast, Operand{x, x_bs, x_ts}, Operand{gate, g_bs, g_ts}, h, h0, reset, B,
      T, D, D / H);
  int st = wxx::after_launch(__FILE__, __LINE__);
  if (scratch) {
    if (st == WXX_OK) st = wxx_reduce(dgate, wide, B * T * H, D / H, 1, 0);
    wxx_free(scratch);
  }
  return st;
}

// One position per sequence: state (B, D) <- a state + (1 - a) x in place,
// x (B, D) and gate (B, H) with row strides x_ld and g_ld.
WXX_EXPORT int wxx_gated_recurrence_step(float* state, const float* x, int64_t x_ld,
                                         const float* gate, int64_t g_ld, int64_t B, int64_t D,
                                         int64_t H) {
  WXX_REQUIRE_INIT();
  if (int st = check_sizes("wxx_gated_recurrence_step", B, 1, D, H)) return st;
  const int64_t n = B * D;
  if (n == 0) return WXX_OK;
  recurrence_step_kernel<<<wxx::grid_for(n, kT), kT, 0, wxx::stream()>>>(state, x, x_ld, gate, g_ld,
                                                                         n, D, D / H);
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}
