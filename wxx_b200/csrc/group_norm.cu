// Group norm over trailing channels with an activation:
//
//   z = (x - mean) inv,  n = gamma z + beta,  y = act(n)  or  n act(gate)
//
// over x (N, S, C): mean and inv = 1 / sqrt(var + eps) of each sample's groups of C / G
// neighbouring channels over all S positions.  Backward, with dn the gradient of n
// (dy act'(n), or dy act(gate)) and u = gamma dn:
//
//   dx = inv (u - mean(u) - z mean(u z)),  dgate = dy n act'(gate)
//   dgamma = sum of dn z,  dbeta = sum of dn  over samples and positions
//
// Memory-bound: the floor reads x (gate, dy) and writes y (dx, dgate) once.

#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common.cuh"

WXX_EXPORT int wxx_malloc(void** out, uint64_t nbytes);
WXX_EXPORT int wxx_free(void* p);

namespace {

constexpr int kT = 256;

enum Act { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

// sigmoid(v) and sigmoid(-v), each good to a few ulp of itself, from e = exp(-|v|) <= 1: e = 2^y
// 2^r with y = -|v| log2 e rounded and r what the product and the constant lost (alone y would
// cost e |y| half ulps), so little that 2^r is 1 + r log 2; 1 + e is what the approximate
// reciprocal takes to an ulp.  From |v| = 87.3 on, where 2^y is below 2^-126, e is taken as 0: SiLU's
// last values above 2^-126 in size, between -92 and there, are 0.  (With the library's exponential and
// division the forward over 8192 x 1024 was bound by its instructions: 28.7 us.)
struct Sigmoid {
  float of, rest;
};
// For two numbers, so that products and sums go in pairs.
__device__ __forceinline__ void sigmoid2(float v0, float v1, Sigmoid& s0, Sigmoid& s1) {
  constexpr float kC = -1.4426950408889634f;
  constexpr float kLow = (float)(-1.4426950408889634 - (double)kC);
  constexpr float kLog2 = 0.6931471805599453f;
  float t0, t1, y0, y1, l0, l1, e0, e1, d0, d1, r0, r1, m0, m1;
  asm("min.NaN.f32 %0, %1, 0f42D00000;" : "=f"(t0) : "f"(fabsf(v0)));   // 104
  asm("min.NaN.f32 %0, %1, 0f42D00000;" : "=f"(t1) : "f"(fabsf(v1)));
  mul2(y0, y1, t0, t1, kC, kC);
  fma2(l0, l1, t0, t1, kC, kC, -y0, -y1);
  fma2(l0, l1, t0, t1, kLow, kLow, l0, l1);
  fma2(l0, l1, l0, l1, kLog2, kLog2, 1.0f, 1.0f);
  mul2(e0, e1, fast_exp2(y0), fast_exp2(y1), l0, l1);
  add2(d0, d1, e0, e1, 1.0f, 1.0f);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(d0));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(d1));
  mul2(m0, m1, e0, e1, r0, r1);
  s0 = v0 >= 0.f ? Sigmoid{r0, m0} : Sigmoid{m0, r0};
  s1 = v1 >= 0.f ? Sigmoid{r1, m1} : Sigmoid{m1, r1};
}

// 1 / sqrt(a) of a normal number: the approximation and one step of Newton's method.
__device__ __forceinline__ float inverse_root(float a) {
  const float r = rsqrtf(a);
  return fmaf(r * 0.5f, fmaf(-a * r, r, 1.0f), r);
}

// GELU is the tanh form with the clamps of gelu_tanh, as v sigmoid(2 u).
__device__ __forceinline__ void gelu_arguments(float v0, float v1, float& u0, float& u1) {
  constexpr float k2C = 2.0f * 0.7978845608f;
  mul2(u0, u1, v0, v1, v0, v1);
  fma2(u0, u1, u0, u1, 0.044715f, 0.044715f, 1.0f, 1.0f);
  mul2(u0, u1, u0, u1, v0, v1);
  mul2(u0, u1, u0, u1, k2C, k2C);
}
__device__ __forceinline__ float clamped(float v, float high, float middle, float low) {
  return v > 10.f ? high : v < -10.f ? low : middle;
}

// Sums for a mean are made of 2^-16 of the numbers: as good, and those of 2^14 numbers of 2^126 fit.
// Squared distances from the mean overflow from 2^64 / sqrt(n) on: their sum is then made of
// distances in units of 2^80, of which 2^24 fit.
constexpr float kDown = 0x1p-16f, kUp = 0x1p16f, kFar = 0x1p-80f;
__device__ __forceinline__ float far_inverse(float variance, float eps) {
  return inverse_root(fmaf(eps * kFar, kFar, variance)) * kFar;
}

// The activations of two numbers, in place.
template <int ACT>
__device__ __forceinline__ void act2(float& v0, float& v1) {
  if (ACT == kRelu) {
    v0 = v0 < 0.f ? 0.f : v0;
    v1 = v1 < 0.f ? 0.f : v1;
  } else if (ACT != kNone) {
    float u0 = v0, u1 = v1;
    Sigmoid p0, p1;
    if (ACT == kGelu) gelu_arguments(v0, v1, u0, u1);
    sigmoid2(u0, u1, p0, p1);
    mul2(u0, u1, v0, v1, p0.of, p1.of);
    v0 = ACT == kGelu ? clamped(v0, v0, u0, 0.f) : u0;
    v1 = ACT == kGelu ? clamped(v1, v1, u1, 0.f) : u1;
  }
}

// The activations of two numbers, in place, and their slopes.
template <int ACT>
__device__ __forceinline__ void act_slope2(float& v0, float& v1, float& s0, float& s1) {
  s0 = s1 = 1.f;
  if (ACT == kRelu) {
    s0 = v0 > 0.f ? 1.f : 0.f;
    s1 = v1 > 0.f ? 1.f : 0.f;
    v0 = v0 < 0.f ? 0.f : v0;
    v1 = v1 < 0.f ? 0.f : v1;
  } else if (ACT == kSilu) {
    Sigmoid p0, p1;
    sigmoid2(v0, v1, p0, p1);
    mul2(v0, v1, v0, v1, p0.of, p1.of);
    fma2(s0, s1, v0, v1, p0.rest, p1.rest, p0.of, p1.of);
  } else if (ACT == kGelu) {
    constexpr float k2C = 2.0f * 0.7978845608f;
    Sigmoid p0, p1;
    float u0, u1, w0, w1;
    gelu_arguments(v0, v1, u0, u1);
    sigmoid2(u0, u1, p0, p1);
    mul2(u0, u1, v0, v1, v0, v1);
    fma2(u0, u1, u0, u1, 0.134145f * k2C, 0.134145f * k2C, k2C, k2C);     // of the argument
    mul2(w0, w1, v0, v1, p0.of, p1.of);
    mul2(u0, u1, u0, u1, p0.rest, p1.rest);
    fma2(s0, s1, w0, w1, u0, u1, p0.of, p1.of);
    s0 = clamped(v0, 1.f, s0, 0.f);
    s1 = clamped(v1, 1.f, s1, 0.f);
    v0 = clamped(v0, v0, w0, 0.f);
    v1 = clamped(v1, v1, w1, 0.f);
  }
}

// For V numbers where the activation is one branch for all threads.
template <int ACT, int V>
__device__ __forceinline__ void act_all(float (&v)[V]) {
  float unused = 0.f;
#pragma unroll
  for (int e = 0; e < V; e += 2) act2<ACT>(v[e], e + 1 < V ? v[e + 1] : unused);
}
template <int V>
__device__ __forceinline__ void act_all(int code, float (&v)[V]) {
  if (code == kSilu)
    act_all<kSilu, V>(v);
  else if (code == kGelu)
    act_all<kGelu, V>(v);
  else if (code == kRelu)
    act_all<kRelu, V>(v);
}
template <int ACT, int V>
__device__ __forceinline__ void act_slope_all(float (&v)[V], float (&s)[V]) {
  float unused = 0.f, none;
#pragma unroll
  for (int e = 0; e < V; e += 2)
    act_slope2<ACT>(v[e], e + 1 < V ? v[e + 1] : unused, s[e], e + 1 < V ? s[e + 1] : none);
}
template <int V>
__device__ __forceinline__ void act_slope_all(int code, float (&v)[V], float (&s)[V]) {
  if (code == kSilu)
    act_slope_all<kSilu, V>(v, s);
  else if (code == kGelu)
    act_slope_all<kGelu, V>(v, s);
  else if (code == kRelu)
    act_slope_all<kRelu, V>(v, s);
  else
    act_slope_all<kNone, V>(v, s);
}

// V numbers at a time, in pairs.
template <int V>
__device__ __forceinline__ void add_all(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
#pragma unroll
  for (int e = 0; e + 1 < V; e += 2) add2(d[e], d[e + 1], a[e], a[e + 1], b[e], b[e + 1]);
  if (V % 2) d[V - 1] = a[V - 1] + b[V - 1];
}
template <int V>
__device__ __forceinline__ void sub_all(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
#pragma unroll
  for (int e = 0; e + 1 < V; e += 2) sub2(d[e], d[e + 1], a[e], a[e + 1], b[e], b[e + 1]);
  if (V % 2) d[V - 1] = a[V - 1] - b[V - 1];
}
template <int V>
__device__ __forceinline__ void mul_all(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
#pragma unroll
  for (int e = 0; e + 1 < V; e += 2) mul2(d[e], d[e + 1], a[e], a[e + 1], b[e], b[e + 1]);
  if (V % 2) d[V - 1] = a[V - 1] * b[V - 1];
}
template <int V>
__device__ __forceinline__ void fma_all(float (&d)[V], const float (&a)[V], const float (&b)[V],
                                        const float (&c)[V]) {
#pragma unroll
  for (int e = 0; e + 1 < V; e += 2)
    fma2(d[e], d[e + 1], a[e], a[e + 1], b[e], b[e + 1], c[e], c[e + 1]);
  if (V % 2) d[V - 1] = fmaf(a[V - 1], b[V - 1], c[V - 1]);
}
template <int V>
__device__ __forceinline__ void fill(float (&d)[V], float v) {
#pragma unroll
  for (int e = 0; e < V; ++e) d[e] = v;
}
template <int V>
__device__ __forceinline__ float total(const float (&v)[V]) {
  if constexpr (V == 4) return (v[0] + v[1]) + (v[2] + v[3]);
  float sum = v[0];
#pragma unroll
  for (int e = 1; e < V; ++e) sum += v[e];
  return sum;
}

template <int V>
struct Pack {
  float v[V];
};
template <int V>
__device__ __forceinline__ Pack<V> load(const float* p) {
  Pack<V> out;
  if constexpr (V == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    out.v[0] = t.x, out.v[1] = t.y, out.v[2] = t.z, out.v[3] = t.w;
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) out.v[e] = p[e];
  }
  return out;
}
template <int V>
__device__ __forceinline__ void store(float* p, const Pack<V>& a) {
  if constexpr (V == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(a.v[0], a.v[1], a.v[2], a.v[3]);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) p[e] = a.v[e];
  }
}

// A sum over neighbouring lanes, a power of two of them.
__device__ __forceinline__ float over_lanes(float v, int lanes) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A count of values with their mean and the sum of their squared distances from it.
struct Moments {
  float n, mean, m2;
};
__device__ __forceinline__ Moments join(Moments a, Moments b) {
  const float n = a.n + b.n;
  if (n == 0.f) return a;
  const float d = b.mean - a.mean, w = b.n / n;
  return {n, fmaf(d, w, a.mean), a.m2 + b.m2 + d * d * a.n * w};
}

struct Shape {
  int64_t N, S;
  int C, G, per;
  int chunks;           // pieces of a sample's positions
  int64_t piece;        // positions of a piece
  float eps;
};

// A block's threads over (position, channel): `wide` neighbouring channels by kT / wide
// positions, so that channels of a position are read together.
struct Lanes {
  int wide, c, row, rows;
  __device__ Lanes(int C) {
    wide = C < kT ? C : kT;
    rows = kT / wide;
    c = threadIdx.x % wide;
    row = threadIdx.x / wide;          // rows: a thread past the last whole position
  }
};

// The moments of each group over a piece of a sample: part (N, chunks, G).  Means are joined as
// distances from one of them: joined themselves, each is rounded to u of its size, and one after the
// other they left the mean of 2352 channels 5 deviations from 0 off by 50 u of it.
__global__ void __launch_bounds__(kT)
    moments_kernel(Moments* __restrict__ part, const float* __restrict__ x, const Shape s) {
  __shared__ Moments sums[kT], here[kT];
  const int64_t n = blockIdx.x / s.chunks;
  const int64_t p0 = (blockIdx.x % s.chunks) * s.piece;
  const int64_t p1 = p0 + s.piece < s.S ? p0 + s.piece : s.S;
  const float* xn = x + n * s.S * s.C;
  const Lanes l(s.C);
  Moments group = {0.f, 0.f, 0.f};     // of group threadIdx.x, in parts of kT groups; from `base`
  float base = 0.f;
  for (int g0 = 0; g0 < s.G; g0 += kT) {
    group = {0.f, 0.f, 0.f};
    const int gs = g0 + kT < s.G ? g0 + kT : s.G;
    for (int c0 = g0 * s.per; c0 < gs * s.per; c0 += l.wide) {
      const int c = c0 + l.c;
      Moments m = {0.f, 0.f, 0.f};
      if (l.row < l.rows && c < gs * s.per) {
        const float first = p0 + l.row < p1 ? xn[(p0 + l.row) * s.C + c] : 0.f;
        for (int64_t p = p0 + l.row; p < p1; p += l.rows) {
          const float v = xn[p * s.C + c] - first;
          m.n += 1.f;
          const float d = v - m.mean;
          m.mean += d / m.n;
          m.m2 += d * (v - m.mean);
        }
        m.mean += first;
      }
      sums[threadIdx.x] = m;
      __syncthreads();
      // the groups among these channels, each by a thread or, where it has many moments, a warp
      const int lanes = min(s.per, l.wide) * l.rows >= 16 ? 32 : 1, lane = threadIdx.x % lanes;
      const int end = min(gs, (c0 + l.wide - 1) / s.per + 1);
      for (int g = c0 / s.per + threadIdx.x / lanes; g < end; g += kT / lanes) {
        const int from = max(g * s.per, c0), to = min((g + 1) * s.per, c0 + l.wide);
        const int span = to - from, count = span * l.rows;
        const float n = (float)span * (float)(p1 - p0), share = 1.f / n;
        const float first = sums[from - c0].mean;
        float off = 0.f, rest = 0.f, m2 = 0.f;        // rest: what the first sum's roundings left
        for (int k = lane; k < count; k += lanes) {
          const Moments& e = sums[k / span * l.wide + from - c0 + k % span];
          off = fmaf(e.n * share, e.mean - first, off);
        }
        off = over_lanes(off, lanes);
        for (int k = lane; k < count; k += lanes) {
          const Moments& e = sums[k / span * l.wide + from - c0 + k % span];
          const float d = e.mean - first - off;
          rest = fmaf(e.n * share, d, rest);
          m2 += fmaf(e.n * d, d, e.m2);
        }
        rest = over_lanes(rest, lanes);
        m2 = over_lanes(m2, lanes);
        if (lane == 0) here[g - g0] = {n, first + (off + rest), m2};
      }
      __syncthreads();
      const int own = g0 + threadIdx.x;
      if (own < gs && own >= c0 / s.per && own < end) {
        const Moments e = here[threadIdx.x];
        if (group.n == 0.f) base = e.mean;
        group = join(group, {e.n, e.mean - base, e.m2});
      }
    }
    group.mean += base;
    if (g0 + threadIdx.x < gs) part[(int64_t)blockIdx.x * s.G + g0 + threadIdx.x] = group;
  }
}

// mean and inv (N, G) from the pieces' moments.
__global__ void __launch_bounds__(kT)
    statistics_kernel(float* __restrict__ mean, float* __restrict__ inv,
                      const Moments* __restrict__ part, const float* __restrict__ x, const Shape s) {
  __shared__ bool far[kT];
  __shared__ float sums[kT / 32];
  const int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x;
  const float count = (float)s.S * (float)s.per;
  bool range = true;
  if (i < s.N * s.G) {
    const int64_t n = i / s.G;
    const int g = (int)(i - n * s.G);
    const Moments* of = part + n * s.chunks * s.G + g;
    Moments m = {0.f, 0.f, 0.f};
    for (int k = 0; k < s.chunks; ++k) {
      const Moments e = of[(int64_t)k * s.G];
      m = join(m, {e.n, e.mean - of->mean, e.m2});
    }
    const float variance = m.m2 / count;
    mean[i] = of->mean + m.mean;
    inv[i] = inverse_root(variance + s.eps);
    range = variance < INFINITY;
  }
  far[threadIdx.x] = !range;
  if (!__syncthreads_or(!range)) return;
  // the groups out of range one after the other, by all threads
  auto block_sum = [&](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = v;
    __syncthreads();
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < kT / 32; ++w) all += sums[w];
    __syncthreads();
    return all;
  };
  for (int t = 0; t < kT; ++t) {
    if (!far[t]) continue;
    const int64_t j = (int64_t)blockIdx.x * kT + t, n = j / s.G;
    const float* group = x + n * s.S * s.C + (j - n * s.G) * s.per;
    const int64_t numbers = s.S * s.per;
    const float mu = mean[j];
    float squares = 0.f;
    for (int64_t k = threadIdx.x; k < numbers; k += kT) {
      const float d = (group[k / s.per * s.C + k % s.per] - mu) * kFar;
      squares = fmaf(d, d, squares);
    }
    const float all = block_sum(squares);
    if (threadIdx.x == 0) inv[j] = far_inverse(all / count, s.eps);
  }
}

template <bool GATED>
__global__ void __launch_bounds__(kT)
    apply_kernel(float* __restrict__ y, const float* __restrict__ x,
                 const float* __restrict__ gate, const float* __restrict__ mean,
                 const float* __restrict__ inv, const float* __restrict__ gamma,
                 const float* __restrict__ beta, const Shape s, const int code) {
  const int64_t sample = s.S * s.C, total = s.N * sample;
  for (int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * kT) {
    const int64_t n = i / sample;
    const int c = (int)((i - n * sample) % s.C);
    const int64_t g = n * s.G + c / s.per;
    const float z = (x[i] - mean[g]) * inv[g];
    const float normal = fmaf(z, gamma ? gamma[c] : 1.f, beta ? beta[c] : 0.f);
    float v[1] = {GATED ? gate[i] : normal};
    act_all<1>(code, v);
    y[i] = GATED ? normal * v[0] : v[0];
  }
}

// From dy the gradients of n and, where GATED, of the gate (in its place), at V places.
template <int V, bool GATED>
__device__ __forceinline__ void inner_gradient(int code, float (&d)[V], const float (&z)[V],
                                               const float (&gamma)[V], const float (&beta)[V],
                                               float (&gate)[V]) {
  float n[V], value[V], slope[V];
  fma_all<V>(n, z, gamma, beta);
#pragma unroll
  for (int e = 0; e < V; ++e) value[e] = GATED ? gate[e] : n[e];
  act_slope_all<V>(code, value, slope);
  if constexpr (GATED) {
    mul_all<V>(n, n, slope);
    mul_all<V>(gate, n, d);
    mul_all<V>(d, d, value);
  } else {
    mul_all<V>(d, d, slope);
  }
}

// For every channel the sums of dn and dn z over a piece of a sample: part (N, chunks,
// 2, C).
template <bool GATED>
__global__ void __launch_bounds__(kT)
    channel_sums_kernel(float* __restrict__ part, const float* __restrict__ dy,
                        const float* __restrict__ x, const float* __restrict__ gate,
                        const float* __restrict__ mean, const float* __restrict__ inv,
                        const float* __restrict__ gamma, const float* __restrict__ beta,
                        const Shape s, const int code) {
  __shared__ float sums[2][kT];
  const int64_t n = blockIdx.x / s.chunks;
  const int64_t p0 = (blockIdx.x % s.chunks) * s.piece;
  const int64_t p1 = p0 + s.piece < s.S ? p0 + s.piece : s.S;
  const int64_t at = n * s.S * s.C;
  const Lanes l(s.C);
  for (int c0 = 0; c0 < s.C; c0 += l.wide) {
    const int c = c0 + l.c;
    float a = 0.f, b = 0.f;
    if (l.row < l.rows && c < s.C) {
      const int64_t g = n * s.G + c / s.per;
      const float mu = mean[g], is = inv[g];
      const float ga[1] = {gamma ? gamma[c] : 1.f}, be[1] = {beta ? beta[c] : 0.f};
      for (int64_t p = p0 + l.row; p < p1; p += l.rows) {
        const int64_t i = at + p * s.C + c;
        const float z[1] = {(x[i] - mu) * is};
        float dn[1] = {dy[i]}, w[1] = {GATED ? gate[i] : 0.f};
        inner_gradient<1, GATED>(code, dn, z, ga, be, w);
        a += dn[0];
        b = fmaf(dn[0], z[0], b);
      }
    }
    sums[0][threadIdx.x] = a;
    sums[1][threadIdx.x] = b;
    __syncthreads();
    if (l.row == 0 && c < s.C) {
      for (int r = 1; r < l.rows; ++r) {
        a += sums[0][r * l.wide + l.c];
        b += sums[1][r * l.wide + l.c];
      }
      float* out = part + (int64_t)blockIdx.x * 2 * s.C;
      out[c] = a;
      out[s.C + c] = b;
    }
    __syncthreads();
  }
}

// The means of u and u z of every group: sums (N, G, 2).
__global__ void __launch_bounds__(kT)
    group_sums_kernel(float2* __restrict__ sums, const float* __restrict__ part,
                      const float* __restrict__ gamma, const Shape s) {
  const int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x;
  if (i >= s.N * s.G) return;
  const int64_t n = i / s.G;
  const int g = (int)(i - n * s.G);
  float a = 0.f, b = 0.f;
  for (int k = 0; k < s.chunks; ++k) {
    const float* row = part + (n * s.chunks + k) * 2 * s.C;
    for (int c = g * s.per; c < (g + 1) * s.per; ++c) {
      const float ga = gamma ? gamma[c] : 1.f;
      a = fmaf(ga, row[c], a);
      b = fmaf(ga, row[s.C + c], b);
    }
  }
  const float count = (float)s.S * (float)s.per;
  sums[i] = make_float2(a / count, b / count);
}

template <bool GATED>
__global__ void __launch_bounds__(kT)
    input_gradient_kernel(float* __restrict__ dx, float* __restrict__ dgate,
                          const float* __restrict__ dy, const float* __restrict__ x,
                          const float* __restrict__ gate, const float* __restrict__ mean,
                          const float* __restrict__ inv, const float* __restrict__ gamma,
                          const float* __restrict__ beta, const float2* __restrict__ sums,
                          const Shape s, const int code) {
  const int64_t sample = s.S * s.C, total = s.N * sample;
  for (int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * kT) {
    const int64_t n = i / sample;
    const int c = (int)((i - n * sample) % s.C);
    const int64_t g = n * s.G + c / s.per;
    const float is = inv[g], z[1] = {(x[i] - mean[g]) * is};
    const float ga[1] = {gamma ? gamma[c] : 1.f}, be[1] = {beta ? beta[c] : 0.f};
    float dn[1] = {dy[i]}, w[1] = {GATED ? gate[i] : 0.f};
    inner_gradient<1, GATED>(code, dn, z, ga, be, w);
    const float2 m = sums[g];
    dx[i] = is * (ga[0] * dn[0] - m.x - z[0] * m.y);
    if (GATED) dgate[i] = w[0];
  }
}

// out (2, C) from rows of 2 C partial sums, in a fixed order: 16 columns by 64 parts of
// the rows a block (32 by 32 has half as many blocks and twice the rows a thread, 0.8 us longer over
// 592 rows of 2 x 1024).  First dbeta, then dgamma.
__global__ void __launch_bounds__(1024)
    column_sums_kernel(float* __restrict__ dbeta, float* __restrict__ dgamma,
                       const float* __restrict__ part, int64_t rows, int C) {
  __shared__ float sums[64][17];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int column = threadIdx.x & 15, share = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + column;
  float a = 0.f;
  if (c < 2 * C) {
    const float* p = part + c;
    int64_t r = share;
    for (; r + 448 < rows; r += 512) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = p[(r + 64 * k) * 2 * C];
      a += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    float v[7];
#pragma unroll
    for (int k = 0; k < 7; ++k) v[k] = r + 64 * k < rows ? p[(r + 64 * k) * 2 * C] : 0.f;
    a += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + v[6]);
  }
  sums[share][column] = a;
  __syncthreads();
  if (warp >= 16) return;
  float v = sums[lane][warp] + sums[lane + 32][warp];      // a warp a column now
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int own = blockIdx.x * 16 + warp;
  if (lane == 0 && own < 2 * C) (own < C ? dbeta[own] : dgamma[own - C]) = v;
}

// ------------------------------------------------------------------ one position a sample
//
// A group is `lanes` threads' registers (a power of two up to 32, K pieces of V channels
// each), so x, the gate and dy are read once.  Backward a thread keeps its channels from
// sample to sample and with them the sums for dgamma and dbeta: `rows` samples are under
// way at once, and as many partial sums are added up by column_sums_kernel.

struct Few {
  int64_t N;
  int C, G, per, lanes, rows, code;
  float eps;
};

template <int V, int K, bool GATED>
__global__ void __launch_bounds__(kT)
    token_kernel(float* __restrict__ y, float* __restrict__ mean, float* __restrict__ inv,
                 const float* __restrict__ x, const float* __restrict__ gate,
                 const float* __restrict__ gamma, const float* __restrict__ beta, const Few f) {
  // a thread's group of channels, and its first sample
  const unsigned slot = (blockIdx.x * kT + threadIdx.x) / f.lanes;
  const int lane = threadIdx.x % f.lanes, g = slot % f.G, row = slot / f.G;
  const bool here = row < f.rows;
  const float share = 1.0f / (float)f.per;
  const unsigned group = f.lanes == 32 ? 0xffffffffu                // the lanes of this group
                                       : ((1u << f.lanes) - 1) << (threadIdx.x & 31 & -f.lanes);
  Pack<V> ga[K], be[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * f.lanes + lane) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) ga[k].v[e] = 1.f, be[k].v[e] = 0.f;
    if (gamma && c < f.per) ga[k] = load<V>(gamma + g * f.per + c);
    if (beta && c < f.per) be[k] = load<V>(beta + g * f.per + c);
  }
  // every lane of a warp takes as many turns (rows differ by one at most)
  for (int64_t n = row; __any_sync(0xffffffffu, here && n < f.N); n += f.rows) {
    const bool on = here && n < f.N;
    const int64_t at = n * f.C + g * f.per;
    Pack<V> v[K], w[GATED ? K : 1];
    float sums[V], means[V], downs[V], units[V];
    fill<V>(sums, 0.f);
    fill<V>(downs, kDown);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * f.lanes + lane) * V;
      const bool in = on && c < f.per;
#pragma unroll
      for (int e = 0; e < V; ++e) v[k].v[e] = 0.f;
      if (in) v[k] = load<V>(x + at + c);
      if (GATED && in) w[k] = load<V>(gate + at + c);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) fma_all<V>(sums, v[k].v, downs, sums);
    const float mu = over_lanes(total<V>(sums), f.lanes) * (share * kUp);
    fill<V>(means, mu);
    fill<V>(sums, 0.f);
    // (the unit of a group by a vote; a branch that makes the sum again, and its code between the
    // rest, cost one position of 32 x 1024 0.5 us)
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      sub_all<V>(v[k].v, v[k].v, means);
      if ((k * f.lanes + lane) * V < f.per)
#pragma unroll
        for (int e = 0; e < V; ++e) top = fmaxf(top, fabsf(v[k].v[e]));
    }
    const bool far = (__ballot_sync(0xffffffffu, top >= 0x1p58f) & group) != 0;
    const float unit = far ? kFar : 1.f;
    fill<V>(units, unit);
#pragma unroll
    for (int k = 0; k < K; ++k)
      if ((k * f.lanes + lane) * V < f.per) {
        float d[V];
        mul_all<V>(d, v[k].v, units);
        fma_all<V>(sums, d, d, sums);
      }
    const float is = inverse_root(fmaf(over_lanes(total<V>(sums), f.lanes), share, f.eps * unit * unit)) * unit;
    if (!on) continue;
    if (lane == 0) {
      mean[n * f.G + g] = mu;
      inv[n * f.G + g] = is;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * f.lanes + lane) * V;
      if (c >= f.per) continue;
      float scales[V];
      fill<V>(scales, is);
      mul_all<V>(v[k].v, v[k].v, scales);
      fma_all<V>(v[k].v, v[k].v, ga[k].v, be[k].v);
      if constexpr (GATED) {
        act_all<V>(f.code, w[k].v);
        mul_all<V>(v[k].v, v[k].v, w[k].v);
      } else {
        act_all<V>(f.code, v[k].v);
      }
      store<V>(y + at + c, v[k]);
    }
  }
}

template <int V, int K, bool GATED>
__global__ void __launch_bounds__(kT)
    token_backward_kernel(float* __restrict__ dx, float* __restrict__ dgate,
                          float* __restrict__ part, const float* __restrict__ dy,
                          const float* __restrict__ x, const float* __restrict__ gate,
                          const float* __restrict__ mean, const float* __restrict__ inv,
                          const float* __restrict__ gamma, const float* __restrict__ beta,
                          const Few f) {
  // a thread's group of channels, and its first sample
  const unsigned slot = (blockIdx.x * kT + threadIdx.x) / f.lanes;
  const int lane = threadIdx.x % f.lanes, g = slot % f.G, row = slot / f.G;
  const bool here = row < f.rows;
  const float share = 1.0f / (float)f.per;
  Pack<V> ga[K], be[K], sum_n[K], sum_z[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * f.lanes + lane) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) ga[k].v[e] = 1.f, be[k].v[e] = sum_n[k].v[e] = sum_z[k].v[e] = 0.f;
    if (gamma && c < f.per) ga[k] = load<V>(gamma + g * f.per + c);
    if (beta && c < f.per) be[k] = load<V>(beta + g * f.per + c);
  }
  // every lane of a warp takes as many turns (rows differ by one at most)
  for (int64_t n0 = row; __any_sync(0xffffffffu, here && n0 < f.N); n0 += f.rows) {
    const bool on = here && n0 < f.N;
    const int64_t at = n0 * f.C + g * f.per;
    const float mu = on ? mean[n0 * f.G + g] : 0.f, is = on ? inv[n0 * f.G + g] : 0.f;
    Pack<V> z[K], d[K], w[GATED ? K : 1];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * f.lanes + lane) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) z[k].v[e] = mu, d[k].v[e] = 0.f;
      if (GATED)
#pragma unroll
        for (int e = 0; e < V; ++e) w[k].v[e] = 0.f;
      if (on && c < f.per) {
        z[k] = load<V>(x + at + c);
        d[k] = load<V>(dy + at + c);
        if (GATED) w[k] = load<V>(gate + at + c);
      }
    }
    float as[V], bs[V], means[V], scales[V];
    fill<V>(as, 0.f);
    fill<V>(bs, 0.f);
    fill<V>(means, mu);
    fill<V>(scales, is);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      sub_all<V>(z[k].v, z[k].v, means);
      mul_all<V>(z[k].v, z[k].v, scales);
      inner_gradient<V, GATED>(f.code, d[k].v, z[k].v, ga[k].v, be[k].v, w[GATED ? k : 0].v);
      add_all<V>(sum_n[k].v, sum_n[k].v, d[k].v);
      fma_all<V>(sum_z[k].v, d[k].v, z[k].v, sum_z[k].v);
      mul_all<V>(d[k].v, d[k].v, ga[k].v);
      add_all<V>(as, as, d[k].v);
      fma_all<V>(bs, d[k].v, z[k].v, bs);
    }
    fill<V>(as, over_lanes(total<V>(as), f.lanes) * share);
    fill<V>(bs, -over_lanes(total<V>(bs), f.lanes) * share);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * f.lanes + lane) * V;
      if (!on || c >= f.per) continue;
      sub_all<V>(d[k].v, d[k].v, as);
      fma_all<V>(d[k].v, z[k].v, bs, d[k].v);
      mul_all<V>(d[k].v, d[k].v, scales);
      store<V>(dx + at + c, d[k]);
      if (GATED) store<V>(dgate + at + c, w[k]);
    }
  }
  if (!here) return;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * f.lanes + lane) * V;
    if (c >= f.per) continue;
    float* out = part + (int64_t)row * 2 * f.C + g * f.per + c;
    store<V>(out, sum_n[k]);
    store<V>(out + f.C, sum_z[k]);
  }
}

// ------------------------------------------------------------------ maps in registers
//
// A block has `wide` channels (whole groups) of all positions of a sample in its
// registers, K pieces of V channels a thread: `across` pieces of a position by `rows`
// positions at a time.  Sums go over the threads through shared memory in a fixed order.

struct Slab {
  int64_t N;
  int S, C, G, per, wide, spans, across, rows, split, code;
  int step_j, step_c;       // 32 / per and 32 % per
  bool folded;
  float eps;
};

// Partial sums over a block's positions of M numbers per channel, from every thread's v (M,
// V) of channels q V ..: (M, split, wide) numbers, at the address that is returned.  Threads
// of a warp with the same channels add theirs first where there is a power of two of them
// (f.folded); up to 16 rows are left as they are, more are added to f.split.
template <int M, int V>
__device__ __forceinline__ const float* channel_sums(float* scratch, float (&v)[M][V], int q,
                                                     int row, bool on, const Slab& f) {
  int rows = f.rows;
  if (f.folded) {
    for (int o = 16; o >= f.across; o >>= 1)
#pragma unroll
      for (int i = 0; i < M; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] += __shfl_xor_sync(0xffffffffu, v[i][e], o);
    rows = blockDim.x >> 5;
    row = threadIdx.x >> 5;
    on = (threadIdx.x & 31) < f.across;
  }
  __syncthreads();                                   // whoever read the last sums is done
  if (on)
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) scratch[(i * rows + row) * f.wide + q * V + e] = v[i][e];
  __syncthreads();
  if (rows == f.split) return scratch;
  float* out = scratch + M * rows * f.wide;
  for (int t = threadIdx.x; t < M * f.split * f.wide; t += blockDim.x) {
    const int c = t % f.wide, j = t / f.wide % f.split, i = t / f.wide / f.split;
    float sum = 0.f;
    for (int r = j; r < rows; r += f.split) sum += scratch[(i * rows + r) * f.wide + c];
    out[t] = sum;
  }
  __syncthreads();
  return out;
}

// The places of a lane's partial sums of the first group: every 32nd of split * per.
template <class F>
__device__ __forceinline__ void each_of_group(const Slab& f, int lane, F take) {
  int j = lane / f.per, c = lane - j * f.per;
#pragma unroll 4
  for (int i = lane; i < f.split * f.per; i += 32) {
    take(j * f.wide + c, c);
    j += f.step_j;
    c += f.step_c;
    const bool on = c >= f.per;
    j += on;
    c -= on ? f.per : 0;
  }
}

// The groups of channels c to c + V - 1.
template <int V>
__device__ __forceinline__ void groups_of(int (&of)[V], int c, int per) {
  of[0] = c / per;
  c -= of[0] * per;
#pragma unroll
  for (int e = 1; e < V; ++e) {
    c = c + 1 == per ? 0 : c + 1;
    of[e] = of[e - 1] + (c == 0);
  }
}

// (64 registers a thread, four blocks of 256 on an SM: over 16 x 4096 x 64 19.9 -> 16.4 us, 64 x
// 1024 x 128 gated 35.7 -> 30.5; over 128 x 1024 x 64, whose pieces of a position are 32 bytes,
// 21.6 -> 22.1, where 3 TB/s go through it: phases of reading, two sums and writing that four
// blocks hide from one another only in part.)
template <int V, int K, bool GATED>
__global__ void __launch_bounds__(512, 2)
    slab_kernel(float* __restrict__ y, float* __restrict__ mean, float* __restrict__ inv,
                const float* __restrict__ x, const float* __restrict__ gate,
                const float* __restrict__ gamma, const float* __restrict__ beta, const Slab f) {
  extern __shared__ float smem[];
  float* group = smem;                               // (wide / per) twice
  float* scratch = smem + 2 * f.wide;
  const int64_t n = blockIdx.x / f.spans;
  const int c0 = blockIdx.x % f.spans * f.wide, wide = min(f.wide, f.C - c0), groups = wide / f.per;
  const int q = threadIdx.x % f.across, row = threadIdx.x / f.across;
  const bool on = row < f.rows, in = on && q * V < wide;
  const int64_t at = n * f.S * f.C + c0 + q * V;
  Pack<V> v[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int p = row + k * f.rows;
#pragma unroll
    for (int e = 0; e < V; ++e) v[k].v[e] = 0.f;
    if (in && p < f.S) v[k] = load<V>(x + at + (int64_t)p * f.C);
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float count = (float)f.S * (float)f.per;
  auto over_groups = [&](const float* sums, float* to, auto finish) {
    for (int g = warp; g < groups; g += blockDim.x >> 5) {
      float sum = 0.f;
      each_of_group(f, lane, [&](int i, int) { sum += sums[i + g * f.per]; });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) to[g] = finish(sum / count, g);
    }
    __syncthreads();
  };
  int of[V];
  groups_of<V>(of, in ? q * V : 0, f.per);
  float part[1][V] = {}, downs[V];
  fill<V>(downs, kDown);
#pragma unroll
  for (int k = 0; k < K; ++k) fma_all<V>(part[0], v[k].v, downs, part[0]);
  const float* sums = channel_sums<1, V>(scratch, part, q, row, on, f);
  over_groups(sums, group, [](float m, int) { return m * kUp; });
  float mu[V], is[V];
#pragma unroll
  for (int e = 0; e < V; ++e) mu[e] = group[of[e]], part[0][e] = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    sub_all<V>(v[k].v, v[k].v, mu);
    if (row + k * f.rows < f.S) fma_all<V>(part[0], v[k].v, v[k].v, part[0]);
  }
  if (!in)
#pragma unroll
    for (int e = 0; e < V; ++e) part[0][e] = 0.f;
  sums = channel_sums<1, V>(scratch, part, q, row, on, f);
  over_groups(sums, group + groups, [&](float m, int g) {
    if (m < INFINITY) return inverse_root(m + f.eps);
    const float* own = x + n * f.S * f.C + c0 + g * f.per;
    float far = 0.f;
    for (int p = 0; p < f.S; ++p)
      for (int c = 0; c < f.per; ++c) {
        const float d = (own[(int64_t)p * f.C + c] - group[g]) * kFar;
        far = fmaf(d, d, far);
      }
    return far_inverse(far / count, f.eps);
  });
  for (int g = threadIdx.x; g < groups; g += blockDim.x) {
    mean[n * f.G + c0 / f.per + g] = group[g];
    inv[n * f.G + c0 / f.per + g] = group[groups + g];
  }
  if (!in) return;
  float ga[V], be[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    is[e] = group[groups + of[e]];
    ga[e] = (gamma ? gamma[c0 + q * V + e] : 1.f);
    be[e] = beta ? beta[c0 + q * V + e] : 0.f;
  }
  // (single channels two positions at a time, for the pairs)
  constexpr int J = V == 1 && K > 1 ? 2 : 1;
#pragma unroll
  for (int k = 0; k < K; k += J) {
    if (row + k * f.rows >= f.S) continue;
    float now[J * V], w[J * V];
    fill<J * V>(w, 0.f);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int p = row + (k + j) * f.rows;
      mul_all<V>(v[k + j].v, v[k + j].v, is);
      fma_all<V>(v[k + j].v, v[k + j].v, ga, be);
      Pack<V> gates;
      fill<V>(gates.v, 0.f);
      if (GATED && p < f.S) gates = load<V>(gate + at + (int64_t)p * f.C);
#pragma unroll
      for (int e = 0; e < V; ++e) now[j * V + e] = v[k + j].v[e], w[j * V + e] = gates.v[e];
    }
    if constexpr (GATED) {
      act_all<J * V>(f.code, w);
      mul_all<J * V>(now, now, w);
    } else {
      act_all<J * V>(f.code, now);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int p = row + (k + j) * f.rows;
#pragma unroll
      for (int e = 0; e < V; ++e) v[k + j].v[e] = now[j * V + e];
      if (p < f.S) store<V>(y + at + (int64_t)p * f.C, v[k + j]);
    }
  }
}

template <int V, int K, bool GATED>
__global__ void __launch_bounds__(512)
    slab_backward_kernel(float* __restrict__ dx, float* __restrict__ dgate,
                         float* __restrict__ part, const float* __restrict__ dy,
                         const float* __restrict__ x, const float* __restrict__ gate,
                         const float* __restrict__ mean, const float* __restrict__ inv,
                         const float* __restrict__ gamma, const float* __restrict__ beta,
                         const Slab f) {
  extern __shared__ float smem[];
  float2* group = reinterpret_cast<float2*>(smem);   // (wide / per)
  float* scratch = smem + 2 * f.wide;
  const int64_t n = blockIdx.x / f.spans;
  const int c0 = blockIdx.x % f.spans * f.wide, wide = min(f.wide, f.C - c0), groups = wide / f.per;
  const int q = threadIdx.x % f.across, row = threadIdx.x / f.across;
  const bool on = row < f.rows, in = on && q * V < wide;
  const int64_t at = n * f.S * f.C + c0 + q * V;
  Pack<V> z[K], d[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int p = row + k * f.rows;
#pragma unroll
    for (int e = 0; e < V; ++e) z[k].v[e] = d[k].v[e] = 0.f;
    if (in && p < f.S) {
      z[k] = load<V>(x + at + (int64_t)p * f.C);
      d[k] = load<V>(dy + at + (int64_t)p * f.C);
    }
  }
  float mu[V], is[V], ga[V], be[V];
  int of[V];
  groups_of<V>(of, in ? q * V : 0, f.per);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    mu[e] = in ? mean[n * f.G + c0 / f.per + of[e]] : 0.f;
    is[e] = in ? inv[n * f.G + c0 / f.per + of[e]] : 0.f;
    ga[e] = in && gamma ? gamma[c0 + q * V + e] : 1.f;
    be[e] = in && beta ? beta[c0 + q * V + e] : 0.f;
  }
  float both[2][V] = {};
  // (single channels two positions at a time, for the pairs)
  constexpr int J = V == 1 && K > 1 ? 2 : 1;
  float gammas[J * V], betas[J * V];
#pragma unroll
  for (int e = 0; e < J * V; ++e) gammas[e] = ga[e % V], betas[e] = be[e % V];
#pragma unroll
  for (int k = 0; k < K; k += J) {
    if (!in || row + k * f.rows >= f.S) continue;
    float zs[J * V], ds[J * V], ws[J * V];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int p = row + (k + j) * f.rows;
      sub_all<V>(z[k + j].v, z[k + j].v, mu);
      mul_all<V>(z[k + j].v, z[k + j].v, is);
      Pack<V> gates;
      fill<V>(gates.v, 0.f);
      if (GATED && p < f.S) gates = load<V>(gate + at + (int64_t)p * f.C);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        zs[j * V + e] = z[k + j].v[e];
        ds[j * V + e] = d[k + j].v[e];
        ws[j * V + e] = gates.v[e];
      }
    }
    inner_gradient<J * V, GATED>(f.code, ds, zs, gammas, betas, ws);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int p = row + (k + j) * f.rows;
      Pack<V> gates;
#pragma unroll
      for (int e = 0; e < V; ++e) d[k + j].v[e] = ds[j * V + e], gates.v[e] = ws[j * V + e];
      if (j > 0 && p >= f.S) continue;
      add_all<V>(both[0], both[0], d[k + j].v);
      fma_all<V>(both[1], d[k + j].v, z[k + j].v, both[1]);
      if (GATED) store<V>(dgate + at + (int64_t)p * f.C, gates);
    }
  }
  const float* sums = channel_sums<2, V>(scratch, both, q, row, on, f);
  // dbeta's and dgamma's share of this sample
  for (int c = threadIdx.x; c < wide; c += blockDim.x) {
    float a = 0.f, b = 0.f;
    for (int j = 0; j < f.split; ++j) {
      a += sums[j * f.wide + c];
      b += sums[(f.split + j) * f.wide + c];
    }
    part[n * 2 * f.C + c0 + c] = a;
    part[n * 2 * f.C + f.C + c0 + c] = b;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float count = (float)f.S * (float)f.per;
  for (int g = warp; g < groups; g += blockDim.x >> 5) {
    float a = 0.f, b = 0.f;
    each_of_group(f, lane, [&](int i, int c) {
      const float w = gamma ? gamma[c0 + g * f.per + c] : 1.f;
      a = fmaf(w, sums[i + g * f.per], a);
      b = fmaf(w, sums[f.split * f.wide + i + g * f.per], b);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (lane == 0) group[g] = make_float2(a / count, b / count);
  }
  __syncthreads();
  if (!in) return;
  // is (ga d - mean of u - z mean of u z)
  float a[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float2 m = group[of[e]];
    a[e] = -is[e] * m.x;
    b[e] = -is[e] * m.y;
    ga[e] *= is[e];
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int p = row + k * f.rows;
    if (p >= f.S) continue;
    fma_all<V>(d[k].v, d[k].v, ga, a);
    fma_all<V>(d[k].v, z[k].v, b, d[k].v);
    store<V>(dx + at + (int64_t)p * f.C, d[k]);
  }
}

int plan(const char* what, Shape& s, int64_t N, int64_t S, int64_t C, int64_t G, int activation,
         float eps) {
  WXX_REQUIRE(N >= 0 && S >= 0 && C >= 0, "%s: negative size", what);
  WXX_REQUIRE(G > 0 && C % G == 0, "%s: %lld channels cannot be split over %lld groups", what,
              (long long)C, (long long)G);
  WXX_REQUIRE(activation >= kNone && activation <= kGelu, "%s: unknown activation %d", what,
              activation);
  WXX_REQUIRE(eps > 0.f, "%s: eps must be positive", what);
  WXX_REQUIRE(C < (int64_t(1) << 24) && N < (int64_t(1) << 31) && S < (int64_t(1) << 31),
              "%s: too many channels, samples or positions", what);
  s = Shape{N, S, (int)C, (int)G, (int)(C / G), 1, S, eps};
  if (N == 0 || S == 0) return WXX_OK;
  // pieces of a sample where there are fewer samples than blocks to fill the GPU
  int64_t chunks = (4 * (int64_t)wxx::num_sms() + N - 1) / N;
  const int64_t most = (S * C + 4095) / 4096;
  if (chunks > most) chunks = most;
  if (chunks > S) chunks = S;
  if (chunks < 1) chunks = 1;
  s.piece = (S + chunks - 1) / chunks;
  s.chunks = (int)((S + s.piece - 1) / s.piece);
  WXX_REQUIRE(N * s.chunks < (int64_t(1) << 31), "%s: too many samples", what);
  return WXX_OK;
}

// Whether rows of `per` channels and all the given memory can be taken 4 channels at a time.
bool fours(const void* const (&memory)[8], int64_t per) {
  uintptr_t all = 0;
  for (const void* p : memory) all |= reinterpret_cast<uintptr_t>(p);
  return (all & 15) == 0 && per % 4 == 0;
}

// A group of one position in the registers of up to 32 threads, if it fits.
bool plan_few(Few& f, int& v, int& k, const Shape& s, int code, bool four, bool two) {
  if (s.S != 1 || s.N * s.G >= (int64_t(1) << 31)) return false;
  v = four ? 4 : 1;
  const int pieces = (s.per + v - 1) / v;
  int lanes = 1;
  // `two` pieces of 4 a thread where they still are whole 128 bytes.  (Over 8192 x 1024 gated:
  // forward 21.6 -> 19.0 us; backward, which then has too many registers, 36.1 -> 39.8.)
  while (lanes < 32 && lanes < pieces && (lanes < 8 || v == 1 || !two || 2 * lanes < pieces))
    lanes <<= 1;
  k = 1;
  while (k * lanes < pieces) k <<= 1;
  if (k > 8) return false;
  f = Few{s.N, s.C, s.G, s.per, lanes, 0, code, s.eps};
  return true;
}

// Samples under way at once: two a thread (forward, least = 1), or (backward, where each costs
// a partial sum of every channel) threads enough for the SMs, and `least` samples a thread
// where there are so many.
unsigned few_grid(Few& f, int least) {
  const int64_t row = (int64_t)f.G * f.lanes, most = (f.N + least - 1) / least;
  int64_t rows = least == 1 ? (f.N + 1) / 2 : ((int64_t)wxx::num_sms() * 1024 + row - 1) / row;
  if (rows > most) rows = most;
  const int64_t counted = ((int64_t(1) << 31) - kT) / row;     // threads are counted in 32 bits
  if (rows > counted) rows = counted;
  f.rows = (int)rows;
  return (unsigned)((rows * row + kT - 1) / kT);
}

// Whole groups of a sample's positions in a block's registers, K pieces a thread at most, if they
// fit: as wide as that allows (long pieces of a position), 256 threads, or 512 where one
// group needs them.
bool plan_slab(Slab& f, int& v, int& k, int& threads, const Shape& s, int code, bool four, int most,
               int sums) {
  if (s.S == 1 || s.S > (1 << 20)) return false;
  v = four ? 4 : 1;
  int unit = s.per;                                  // channels of whole groups and pieces
  while (unit % v) unit += s.per;
  for (threads = 256; threads <= 512; threads *= 2) {
    int wide = 0;
    for (int w = unit; w <= s.C + unit - 1 && w / v <= threads; w += unit) {
      const int rows = threads / (w / v);
      const int64_t bytes = (int64_t)(sums * (rows + 16) + 2) * w * 4;
      if ((s.S + rows - 1) / rows > most || bytes > 48 * 1024) break;
      wide = w;
      // blocks enough for the SMs before pieces of more than 64 bytes
      if (w * 4 >= 64 && s.N * ((s.C + w - 1) / w) < 2 * wxx::num_sms()) break;
    }
    if (wide == 0) continue;
    const int across = wide / v;
    int rows = threads / across;
    if (rows > s.S) rows = (int)s.S;
    k = (int)((s.S + rows - 1) / rows);
    const bool folded = across <= 16 && (across & (across - 1)) == 0;
    int split = folded ? threads / 32 : rows;
    if (split > 16) {
      split = threads / wide;
      if (split > 16) split = 16;
      if (split < 1) split = 1;
    }
    f = Slab{s.N,    (int)s.S, s.C,  s.G,   s.per, wide,  (s.C + wide - 1) / wide,
             across, rows,     split, code, 32 / s.per, 32 % s.per, folded, s.eps};
    return s.N * f.spans < (int64_t(1) << 31);
  }
  return false;
}

// Shared memory of a block: the groups' results, the threads' sums and partial sums of them.
size_t slab_bytes(const Slab& f, int threads, int sums) {
  const size_t rows = f.folded ? threads / 32 : f.rows;
  return (2 + sums * (rows + f.split)) * f.wide * sizeof(float);
}

template <int K>
using Pieces = std::integral_constant<int, K>;
template <class F>
void with_pieces(int v, int k, F f) {
  auto with_k = [&](auto vv) {
    if (k <= 1) return f(vv, Pieces<1>{});
    if (k <= 2) return f(vv, Pieces<2>{});
    if (k <= 4) return f(vv, Pieces<4>{});
    return f(vv, Pieces<8>{});
  };
  if (v == 4)
    with_k(Pieces<4>{});
  else
    with_k(Pieces<1>{});
}

}  // namespace

// y, mean and inv (N, G) from x (N, S, C); gamma, beta (C) and gate (like x) may be NULL.
// activation: 0 none, 1 ReLU, 2 SiLU, 3 GELU (tanh form), of the result, or with a gate of
// the gate, which multiplies the result.
WXX_EXPORT int wxx_group_norm(float* y, float* mean, float* inv, const float* x,
                              const float* gate, const float* gamma, const float* beta, int64_t N,
                              int64_t S, int64_t C, int64_t G, int activation, float eps) {
  WXX_REQUIRE_INIT();
  Shape s;
  if (int st = plan("wxx_group_norm", s, N, S, C, G, activation, eps)) return st;
  if (N * S * C == 0) {                    // the statistics of nothing
    if (N > 0) {
      WXX_CUDA_CHECK(cudaMemsetAsync(mean, 0, (size_t)(N * G) * sizeof(float), wxx::stream()));
      WXX_CUDA_CHECK(cudaMemsetAsync(inv, 0, (size_t)(N * G) * sizeof(float), wxx::stream()));
    }
    return WXX_OK;
  }
  const bool four = fours({y, x, gate, gamma, beta, nullptr, nullptr, nullptr}, C);
  Few few;
  Slab slab;
  int v, k, threads;
  if (plan_few(few, v, k, s, activation, four && s.per % 4 == 0, true)) {
    const unsigned grid = few_grid(few, 1);
    with_pieces(v, k, [&](auto vv, auto kk) {
      constexpr int V = decltype(vv)::value, K = decltype(kk)::value;
      auto kernel = gate ? token_kernel<V, K, true> : token_kernel<V, K, false>;
      kernel<<<grid, kT, 0, wxx::stream()>>>(y, mean, inv, x, gate, gamma, beta, few);
    });
    WXX_LAUNCH_CHECK();
    return WXX_OK;
  }
  if (plan_slab(slab, v, k, threads, s, activation, four, 8, 1)) {
    const size_t bytes = slab_bytes(slab, threads, 1);
    with_pieces(v, k, [&](auto vv, auto kk) {
      constexpr int V = decltype(vv)::value, K = decltype(kk)::value;
      auto kernel = gate ? slab_kernel<V, K, true> : slab_kernel<V, K, false>;
      kernel<<<(unsigned)(N * slab.spans), threads, bytes, wxx::stream()>>>(y, mean, inv, x, gate, gamma,
                                                                           beta, slab);
    });
    WXX_LAUNCH_CHECK();
    return WXX_OK;
  }
  void* part = nullptr;
  if (int st = wxx_malloc(&part, (uint64_t)(N * s.chunks * G) * sizeof(Moments))) return st;
  Moments* m = static_cast<Moments*>(part);
  moments_kernel<<<(unsigned)(N * s.chunks), kT, 0, wxx::stream()>>>(m, x, s);
  int st = wxx::after_launch(__FILE__, __LINE__);
  if (st == WXX_OK) {
    statistics_kernel<<<(unsigned)((N * G + kT - 1) / kT), kT, 0, wxx::stream()>>>(mean, inv, m, x, s);
    st = wxx::after_launch(__FILE__, __LINE__);
  }
  wxx_free(part);
  if (st != WXX_OK) return st;
  auto apply = gate ? apply_kernel<true> : apply_kernel<false>;
  apply<<<wxx::grid_for(N * S * C, kT), kT, 0, wxx::stream()>>>(y, x, gate, mean, inv, gamma, beta, s,
                                                               activation);
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}

// dx, dgate (NULL without a gate), dgamma and dbeta (C) from dy, the forward's inputs and
// its mean and inv.
WXX_EXPORT int wxx_group_norm_backward(float* dx, float* dgamma, float* dbeta, float* dgate,
                                       const float* dy, const float* x, const float* gate,
                                       const float* gamma, const float* beta, const float* mean,
                                       const float* inv, int64_t N, int64_t S, int64_t C,
                                       int64_t G, int activation) {
  WXX_REQUIRE_INIT();
  Shape s;
  if (int st = plan("wxx_group_norm_backward", s, N, S, C, G, activation, 1.f)) return st;
  if (N * S * C == 0) {                    // the sums over nothing
    if (C > 0) {
      WXX_CUDA_CHECK(cudaMemsetAsync(dgamma, 0, (size_t)C * sizeof(float), wxx::stream()));
      WXX_CUDA_CHECK(cudaMemsetAsync(dbeta, 0, (size_t)C * sizeof(float), wxx::stream()));
    }
    return WXX_OK;
  }
  const bool four = fours({dx, dgate, dy, x, gate, gamma, beta, nullptr}, C);
  Few few;
  Slab slab;
  int v, k, threads;
  const bool tokens = plan_few(few, v, k, s, activation, four && s.per % 4 == 0, false);
  if (tokens || plan_slab(slab, v, k, threads, s, activation, four, 8, 2)) {
    const unsigned grid = tokens ? few_grid(few, 2) : 0;
    const int64_t rows = tokens ? few.rows : N;
    void* scratch = nullptr;
    if (int st = wxx_malloc(&scratch, (uint64_t)(rows * 2 * C) * sizeof(float))) return st;
    float* part = static_cast<float*>(scratch);
    with_pieces(v, k, [&](auto vv, auto kk) {
      constexpr int V = decltype(vv)::value, K = decltype(kk)::value;
      if (tokens) {
        auto kernel = gate ? token_backward_kernel<V, K, true> : token_backward_kernel<V, K, false>;
        kernel<<<grid, kT, 0, wxx::stream()>>>(dx, dgate, part, dy, x, gate, mean, inv, gamma, beta, few);
      } else {
        const size_t bytes = slab_bytes(slab, threads, 2);
        auto kernel = gate ? slab_backward_kernel<V, K, true> : slab_backward_kernel<V, K, false>;
        kernel<<<(unsigned)(N * slab.spans), threads, bytes, wxx::stream()>>>(
            dx, dgate, part, dy, x, gate, mean, inv, gamma, beta, slab);
      }
    });
    int st = wxx::after_launch(__FILE__, __LINE__);
    if (st == WXX_OK) {
      column_sums_kernel<<<(unsigned)((2 * C + 15) / 16), 1024, 0, wxx::stream()>>>(dbeta, dgamma, part,
                                                                                 rows, (int)C);
      st = wxx::after_launch(__FILE__, __LINE__);
    }
    wxx_free(scratch);
    return st;
  }
  const int64_t rows = N * s.chunks;
  void* scratch = nullptr;
  if (int st = wxx_malloc(&scratch, (uint64_t)(rows * 2 * C) * sizeof(float) +
                                        (uint64_t)(N * G) * sizeof(float2)))
    return st;
  float2* sums = static_cast<float2*>(scratch);
  float* part = reinterpret_cast<float*>(sums + N * G);
  auto sum = gate ? channel_sums_kernel<true> : channel_sums_kernel<false>;
  sum<<<(unsigned)rows, kT, 0, wxx::stream()>>>(part, dy, x, gate, mean, inv, gamma, beta, s, activation);
  int st = wxx::after_launch(__FILE__, __LINE__);
  if (st == WXX_OK) {
    group_sums_kernel<<<(unsigned)((N * G + kT - 1) / kT), kT, 0, wxx::stream()>>>(sums, part,
                                                                                  gamma, s);
    st = wxx::after_launch(__FILE__, __LINE__);
  }
  if (st == WXX_OK) {
    auto input = gate ? input_gradient_kernel<true> : input_gradient_kernel<false>;
    input<<<wxx::grid_for(N * S * C, kT), kT, 0, wxx::stream()>>>(dx, dgate, dy, x, gate, mean, inv,
                                                                 gamma, beta, sums, s, activation);
    st = wxx::after_launch(__FILE__, __LINE__);
  }
  if (st == WXX_OK) {
    column_sums_kernel<<<(unsigned)((2 * C + 15) / 16), 1024, 0, wxx::stream()>>>(dbeta, dgamma, part,
                                                                               rows, (int)C);
    st = wxx::after_launch(__FILE__, __LINE__);
  }
  wxx_free(scratch);
  return st;
}
