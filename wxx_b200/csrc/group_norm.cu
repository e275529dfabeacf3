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

#include "common.cuh"

WXX_EXPORT int wxx_malloc(void** out, uint64_t nbytes);
WXX_EXPORT int wxx_free(void* p);

namespace {

constexpr int kT = 256;

enum Act { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

// 1 / (1 + exp(-v)), good to a few ulp: exp is the library's, and infinite where the
// quotient is 0.
__device__ __forceinline__ float logistic(float v) { return 1.0f / (1.0f + expf(-v)); }

// GELU is the tanh form with the clamps of gelu_tanh, as x s(2 u).
__device__ __forceinline__ float gelu_argument(float v) {
  return 2.0f * 0.7978845608f * (v + 0.044715f * v * v * v);
}

template <int ACT>
__device__ __forceinline__ float act(float v) {
  if (ACT == kRelu) return v < 0.f ? 0.f : v;
  if (ACT == kSilu) return v * logistic(v);
  if (ACT == kGelu) {
    const float r = v * logistic(gelu_argument(v));
    return v > 10.f ? v : v < -10.f ? 0.f : r;
  }
  return v;
}

template <int ACT>
__device__ __forceinline__ float slope(float v) {
  if (ACT == kRelu) return v > 0.f ? 1.f : 0.f;
  if (ACT == kSilu) {
    const float p = logistic(v);
    return p * (1.0f + v * (1.0f - p));
  }
  if (ACT == kGelu) {
    const float p = logistic(gelu_argument(v));
    const float r = p + v * p * (1.0f - p) * (2.0f * 0.7978845608f) * (1.0f + 0.134145f * v * v);
    return v > 10.f ? 1.f : v < -10.f ? 0.f : r;
  }
  return 1.f;
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

// The moments of each group over a piece of a sample: part (N, chunks, G).
__global__ void __launch_bounds__(kT)
    moments_kernel(Moments* __restrict__ part, const float* __restrict__ x, const Shape s) {
  __shared__ Moments sums[kT];
  const int64_t n = blockIdx.x / s.chunks;
  const int64_t p0 = (blockIdx.x % s.chunks) * s.piece;
  const int64_t p1 = p0 + s.piece < s.S ? p0 + s.piece : s.S;
  const float* xn = x + n * s.S * s.C;
  const Lanes l(s.C);
  Moments group = {0.f, 0.f, 0.f};     // of group threadIdx.x, in parts of kT groups
  for (int g0 = 0; g0 < s.G; g0 += kT) {
    group = {0.f, 0.f, 0.f};
    const int gs = g0 + kT < s.G ? g0 + kT : s.G;
    for (int c0 = g0 * s.per; c0 < gs * s.per; c0 += l.wide) {
      const int c = c0 + l.c;
      Moments m = {0.f, 0.f, 0.f};
      if (l.row < l.rows && c < gs * s.per) {
        for (int64_t p = p0 + l.row; p < p1; p += l.rows) {
          const float v = xn[p * s.C + c];
          m.n += 1.f;
          const float d = v - m.mean;
          m.mean += d / m.n;
          m.m2 += d * (v - m.mean);
        }
      }
      sums[threadIdx.x] = m;
      __syncthreads();
      // the group's thread joins its channels among these, in their order
      const int g = g0 + threadIdx.x;
      if (g < gs) {
        const int from = max(g * s.per, c0), to = min((g + 1) * s.per, c0 + l.wide);
        for (int k = from; k < to; ++k)
          for (int r = 0; r < l.rows; ++r) group = join(group, sums[r * l.wide + k - c0]);
      }
      __syncthreads();
    }
    if (g0 + threadIdx.x < gs) part[(int64_t)blockIdx.x * s.G + g0 + threadIdx.x] = group;
  }
}

// mean and inv (N, G) from the pieces' moments.
__global__ void __launch_bounds__(kT)
    statistics_kernel(float* __restrict__ mean, float* __restrict__ inv,
                      const Moments* __restrict__ part, const Shape s) {
  const int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x;
  if (i >= s.N * s.G) return;
  const int64_t n = i / s.G;
  const int g = (int)(i - n * s.G);
  Moments m = {0.f, 0.f, 0.f};
  for (int k = 0; k < s.chunks; ++k) m = join(m, part[(n * s.chunks + k) * s.G + g]);
  mean[i] = m.mean;
  inv[i] = 1.0f / sqrtf(m.m2 / ((float)s.S * (float)s.per) + s.eps);
}

template <int ACT, bool GATED>
__global__ void __launch_bounds__(kT)
    apply_kernel(float* __restrict__ y, const float* __restrict__ x,
                 const float* __restrict__ gate, const float* __restrict__ mean,
                 const float* __restrict__ inv, const float* __restrict__ gamma,
                 const float* __restrict__ beta, const Shape s) {
  const int64_t sample = s.S * s.C, total = s.N * sample;
  for (int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * kT) {
    const int64_t n = i / sample;
    const int c = (int)((i - n * sample) % s.C);
    const int64_t g = n * s.G + c / s.per;
    const float z = (x[i] - mean[g]) * inv[g];
    const float v = fmaf(z, gamma ? gamma[c] : 1.f, beta ? beta[c] : 0.f);
    y[i] = GATED ? v * act<ACT>(gate[i]) : act<ACT>(v);
  }
}

// The gradient of n at one place, and where GATED that of the gate.
template <int ACT, bool GATED>
__device__ __forceinline__ float inner_gradient(float dy, float z, float gamma, float beta,
                                                float gate, float* dgate) {
  const float v = fmaf(z, gamma, beta);
  if (!GATED) return dy * slope<ACT>(v);
  *dgate = dy * v * slope<ACT>(gate);
  return dy * act<ACT>(gate);
}

// For every channel the sums of dn and dn z over a piece of a sample: part (N, chunks,
// 2, C).
template <int ACT, bool GATED>
__global__ void __launch_bounds__(kT)
    channel_sums_kernel(float* __restrict__ part, const float* __restrict__ dy,
                        const float* __restrict__ x, const float* __restrict__ gate,
                        const float* __restrict__ mean, const float* __restrict__ inv,
                        const float* __restrict__ gamma, const float* __restrict__ beta,
                        const Shape s) {
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
      const float ga = gamma ? gamma[c] : 1.f, be = beta ? beta[c] : 0.f;
      for (int64_t p = p0 + l.row; p < p1; p += l.rows) {
        const int64_t i = at + p * s.C + c;
        const float z = (x[i] - mu) * is;
        float unused;
        const float dn = inner_gradient<ACT, GATED>(dy[i], z, ga, be, GATED ? gate[i] : 0.f,
                                                    &unused);
        a += dn;
        b = fmaf(dn, z, b);
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

template <int ACT, bool GATED>
__global__ void __launch_bounds__(kT)
    input_gradient_kernel(float* __restrict__ dx, float* __restrict__ dgate,
                          const float* __restrict__ dy, const float* __restrict__ x,
                          const float* __restrict__ gate, const float* __restrict__ mean,
                          const float* __restrict__ inv, const float* __restrict__ gamma,
                          const float* __restrict__ beta, const float2* __restrict__ sums,
                          const Shape s) {
  const int64_t sample = s.S * s.C, total = s.N * sample;
  for (int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * kT) {
    const int64_t n = i / sample;
    const int c = (int)((i - n * sample) % s.C);
    const int64_t g = n * s.G + c / s.per;
    const float is = inv[g], z = (x[i] - mean[g]) * is;
    const float ga = gamma ? gamma[c] : 1.f;
    float dg;
    const float dn = inner_gradient<ACT, GATED>(dy[i], z, ga, beta ? beta[c] : 0.f,
                                                GATED ? gate[i] : 0.f, &dg);
    const float2 m = sums[g];
    dx[i] = is * (ga * dn - m.x - z * m.y);
    if (GATED) dgate[i] = dg;
  }
}

// out (2, C) from rows of 2 C partial sums, in a fixed order: 32 columns by 8 parts of
// the rows a block.  first: dbeta, then dgamma.
__global__ void __launch_bounds__(kT)
    column_sums_kernel(float* __restrict__ dbeta, float* __restrict__ dgamma,
                       const float* __restrict__ part, int64_t rows, int C) {
  __shared__ float sums[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float a = 0.f;
  if (c < 2 * C)
    for (int64_t r = warp; r < rows; r += 8) a += part[r * 2 * C + c];
  sums[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && c < 2 * C) {
    for (int w = 1; w < 8; ++w) a += sums[w][lane];
    (c < C ? dbeta[c] : dgamma[c - C]) = a;
  }
}

// Calls f with the activation and whether there is a gate as constants.
template <int V>
struct Const {
  static constexpr int value = V;
};
template <class F>
void with_form(int activation, bool gated, F f) {
  auto with_act = [&](auto g) {
    switch (activation) {
      case kRelu: return f(Const<kRelu>{}, g);
      case kSilu: return f(Const<kSilu>{}, g);
      case kGelu: return f(Const<kGelu>{}, g);
      default: return f(Const<kNone>{}, g);
    }
  };
  if (gated)
    with_act(Const<1>{});
  else
    with_act(Const<0>{});
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
  void* part = nullptr;
  if (int st = wxx_malloc(&part, (uint64_t)(N * s.chunks * G) * sizeof(Moments))) return st;
  Moments* m = static_cast<Moments*>(part);
  moments_kernel<<<(unsigned)(N * s.chunks), kT, 0, wxx::stream()>>>(m, x, s);
  int st = wxx::after_launch(__FILE__, __LINE__);
  if (st == WXX_OK) {
    statistics_kernel<<<(unsigned)((N * G + kT - 1) / kT), kT, 0, wxx::stream()>>>(mean, inv, m, s);
    st = wxx::after_launch(__FILE__, __LINE__);
  }
  wxx_free(part);
  if (st != WXX_OK) return st;
  with_form(activation, gate != nullptr, [&](auto a, auto g) {
    apply_kernel<decltype(a)::value, decltype(g)::value>
        <<<wxx::grid_for(N * S * C, kT), kT, 0, wxx::stream()>>>(y, x, gate, mean, inv, gamma, beta,
                                                                 s);
  });
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
  const int64_t rows = N * s.chunks;
  void* scratch = nullptr;
  if (int st = wxx_malloc(&scratch, (uint64_t)(rows * 2 * C) * sizeof(float) +
                                        (uint64_t)(N * G) * sizeof(float2)))
    return st;
  float2* sums = static_cast<float2*>(scratch);
  float* part = reinterpret_cast<float*>(sums + N * G);
  with_form(activation, gate != nullptr, [&](auto a, auto g) {
    channel_sums_kernel<decltype(a)::value, decltype(g)::value>
        <<<(unsigned)rows, kT, 0, wxx::stream()>>>(part, dy, x, gate, mean, inv, gamma, beta, s);
  });
  int st = wxx::after_launch(__FILE__, __LINE__);
  if (st == WXX_OK) {
    group_sums_kernel<<<(unsigned)((N * G + kT - 1) / kT), kT, 0, wxx::stream()>>>(sums, part,
                                                                                  gamma, s);
    st = wxx::after_launch(__FILE__, __LINE__);
  }
  if (st == WXX_OK) {
    with_form(activation, gate != nullptr, [&](auto a, auto g) {
      input_gradient_kernel<decltype(a)::value, decltype(g)::value>
          <<<wxx::grid_for(N * S * C, kT), kT, 0, wxx::stream()>>>(dx, dgate, dy, x, gate, mean,
                                                                   inv, gamma, beta, sums, s);
    });
    st = wxx::after_launch(__FILE__, __LINE__);
  }
  if (st == WXX_OK) {
    column_sums_kernel<<<(unsigned)((2 * C + 31) / 32), kT, 0, wxx::stream()>>>(dbeta, dgamma, part,
                                                                               rows, (int)C);
    st = wxx::after_launch(__FILE__, __LINE__);
  }
  wxx_free(scratch);
  return st;
}
