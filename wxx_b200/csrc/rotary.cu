// Rotary positions: the first r channels of every head are pairs (a, b), turned by
// the position's angle,
//
//   a' = m (a cos t - b sin t),  b' = m (a sin t + b cos t),  t = position f_i
//
// with f_i and the factor m the caller's (frequencies scaled for long contexts come
// with a factor); the other channels are copied.  The gradient is the same map with
// the angle's sign turned.
//
// Memory-bound: x is read and y written once (8 bytes a channel).  A block takes a few
// positions, makes the cosines and sines of theirs once (in 64 bits: at position 10^6
// an angle in 32 bits is off by 0.03) and uses them for every head.

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace {

constexpr int kT = 256;
constexpr int kMostPairs = 256;
constexpr int kSinCos = 4096;        // pairs of a block, at most (32 KB)
constexpr int kElements = 4096;      // channels of a block's positions, about

// n / d for n < 2^31 as a product: d <= 2^s, m = ceil(2^(31 + s) / d) < 2^32.
struct Divider {
  unsigned m, s;
  static Divider of(unsigned d) {
    unsigned s = 0;
    while ((1ull << s) < d) ++s;
    return {(unsigned)(((1ull << (31 + s)) + d - 1) / d), 31 + s};
  }
  __device__ __forceinline__ int operator()(int n) const {
    return (int)(((unsigned long long)(unsigned)n * m) >> s);
  }
};

struct Turns {
  double per[kMostPairs];            // full turns a position, per pair
};

struct Shape {
  int64_t x_bs, x_ts;                // strides of x's batch and time
  const uint32_t* positions;         // (T) or (B, T), NULL: 0, 1, ...
  int64_t p_bs;
  int64_t offset;                    // added to every position
  int T, heads, d, r;
  int at_once;                       // positions of a block
  int tiles;                         // blocks of a sequence
  float gain;                        // m
  float sign;                        // 1, or -1: the gradient
  Divider by_pairs, by_row, by_items;    // pairs of a head, items of a position and a head
};

// cos and sin of `turns` full turns: the quarter taken off in 64 bits, so that the
// rest, at most half a quarter, is exact to 2^-26 of a quarter.
__device__ __forceinline__ float2 cos_sin(double turns) {
  const double part = 4.0 * (turns - rint(turns));
  const double quarter = rint(part);
  float s, c;
  sincospif(0.5f * (float)(part - quarter), &s, &c);
  const int q = (int)quarter & 3;
  const float2 even = q & 2 ? make_float2(-c, -s) : make_float2(c, s);
  return q & 1 ? make_float2(-even.y, even.x) : even;
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
  } else if constexpr (V == 2) {
    const float2 t = *reinterpret_cast<const float2*>(p);
    out.v[0] = t.x, out.v[1] = t.y;
  } else {
    out.v[0] = *p;
  }
  return out;
}
template <int V>
__device__ __forceinline__ void store(float* p, const Pack<V>& a) {
  if constexpr (V == 4)
    *reinterpret_cast<float4*>(p) = make_float4(a.v[0], a.v[1], a.v[2], a.v[3]);
  else if constexpr (V == 2)
    *reinterpret_cast<float2*>(p) = make_float2(a.v[0], a.v[1]);
  else
    *p = a.v[0];
}

__device__ __forceinline__ void turn(float& a, float& b, float2 by) {
  const float x = a, y = b;
  a = fmaf(x, by.x, -y * by.y);
  b = fmaf(x, by.y, y * by.x);
}

// V channels at a time; APART: a pair's channels are r / 2 apart, else neighbours.
// One item is V pairs (APART, or V = 1), V / 2 pairs, or V channels that are copied.
template <int V, bool APART>
__global__ void __launch_bounds__(kT)
    rotary_kernel(float* __restrict__ y, const float* __restrict__ x,
                  const __grid_constant__ Turns turns, const Shape s) {
  __shared__ float2 table[kSinCos];
  const int b = blockIdx.x / s.tiles, t0 = (blockIdx.x % s.tiles) * s.at_once;
  const int n = min(s.at_once, s.T - t0), pairs = s.r / 2;
  for (int e = threadIdx.x; e < n * pairs; e += kT) {
    const int at = s.by_pairs(e), i = e - at * pairs;
    int64_t p = s.offset;
    p += s.positions ? (int64_t)s.positions[b * s.p_bs + t0 + at] : (int64_t)(t0 + at);
    const float2 cs = cos_sin((double)p * turns.per[i]);
    table[e] = make_float2(s.gain * cs.x, s.gain * s.sign * cs.y);
  }
  __syncthreads();
  constexpr int kPairs = APART || V == 1 ? V : V / 2;      // pairs of an item
  const int turned = pairs / kPairs, items = turned + (s.d - s.r) / V;
  const int row = s.heads * items, D = s.heads * s.d;
  const float* xb = x + b * s.x_bs + t0 * s.x_ts;
  float* yb = y + ((int64_t)b * s.T + t0) * D;
  // U items under way together
  constexpr int U = V == 4 ? 2 : 4, kBoth = APART || V == 1 ? 2 : 1;
  for (int e0 = threadIdx.x; e0 < n * row; e0 += U * kT) {
    Pack<V> p[U][kBoth];
    const float2* cs[U];
    float* to[U];
    int apart[U];                    // of the item's two packs; 0: copied or absent
    bool here[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * kT;
      here[u] = e < n * row;
      if (!here[u]) continue;
      const int at = s.by_row(e), h = s.by_items(e - at * row), k = e - at * row - h * items;
      const bool turns = k < turned;
      const int c = turns ? (APART ? k * V : 2 * k * kPairs) : s.r + (k - turned) * V;
      const float* from = xb + at * s.x_ts + h * s.d + c;
      to[u] = yb + (int64_t)at * D + h * s.d + c;
      cs[u] = table + at * pairs + k * kPairs;
      apart[u] = turns ? (APART ? pairs : 1) : 0;
      p[u][0] = load<V>(from);
      if (kBoth == 2 && turns) p[u][kBoth - 1] = load<V>(from + apart[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!here[u]) continue;
      if (apart[u]) {
        if (kBoth == 2) {
#pragma unroll
          for (int i = 0; i < V; ++i) turn(p[u][0].v[i], p[u][kBoth - 1].v[i], cs[u][i]);
          store<V>(to[u] + apart[u], p[u][kBoth - 1]);
        } else {
#pragma unroll
          for (int i = 0; i + 1 < V; i += 2) turn(p[u][0].v[i], p[u][0].v[i + 1], cs[u][i / 2]);
        }
      }
      store<V>(to[u], p[u][0]);
    }
  }
}

template <bool APART>
void launch(int v, unsigned grid, float* y, const float* x, const Turns& turns, const Shape& s) {
  if (v == 4)
    rotary_kernel<4, APART><<<grid, kT, 0, wxx::stream()>>>(y, x, turns, s);
  else if (v == 2)
    rotary_kernel<2, APART><<<grid, kT, 0, wxx::stream()>>>(y, x, turns, s);
  else
    rotary_kernel<1, APART><<<grid, kT, 0, wxx::stream()>>>(y, x, turns, s);
}

}  // namespace

// y (B, T, heads * d) from x (unit stride inside, batch and time strides x_bs and x_ts);
// turns (host): r / 2 numbers, the full turns a position of every pair; gain: the factor on
// the turned channels; apart: pairs are (i, i + r / 2), else (2 i, 2 i + 1); back: the
// gradient's map.  positions (NULL: 0, 1, ...): (B, T) with batch stride p_bs (0: one row
// for all); offset is added to them.
WXX_EXPORT int wxx_rotary(float* y, const float* x, int64_t x_bs, int64_t x_ts,
                          const uint32_t* positions, int64_t p_bs, int64_t offset,
                          const double* turns, int r, float gain, int64_t B, int64_t T,
                          int64_t heads, int64_t d, int apart, int back) {
  WXX_REQUIRE_INIT();
  WXX_REQUIRE(B >= 0 && T >= 0 && heads >= 0 && d >= 0, "wxx_rotary: negative size");
  WXX_REQUIRE(r >= 0 && r % 2 == 0 && r <= d && r <= 2 * kMostPairs,
              "wxx_rotary: %d turned channels of %lld (even, at most %d)", r, (long long)d,
              2 * kMostPairs);
  WXX_REQUIRE(heads * d < (int64_t(1) << 22) && T < (int64_t(1) << 31) - 1,
              "wxx_rotary: %lld channels or %lld positions are too many", (long long)(heads * d),
              (long long)T);
  if (B * T * heads * d == 0) return WXX_OK;
  Turns table;
  for (int i = 0; i < r / 2; ++i) table.per[i] = turns[i];
  for (int i = r / 2; i < kMostPairs; ++i) table.per[i] = 0;
  // Positions of a block: enough channels to keep its threads in loads, a table that fits,
  // and blocks enough for the GPU's SMs where there are positions for them.
  const int64_t D = heads * d;
  int64_t at_once = kElements / D;
  if (r > 0 && at_once > kSinCos / (r / 2)) at_once = kSinCos / (r / 2);
  const int64_t spread = B * T / (4 * (int64_t)wxx::num_sms());
  if (at_once > spread) at_once = spread;
  if (at_once < 1) at_once = 1;
  if (at_once > T) at_once = T;
  const int64_t tiles = (T + at_once - 1) / at_once;
  WXX_REQUIRE(B * tiles < (int64_t(1) << 31), "wxx_rotary: too many positions");
  // Channels at a time: as many as divide a head's parts and every row's alignment.
  const uint64_t address = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y);
  auto fits = [&](int v) {
    return address % (4 * v) == 0 && ((B > 1 ? x_bs : 0) | x_ts | d) % v == 0 &&
           (apart ? r / 2 : r) % v == 0;
  };
  const int v = fits(4) ? 4 : fits(2) ? 2 : 1;
  const int kept = (int)d - r, items = (apart || v == 1 ? r / 2 / v : r / v) + kept / v;
  const Shape s{x_bs, x_ts, positions, p_bs, offset, (int)T, (int)heads, (int)d, r, (int)at_once,
                (int)tiles, gain, back ? -1.0f : 1.0f, Divider::of((unsigned)(r > 1 ? r / 2 : 1)),
                Divider::of((unsigned)(heads * items)), Divider::of((unsigned)items)};
  const unsigned grid = (unsigned)(B * tiles);
  if (apart)
    launch<true>(v, grid, y, x, table, s);
  else
    launch<false>(v, grid, y, x, table, s);
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}
