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
constexpr int kSteps = 16;          // positions of a thread
constexpr int kWarps = 8;           // pieces of a tile, at most
constexpr int kGroup = 32;          // tiles joined without a chain
constexpr int kSeg = kGroup / kWarps;
constexpr int kWaitLimit = 1 << 21; // polls of a published word (about a second)

// A gate as its smaller weight (<= 1/2) with the sign telling which it is:
// positive: z = 1 - a, the state is kept for the most part; negative: a.  With
// e = exp(-|g|) the smaller weight is e / (1 + e), good to a few ulp of itself
// (e^(-|g|) carries half an ulp of |g| log2 e).
__device__ __forceinline__ float gate_weight(float g) {
  const float e = fast_exp2(fabsf(g) * -1.4426950408889634f);
  const float w = __fdividef(e, 1.0f + e);
  return copysignf(w, g);          // a NaN stays one
}
__device__ __forceinline__ bool keeps(float w) { return __float_as_int(w) >= 0; }
__device__ __forceinline__ float weight_a(float w) { return keeps(w) ? 1.0f - w : -w; }
__device__ __forceinline__ float weight_z(float w) { return keeps(w) ? w : 1.0f + w; }

// a h + z x as the larger-weighted of the two plus the smaller weight times
// their difference: a constant gate's fixed point stays where it is (a and z,
// each rounded, do not add up to 1: at z = 1e-3 that error is multiplied by
// 1000), and a saturated gate keeps or replaces h exactly.
__device__ __forceinline__ float mix(float w, float h, float x) {
  const float base = keeps(w) ? h : x, other = keeps(w) ? x : h;
  return fmaf(fabsf(w), other - base, base);
}

// What a stretch of positions does to the state before it: h -> A h + b.  A
// reset inside cuts the state off, whatever it is (NaN included): A = -0, which
// no product of weights gives, stands for that.
struct Stretch {
  float A, b;
};
__device__ __forceinline__ bool cuts(float A) { return __float_as_uint(A) == 0x80000000u; }
__device__ __forceinline__ float through(Stretch s, float h) {
  return cuts(s.A) ? s.b : fmaf(s.A, h, s.b);
}
__device__ __forceinline__ Stretch join(Stretch first, Stretch then) {
  return {cuts(then.A) ? then.A : first.A * then.A, through(then, first.b)};
}

struct Operand {            // (B, T, ...) with unit stride inside
  const float* p;
  int64_t bs, ts;
};

// Scratch of a row of tiles, zero at launch.  Every published number travels
// with a flag in the upper half of its 64-bit word, so a reader needs no fence.
struct Chain {
  unsigned* ticket;
  ulonglong2* tile;         // {A, b} of a tile, 32 channels
  unsigned long long* group;  // the state after each group of kGroup tiles
  int64_t blocks;           // blocks of 32 channels
  int tiles;                // tiles of a row
  int* err;
};

__device__ __forceinline__ unsigned long long flagged(float v) {
  return (1ull << 32) | __float_as_uint(v);
}
__device__ __forceinline__ void publish(unsigned long long* p, float v) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(flagged(v)) : "memory");
}
__device__ __forceinline__ void publish(ulonglong2* p, Stretch s) {
  asm volatile("st.relaxed.gpu.global.v2.u64 [%0], {%1, %2};" ::"l"(p), "l"(flagged(s.A)),
               "l"(flagged(s.b))
               : "memory");
}
__device__ __forceinline__ bool peek(const unsigned long long* p, float& v) {
  unsigned long long u;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(u) : "l"(p) : "memory");
  v = __uint_as_float((unsigned)u);
  return (u >> 32) != 0;
}
__device__ __forceinline__ bool peek(const ulonglong2* p, Stretch& s) {
  unsigned long long u, v;
  asm volatile("ld.relaxed.gpu.global.v2.u64 {%0, %1}, [%2];" : "=l"(u), "=l"(v) : "l"(p) : "memory");
  s.A = __uint_as_float((unsigned)u);
  s.b = __uint_as_float((unsigned)v);
  return (u >> 32) != 0 && (v >> 32) != 0;
}
// Polls end when every lane has its words, or give up: at the limit (error word
// set) or as soon as another block has given up.  Returns whether to stop.
__device__ __forceinline__ bool poll_over(bool ready, int& n, int* err) {
  if (__all_sync(0xffffffffu, ready)) return true;
  ++n;
  if (n >= kWaitLimit) {
    wxx_device_fail(err, WXX_DEV_ERR_MBAR_TIMEOUT);
    return true;
  }
  return (n & 1023) == 0 && *reinterpret_cast<volatile int*>(err) == WXX_DEV_ERR_MBAR_TIMEOUT;
}

struct Joint {               // shared memory of a tile's join
  Stretch piece[kWarps][32];
  Stretch before[kWarps][32];
  float group[32];
  int tile;
};

// The tile that this block takes.  Tiles are handed out in the order of their
// rows' join, so whoever a block waits for has started before it.
__device__ __forceinline__ int64_t take_tile(const Chain& c, Joint& s) {
  if (c.tiles == 1) return blockIdx.x;
  if (threadIdx.x == 0) s.tile = (int)atomicAdd(c.ticket, 1u);
  __syncthreads();
  return s.tile;
}

// Joins the pieces of a tile (warp i of the order holds piece `mine`) with
// everything before it.  j: the tile's place in its row, q: its channel block.
// Returns the state before this warp's piece.  The order of the additions
// depends on j alone: the tiles of the same group so far, in kWarps segments,
// then the state after the group before.
__device__ float join_tile(const Chain& c, Joint& s, int i, Stretch mine, int j, int64_t q,
                           float start) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  s.piece[i][lane] = mine;
  __syncthreads();
  if (c.tiles == 1) {
    float h = start;
    for (int k = 0; k < i; ++k) h = through(s.piece[k][lane], h);
    return h;
  }
  const int r = j % kGroup, g = j / kGroup;
  const int64_t row = q * c.tiles;
  if (i == 0) {
    Stretch all = mine;
    for (int k = 1; k < warps; ++k) all = join(all, s.piece[k][lane]);
    publish(c.tile + (row + j) * 32 + lane, all);
  }
  // segment i: tiles i kSeg .. of the group, those before r
  Stretch seg[kSeg];
  int n = 0;
  while (true) {
    bool ready = true;
#pragma unroll
    for (int k = 0; k < kSeg; ++k) {
      seg[k] = {1.0f, 0.0f};
      if (i * kSeg + k < r)
        ready = peek(c.tile + (row + g * kGroup + i * kSeg + k) * 32 + lane, seg[k]) && ready;
    }
    if (poll_over(ready, n, c.err)) break;
  }
  Stretch before = seg[0];
#pragma unroll
  for (int k = 1; k < kSeg; ++k) before = join(before, seg[k]);
  s.before[i][lane] = before;
  if (i == 0) {
    float h = start;
    if (g > 0) {
      n = 0;
      while (!poll_over(peek(c.group + (q * ((c.tiles + kGroup - 1) / kGroup) + g - 1) * 32 + lane, h),
                        n, c.err)) {
      }
    }
    s.group[lane] = h;
  }
  __syncthreads();
  float h = s.group[lane];
#pragma unroll
  for (int k = 0; k < kWarps; ++k) h = through(s.before[k][lane], h);
  for (int k = 0; k < i; ++k) h = through(s.piece[k][lane], h);
  if (i == warps - 1 && r == kGroup - 1)
    publish(c.group + (q * ((c.tiles + kGroup - 1) / kGroup) + g) * 32 + lane, through(mine, h));
  return h;
}

__device__ __forceinline__ int positions_left(int64_t T, int64_t t0) {
  const int64_t n = T - t0;
  return n < 0 ? 0 : n < kSteps ? (int)n : kSteps;
}

// Positions t0 .. t0 + kSteps - 1 of sequence b that start a document, as bits.
__device__ __forceinline__ unsigned reset_bits(const uint32_t* __restrict__ reset, int64_t b,
                                               int64_t T, int64_t t0, bool in) {
  if (!reset) return 0u;
  const int lane = threadIdx.x & 31;
  const int64_t b0 = __shfl_sync(0xffffffffu, b, 0);
  if (__all_sync(0xffffffffu, !in || b == b0))   // one sequence: a lane per position
    return __ballot_sync(0xffffffffu,
                         lane < kSteps && t0 + lane < T && reset[b0 * T + t0 + lane] != 0);
  unsigned bits = 0;
  if (in)
    for (int k = 0; k < kSteps; ++k)
      bits |= (unsigned)(t0 + k < T && reset[b * T + t0 + k] != 0) << k;
  return bits;
}

// A tile is 32 channels (of the batch x channels rows side by side) by up to
// kWarps pieces of kSteps positions, one piece a warp: the piece's inputs stay in
// registers while the state before it is found, so each is read once and h is
// written once, 12 bytes a position.  A piece is first run from a zero state for
// its (A, b), then once more from the state that the join gives.
__global__ void __launch_bounds__(kT)
    recurrence_forward_kernel(float* __restrict__ h, float* __restrict__ h_last, Operand x,
                              Operand g, const float* __restrict__ h0,
                              const uint32_t* __restrict__ reset, int64_t B, int64_t T, int64_t D,
                              int64_t per, Chain c) {
  __shared__ Joint s;
  const int64_t id = take_tile(c, s);
  const int j = (int)(id / c.blocks);
  const int64_t q = id - j * c.blocks, ch = q * 32 + (threadIdx.x & 31);
  const int i = threadIdx.x >> 5;
  const int64_t t0 = ((int64_t)j * (blockDim.x >> 5) + i) * kSteps;
  const bool in = ch < B * D;
  const int64_t b = in ? ch / D : 0, d = in ? ch - b * D : 0;
  const float* xp = x.p + b * x.bs + t0 * x.ts + d;
  const float* gp = g.p + b * g.bs + t0 * g.ts + d / per;
  const int left = in ? positions_left(T, t0) : 0;
  float xv[kSteps], w[kSteps];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    xv[k] = k < left ? *xp : 0.f;
    w[k] = k < left ? *gp : INFINITY;         // past the end: keep the state
    xp += x.ts;
    gp += g.ts;
  }
  const unsigned cut = reset_bits(reset, b, T, t0, in);
  Stretch mine = {1.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    w[k] = gate_weight(w[k]);
    if (cut >> k & 1) mine = {-0.0f, 0.0f};
    mine.b = mix(w[k], mine.b, xv[k]);
    mine.A *= weight_a(w[k]);
  }
  float v = join_tile(c, s, i, mine, j, q, in && h0 ? h0[ch] : 0.f);
  float* hp = h + (b * T + t0) * D + d;
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    if (cut >> k & 1) v = 0.f;
    v = mix(w[k], v, xv[k]);
    if (k < left) *hp = v;
    if (k == left - 1 && t0 + left == T) h_last[ch] = v;
    hp += D;
  }
}

// The same tiles with time reversed: c_t = a_t r_t (dh_t + c_{t+1}) is what
// position t hands to t - 1.  Reads dh, x, gate, h, writes dx, dgate: 24 bytes a
// position.  DG: where the gate's gradient goes -- 1: sums over the `per` lanes
// of a head (a power of two up to 32; lane 0 of them writes), 32: sums over the
// warp, one partial sum per block of 32 channels; 0: every channel's own.
template <int DG>
__global__ void __launch_bounds__(kT)
    recurrence_backward_kernel(float* __restrict__ dx, float* __restrict__ dg,
                               float* __restrict__ dh0, const float* __restrict__ dh,
                               const float* __restrict__ dlast, Operand x, Operand g,
                               const float* __restrict__ h, const float* __restrict__ h0,
                               const uint32_t* __restrict__ reset, int64_t B, int64_t T, int64_t D,
                               int64_t per, Chain c) {
  __shared__ Joint s;
  const int64_t id = take_tile(c, s);
  const int j = (int)(id / c.blocks);
  const int64_t q = id - j * c.blocks, ch = q * 32 + (threadIdx.x & 31);
  const int warps = blockDim.x >> 5, i = threadIdx.x >> 5;
  // the order runs from the last position: warp i holds piece i of it
  const int64_t t0 = ((int64_t)(c.tiles - 1 - j) * warps + (warps - 1 - i)) * kSteps;
  const bool in = ch < B * D;
  const int64_t b = in ? ch / D : 0, d = in ? ch - b * D : 0;
  const int64_t at = (b * T + t0) * D + d;
  const float* xp = x.p + b * x.bs + t0 * x.ts + d;
  const float* gp = g.p + b * g.bs + t0 * g.ts + d / per;
  const int left = in ? positions_left(T, t0) : 0;
  const float *dp = dh + at, *hp = h + at;
  float u[kSteps], w[kSteps], gv[kSteps], xv[kSteps];
  u[0] = left == 0 ? 0.f : t0 > 0 ? *(hp - D) : h0 ? h0[ch] : 0.f;
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    w[k] = k < left ? *gp : INFINITY;
    gv[k] = k < left ? *dp : 0.f;
    xv[k] = k < left ? *xp : 0.f;
    if (k + 1 < kSteps) u[k + 1] = k + 1 < left ? *hp : 0.f;
    gp += g.ts;
    dp += D;
    xp += x.ts;
    hp += D;
  }
  const unsigned cut = reset_bits(reset, b, T, t0, in);
  Stretch mine = {1.0f, 0.0f};
#pragma unroll
  for (int k = kSteps - 1; k >= 0; --k) {
    w[k] = gate_weight(w[k]);
    const float a = weight_a(w[k]);
    mine.b = a * (gv[k] + mine.b);
    mine.A *= a;
    if (cut >> k & 1) {
      mine = {-0.0f, 0.0f};
      u[k] = 0.f;
    }
    // d a / d gate = a z
    u[k] = (u[k] - xv[k]) * (fabsf(w[k]) * (1.0f - fabsf(w[k])));
  }
  float v = join_tile(c, s, i, mine, j, q, in && dlast ? dlast[ch] : 0.f);
  const int64_t heads = DG == 1 ? D / per : DG == 32 ? D / 32 : D;
  const int64_t lanes = DG == 1 ? per : DG == 32 ? 32 : 1;
  float* xo = dx + at + (kSteps - 1) * D;
  float* go = dg + (b * T + t0 + kSteps - 1) * heads + d / lanes;
#pragma unroll
  for (int k = kSteps - 1; k >= 0; --k) {
    const float G = gv[k] + v;
    if (k < left) *xo = weight_z(w[k]) * G;
    float e = G * u[k];
    if (DG == 1) {
      for (int o = 1; o < per; o <<= 1) e += __shfl_xor_sync(0xffffffffu, e, o);
    } else if (DG == 32) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) e += __shfl_xor_sync(0xffffffffu, e, o);
    }
    if (k < left && (DG == 0 || d % lanes == 0)) *go = e;
    v = cut >> k & 1 ? 0.f : weight_a(w[k]) * G;
    xo -= D;
    go -= heads;
  }
  if (dh0 && in && t0 == 0) dh0[ch] = v;
}

__global__ void recurrence_step_kernel(float* __restrict__ state, const float* __restrict__ x,
                                       int64_t x_ld, const float* __restrict__ g, int64_t g_ld,
                                       int64_t n, int64_t D, int64_t per) {
  for (int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * kT) {
    const int64_t b = i / D, d = i - b * D;
    state[i] = mix(gate_weight(g[b * g_ld + d / per]), state[i], x[b * x_ld + d]);
  }
}

// Threads and blocks of a scan, and its scratch (freed by the caller).
int plan_scan(const char* what, int64_t B, int64_t T, int64_t D, Chain& c, unsigned& threads,
              unsigned& grid, void** scratch) {
  const int64_t pieces = (T + kSteps - 1) / kSteps;
  const int64_t warps = pieces < kWarps ? pieces : kWarps;
  c.tiles = (int)((pieces + warps - 1) / warps);
  c.blocks = (B * D + 31) / 32;
  c.err = wxx::device_error_word();
  c.ticket = nullptr;
  c.tile = nullptr;
  c.group = nullptr;
  *scratch = nullptr;
  threads = (unsigned)(warps * 32);
  WXX_REQUIRE(c.blocks * c.tiles < (int64_t(1) << 31), "%s: too many elements", what);
  grid = (unsigned)(c.blocks * c.tiles);
  if (c.tiles == 1) return WXX_OK;
  const int64_t groups = (c.tiles + kGroup - 1) / kGroup;
  const size_t tile_bytes = (size_t)c.blocks * c.tiles * 32 * sizeof(ulonglong2);
  const size_t bytes = 256 + tile_bytes + (size_t)c.blocks * groups * 32 * 8;
  if (int st = wxx_malloc(scratch, bytes)) return st;
  char* p = static_cast<char*>(*scratch);
  c.ticket = reinterpret_cast<unsigned*>(p);
  c.tile = reinterpret_cast<ulonglong2*>(p + 256);
  c.group = reinterpret_cast<unsigned long long*>(p + 256 + tile_bytes);
  cudaError_t e = cudaMemsetAsync(p, 0, bytes, wxx::stream());
  if (e != cudaSuccess) {
    wxx_free(*scratch);
    wxx::set_error("%s: clearing the scratch failed: %s", what, cudaGetErrorString(e));
    return WXX_E_CUDA;
  }
  return WXX_OK;
}

// The state after no positions: `from` or zero.
int copy_state(float* to, const float* from, int64_t n) {
  if (from)
    WXX_CUDA_CHECK(cudaMemcpyAsync(to, from, (size_t)n * sizeof(float), cudaMemcpyDeviceToDevice,
                                   wxx::stream()));
  else
    WXX_CUDA_CHECK(cudaMemsetAsync(to, 0, (size_t)n * sizeof(float), wxx::stream()));
  return WXX_OK;
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
  if (T == 0) return copy_state(h_last, h0, B * D);
  Chain c;
  unsigned threads, grid;
  void* scratch;
  if (int st = plan_scan("wxx_gated_recurrence", B, T, D, c, threads, grid, &scratch)) return st;
  recurrence_forward_kernel<<<grid, threads, 0, wxx::stream()>>>(
      h, h_last, Operand{x, x_bs, x_ts}, Operand{gate, g_bs, g_ts}, h0, reset, B, T, D, D / H, c);
  const int st = wxx::after_launch(__FILE__, __LINE__);
  if (scratch) wxx_free(scratch);
  return st;
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
  if (T == 0) return dh0 ? copy_state(dh0, dlast, B * D) : WXX_OK;
  // The gate's gradient is summed over a head's channels in the kernel where
  // they lie in one warp's 32 neighbours, by partial sums per 32 channels where
  // they are several warps', and from every channel's own otherwise.
  const int64_t per = D / H;
  const bool inside = per <= 32 && (per & (per - 1)) == 0, partial = per > 32 && per % 32 == 0;
  const int64_t parts = partial ? per / 32 : per;
  float* sums = dgate;
  void *scratch = nullptr, *wide = nullptr;
  Chain c;
  unsigned threads, grid;
  if (!inside) {
    if (int st = wxx_malloc(&wide, (uint64_t)(B * T * H * parts) * sizeof(float))) return st;
    sums = static_cast<float*>(wide);
  }
  int st = plan_scan("wxx_gated_recurrence_backward", B, T, D, c, threads, grid, &scratch);
  if (st == WXX_OK) {
    auto kernel = per == 1 || (!inside && !partial) ? recurrence_backward_kernel<0>
                  : inside                          ? recurrence_backward_kernel<1>
                                                    : recurrence_backward_kernel<32>;
    kernel<<<grid, threads, 0, wxx::stream()>>>(dx, sums, dh0, dh, dlast, Operand{x, x_bs, x_ts},
                                                Operand{gate, g_bs, g_ts}, h, h0, reset, B, T, D,
                                                per, c);
    st = wxx::after_launch(__FILE__, __LINE__);
    if (st == WXX_OK && wide) st = wxx_reduce(dgate, sums, B * T * H, parts, 1, 0);
  }
  if (scratch) wxx_free(scratch);
  if (wide) wxx_free(wide);
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
