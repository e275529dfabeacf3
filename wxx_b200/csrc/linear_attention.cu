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

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "tc_gemm.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

WXX_EXPORT int wxx_malloc(void** out, uint64_t nbytes);
WXX_EXPORT int wxx_free(void* p);

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
  // the scales as units in [1, 2) (or 0) and powers of two, which stay in range beside others
  float y_unit, out_unit;
  int y_exp, out_exp;
};
float unit_of(float scale, int& exp) {
  const float half = frexpf(scale, &exp);
  --exp;
  return 2.f * half;
}

struct Shape {
  const float* log_decay;   // (H)
  const uint32_t* reset;    // (B, T) or NULL
  int T, H;
};

constexpr int kT = 256;

// One position's decay of a state, l X.  A decay near 1 is applied as X + (l - 1) X: l alone
// is rounded to 2^-25, which n positions in a row make n 2^-25.
// (An infinite state takes l itself: of the two terms' signs one is the other's opposite.)
// The same for n positions at once, with n log l in the place of log l: a chunk's l^64, rounded
// alike in every chunk, left a state after 32768 positions with a memory of 2^18 off by 7e-6, h0's
// part of it by 1.5e-5; now 2.4e-7 and 3e-7.
__device__ __forceinline__ float whole_of(float log_decay) { return log_decay > -0.5f ? 1.f : 0.f; }
__device__ __forceinline__ float less_of(float log_decay) {
  return log_decay > -0.5f ? expm1f(log_decay) : expf(log_decay);
}
struct Decay {
  float l, less, whole;
  __device__ explicit Decay(float log_decay)
      : l(expf(log_decay)), less(less_of(log_decay)), whole(whole_of(log_decay)) {}
  __device__ __forceinline__ float operator()(float X) const {
    return fabsf(X) < INFINITY ? fmaf(less, X, whole * X) : l * X;
  }
};

// A block per sequence, head and 32 columns of X: lane = column, warp = every 8th row,
// K rows a thread.  One position after the other: for heads of more than 128 channels, whose
// state the chunks' kernel has no room for.
__global__ void __launch_bounds__(kT) sweep_kernel(const Pass a, const Shape s) {
  constexpr int K = 32, kTile = 8;      // rows, positions of a tile
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

// ------------------------------------------------------------------ chunks
//
// A chunk of 64 positions at a time, so that the work is products of matrices.  With X the
// state that applies to the chunk's first position (its decay and a reset there already
// taken), i and j positions of the chunk and l^n powers of the decay, forwards:
//
//   out_i = l^i X^T x_i + sum over j <= i of l^(i - j) (x_i . y_j) z_j
//   X' = l^n X + sum of l^(n - j) y_j z_j^T
//
// with every term left out that a reset separates; backwards the same from the chunk's
// other end.
//
// Four products a chunk (x y^T, its result with z, x X, y^T z) of 26.6 thousand operations a
// position at 64 channels, four times the bytes: on FP32 units (65 TFLOP/s measured) they
// would take 2.5 times as long as the memory.  They run on the tensor cores in half
// precision, three products for one: every operand is split into a high and a low half of
// 11 bits each, hi hi + hi lo + lo hi, which leaves out 2^-22 of a product.  Half numbers
// reach from 2^-24 to 2^16 only, so each row (a position's vector of x, y or z, a row of the
// position-by-position matrix) is scaled by a power of two that brings its length (in the
// matrix its largest entry) to 2^13, and a state by one for all of it; the powers are put
// back in 32 bits.  Entries far below their row's length lose accuracy from 2^-20 of it on
// (they are good to 2^-38 of it).  (Measured, mma.sync: half 554, tf32 277 TFLOP/s; three
// products of tf32 need no scaling, but would be bound by that rate.  On tcgen05, kind::tf32
// with sums in TMEM, chunks of 128 took as long, and the truncated sums made the error 1.6e-6
// instead of 5e-7 to 7e-7.)  The state stays in 32-bit registers, a chunk's products are added to
// it in 32 bits.
//
// NaN and infinities cannot take part: 0 times NaN would carry them to earlier positions
// and other documents.  A chunk with a row whose length is not between 2^-60 and 2^63 (or 0),
// or with a state longer than that, is worked through position by position (rare_chunk); and one whose products
// of lengths |y_j| |z_j| are more than 2^110 apart, so that a later position, or another
// document's, cannot cost one its value.

using wxx_tc::mbar_arrive_expect_tx;
using wxx_tc::mbar_init;
using wxx_tc::mbar_wait;
using wxx_tc::tma_load_4d;

constexpr int kC = 64;                  // positions of a chunk
constexpr int kThreads = 128;           // 4 warps of 16 positions
constexpr int kTop = 13;                // a scaled row's length is in [2^13, 2^14)

__device__ __forceinline__ uint32_t smem_address(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void copy4(uint32_t to, const float* from, bool take) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from),
               "r"(take ? 4 : 0));
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Four 8 x 8 matrices of halves at `at` and a constant; turned: each the other way round.
template <int OFF>
__device__ __forceinline__ void load4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at), "n"(OFF)
               : "memory");
}
template <int OFF>
__device__ __forceinline__ void load4_turned(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at), "n"(OFF)
               : "memory");
}
template <int OFF>
__device__ __forceinline__ void store4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0 + %5], {%1, %2, %3, %4};" ::"r"(at),
               "r"(a), "r"(b), "r"(c), "r"(d), "n"(OFF)
               : "memory");
}
// f with each of 0 to N - 1 as a constant.
template <int N, int I = 0, class F>
__device__ __forceinline__ void for_each(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    for_each<N, I + 1>(f);
  }
}
__device__ __forceinline__ void product(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Products to 22 bits of a left operand with two right ones next to each other: the halves'
// but that of the two low ones, the small ones first.
__device__ __forceinline__ void products(float (&c0)[4], float (&c1)[4], const uint32_t (&hi)[4],
                                         const uint32_t (&lo)[4], const uint32_t (&bh)[4],
                                         const uint32_t (&bl)[4]) {
  product(c0, lo, bh[0], bh[1]);
  product(c1, lo, bh[2], bh[3]);
  product(c0, hi, bl[0], bl[1]);
  product(c1, hi, bl[2], bl[3]);
  product(c0, hi, bh[0], bh[1]);
  product(c1, hi, bh[2], bh[3]);
}

// The high and low halves of two numbers times `up`.  (The low one from a product of mixed types,
// exact: f - hi 1; unpacked and subtracted the forward over 37 x 1024 tokens of 16 heads of 64
// took 265 instead of 260 us.)
__device__ __forceinline__ void split(float a, float b, float up, uint32_t& hi, uint32_t& lo) {
  mul2(a, b, a, b, up, up);
  const __half2 h = __floats2half2_rn(a, b);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  asm("{\n\t.reg .f16 x, y, minus;\n\tmov.b32 {x, y}, %2;\n\tmov.b16 minus, 0xBC00;\n\t"
      "fma.rn.f32.f16 %0, x, minus, %0;\n\tfma.rn.f32.f16 %1, y, minus, %1;\n\t}"
      : "+f"(a), "+f"(b)
      : "r"(hi));
  const __half2 l = __floats2half2_rn(a, b);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {      // two halves each
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Sums of squares, in two parts.
__device__ __forceinline__ void square2(float& s0, float& s1, float a, float b) {
  fma2(s0, s1, a, b, a, b, s0, s1);
}
// Whether a row of this square (or a state, of the larger one) cannot be scaled; 0 alone says
// nothing yet.
constexpr float kShort = 0x1p-120f, kLong = 0x1p126f;
// Rows of y and z with squares between these are not too far apart, and with x up to the larger and a
// state up to its square what decays below 2^-126 is below 2^-45, and taken as 0; in a chunk beyond
// them such decays are worked through position by position.
constexpr float kBelow = 0x1p-54f, kAbove = 0x1p54f;
constexpr int kApart = 110;
// A state shorter than 2^-60, as the decays leave it behind a sequence's last token, is scaled by its
// largest entry (times 64: its length is 90 of them at most), and by 2^127 at most: halves then leave
// out less than 2^-150, which 32 bits cannot say either.  (Position by position a row of 4096
// positions whose last 3584 have keys and values of 0 took 1490 us instead of 141, 64 channels, 40
// sequences; backward 12.0 ms instead of 0.4.)
constexpr int kNoState = -1000;
// The exponent of a length with this square.
__device__ __forceinline__ int exponent(float square) {
  return ((int)(__float_as_uint(square) >> 23) - 127) >> 1;
}
__device__ __forceinline__ float power2(int e) {            // -126 <= e <= 127
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// f 2^e, f about 1, in two steps: the second is 1 unless 2^e is out of range.
struct Scale {
  float first, then;
  __device__ Scale(float f, int e) {
    e = min(max(e, -250), 250);
    const int one = min(max(e, -125), 125);
    first = f * power2(one);
    then = power2(e - one);
  }
};

// Tiles of W half numbers a row for ldmatrix: 16-byte pieces of a row exchanged so that
// the same piece of 8 rows lies in 8 different sets of banks.  (q ^ k << 1 is the address of q
// with k << 5 exchanged: how the products below step through a row.)
template <int W>
__device__ __forceinline__ uint32_t piece(int row, int q) {
  const int turn = W == 32 ? (row >> 1) & 3 : row & 7;
  return (uint32_t)(row * W * 2 + ((q ^ turn) << 4));
}
// 32 columns of all positions as the copy engine leaves them, 16-byte pieces exchanged.
__device__ __forceinline__ int raw_piece(int row, int q) { return row * 8 + (q ^ (row & 7)); }
constexpr int kRaw = kC * 128;          // their bytes

// (STATE does without x and the state's tile, which makes room for a third block of 64 by 64: 366
// -> 338 us forward over 16 x 8192 tokens of 4 heads of 64, 110 -> 92 over 3 x 4097 of 5 heads of
// 40 by 72.)
template <int P, int R, bool STATE, bool AHEAD>
struct Layout {
  static constexpr int kRawX = 0, kRawY = STATE ? 0 : P / 32 * kRaw, kRawZ = kRawY + P / 32 * kRaw;
  // high halves, then low halves, of y and z (AHEAD: not where the copies go) and the state
  static constexpr int kY = AHEAD ? kRawZ + R / 32 * kRaw : kRawY, kZ = kY + kC * P * 4;
  static constexpr int kState = kZ + kC * R * 4, kTiles = AHEAD ? kY : 0;
  static constexpr int kEnd = kState + (STATE ? 0 : P * R * 4), kBytes = kEnd + 1024;
  static_assert((P * R + kThreads) * 4 + kC <= (AHEAD ? kState : kEnd) - kTiles, "rare_chunk's room");
  // the warps' parts of the state: kRowTiles times 16 rows by kColTiles tiles of 8 columns
  static constexpr int kRowTiles = P >= 64 ? P / 64 : 1, kColTiles = P >= 64 ? R / 8 : R / 16;
  static constexpr int kBlocks = P == 128                ? (STATE ? 2 : 1)
                                 : P == 64 && R == 64 ? (AHEAD && !STATE ? 2 : 3)
                                 : P == 32 && R == 32 ? 4
                                                      : 3;
};

struct Segments {           // pieces of a row that are worked on side by side
  int count, chunks;        // pieces, chunks of a piece
  float* state;             // (passes, count - 1, B H, p * r): after each piece but the last
  float2* kept;             // (passes, count - 1, B H): what a piece leaves of a state X before it, y =
                            // 1: X + x X; 0: x^2 X (l^n may be out of range); -1: 0, a reset is in it
};

// The chunk's weights of decay and resets.
struct Weights {
  unsigned long long inner; // the resets after the chunk's first position
  int first, last;          // of these; 64 and 0: none
  int n, tail;              // positions; 1 where the state goes on past the chunk's end
  bool drop;                // a reset there: the next chunk starts from zero
  __device__ Weights(unsigned long long cuts, int n_, int tail_, bool drop_)
      : inner(cuts & ~1ull), n(n_), tail(tail_), drop(drop_) {
    first = inner ? __ffsll((long long)inner) - 1 : 64;
    last = inner ? 63 - __clzll((long long)inner) : 0;
  }
  // exponents of l, -1: no weight
  __device__ __forceinline__ int reach(int i, bool back) const {     // of the state, at i
    return back ? (i >= last && i < n ? n - 1 - i : -1) : (i < first && i < n ? i : -1);
  }
  __device__ __forceinline__ int added(int j, bool back) const {     // of j, to the state
    if (drop || j >= n) return -1;
    return back ? (j < first ? j + 1 : -1) : (j >= last ? n - 1 - j + tail : -1);
  }
  __device__ __forceinline__ int kept(bool back) const {
    return drop || inner ? -1 : n - 1 + (back ? 1 : tail);
  }
  __device__ __forceinline__ int document(int i) const {
    return __popcll(inner & ((2ull << i) - 1));
  }
};

// A power of l as rest 2^e with rest in [1, 2); below 2^-126 it is none.
struct Decayed {
  bool any;
  int e;
  float rest;
  __device__ Decayed(const float* power, int u) {
    const uint32_t bits = u < 0 ? 0u : __float_as_uint(power[u]);
    any = bits >= 0x00800000u;
    e = any ? (int)(bits >> 23) - 127 : 0;
    rest = any ? __uint_as_float((bits & 0x007fffffu) | 0x3f800000u) : 1.f;
  }
};

// Whether the products of the lengths of a chunk's rows are too far apart, from their squares.
__device__ __forceinline__ bool far_apart(const float* square_y, const float* square_z) {
  int most = -1000, least = 1000;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int j = (threadIdx.x & 31) + 32 * k;
    if (square_y[j] == 0.f || square_z[j] == 0.f) continue;          // nothing there
    const int e = exponent(square_y[j]) + exponent(square_z[j]);
    most = max(most, e);
    least = min(least, e);
  }
  return __reduce_max_sync(0xffffffffu, most) - __reduce_min_sync(0xffffffffu, least) > kApart;
}

// The parts of shared memory that are not tiles.
struct alignas(16) Small {
  float square_y[kC], square_z[kC];     // of the rows
  float square_state[4];                // by warp; where that is short, minus the largest entry
  // per position j: 2^(exponents of y_j and z_j, below the largest) / what z_j's scale has more,
  // and that times l^(15 - j % 16) (back: l^(j % 16))
  float2 weight[kC];
  uint16_t added[2][kC];                // j's weight in the state, as a product of two halves
  float power[kC + 4];                  // l^n
  float2 kept[kC + 4];                  // what n positions leave of a state: Decay's less and whole
  int document[kC];
  uint64_t arrived;                     // y, z and x are here
  int look;                             // the last chunk that may have rows too far apart
  int abort;
};

// The passes of one launch: sweeps over the same B, T and H whose heads have the same
// padded sizes; and the maps of their operands, where the copy engine takes them.
struct Passes {
  Pass at[3];
};
struct Maps {
  CUtensorMap x[3], y[3], z[3];
};

// Position by position, for a chunk with numbers that are not finite or that cannot be
// scaled: the state in shared memory, columns over the lanes, rows over kThreads / R groups
// of threads.
template <int R, bool STATE>
__device__ void rare_chunk(float* state, float* sums, const unsigned char* cuts, const Pass& a,
                           const Shape& s, int n, bool tail, bool next_cut, Decay l, int64_t b,
                           int h, int t0, int slice) {
  constexpr int kGroups = kThreads / R;
  const int c = threadIdx.x % R, group = threadIdx.x / R, r = slice * R + c;
  for (int k = 0; k < n; ++k) {
    const int i = a.back ? n - 1 - k : k;
    const float* x = a.x.p + b * a.x.bs + (t0 + i) * a.x.ts + (int64_t)h * a.p;
    const float* y = a.y.p + b * a.y.bs + (t0 + i) * a.y.ts + (int64_t)h * a.p;
    const float z = r < a.r ? a.z.p[b * a.z.bs + (t0 + i) * a.z.ts + (int64_t)h * a.r + r] : 0.f;
    const bool on = k < n - 1 || a.back || tail;           // the state goes on from here
    const bool cut = a.back ? cuts[i] : k < n - 1 ? cuts[i + 1] : next_cut;
    float sum = 0.f;
    for (int p = group; p < a.p; p += kGroups) {
      float now = fmaf(a.y_scale * y[p], z, state[p * R + c]);
      if (!STATE) sum = fmaf(x[p], now, sum);
      if (on) now = cut ? 0.f : l(now);
      state[p * R + c] = now;
    }
    if (STATE) continue;
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (group == 0) {
      for (int g = 1; g < kGroups; ++g) sum += sums[g * R + c];
      if (r < a.r) a.out[((b * s.T + t0 + i) * s.H + h) * a.r + r] = a.out_scale * sum;
    }
    __syncthreads();
  }
}

// A block: one sequence, head, slice of R columns of z and piece of the row; STATE: only
// the state after the piece is wanted.  A warp has 16 positions of x and their outputs, and
// a part of the state; y and z are split by all warps and read by all.  AHEAD: the next
// chunk's operands are copied meanwhile; else they are copied, and split, in the place of this
// chunk's, which more blocks on an SM have room for (plan_of chooses).
template <int P, int R, bool STATE, bool AHEAD>
__global__ void __launch_bounds__(kThreads, Layout<P, R, STATE, AHEAD>::kBlocks)
    chunk_kernel(const __grid_constant__ Passes passes, const __grid_constant__ Maps maps,
                 const bool tma, const Shape s, const Segments g, const unsigned per_pass,
                 int* err) {
  using L = Layout<P, R, STATE, AHEAD>;
  extern __shared__ __align__(1024) unsigned char raw_smem[];
  __shared__ Small m;
  unsigned char* smem = raw_smem + ((1024 - (smem_address(raw_smem) & 1023)) & 1023);
  const uint32_t base = smem_address(smem);
  const unsigned pass = blockIdx.x / per_pass;
  const Pass& a = passes.at[pass];
  unsigned at = blockIdx.x % per_pass;
  const int slices = (a.r + R - 1) / R, pieces = STATE ? g.count - 1 : g.count;
  const int slice = at % slices;
  at /= slices;
  const int seg = at % pieces;
  at /= pieces;
  const int h = at % s.H;
  const int64_t b = at / s.H, heads = per_pass / (unsigned)(slices * pieces);   // B H
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, t = lane & 3;
  const int mat = lane >> 3, mat_row = lane & 7;
  const bool back = a.back;
  const Decay l(s.log_decay[h]);
  if (threadIdx.x <= kC) {
    const float n_log = (float)threadIdx.x * s.log_decay[h];
    const float power = threadIdx.x == 0 ? 1.f : expf(n_log), whole = whole_of(n_log);
    m.power[threadIdx.x] = power;
    m.kept[threadIdx.x] = make_float2(whole != 0.f ? expm1f(n_log) : power, whole);
  }

  const int chunks = (s.T + kC - 1) / kC;
  const int c0 = seg * g.chunks, c1 = min(c0 + g.chunks, chunks);
  // pieces and chunks are counted in the direction of the sweep
  auto start = [&](int c) { return (back ? chunks - 1 - c : c) * kC; };
  const uint32_t* marks = s.reset ? s.reset + b * s.T : nullptr;

  // x, y and z of a chunk into shared memory, 32 columns of all positions at a time
  auto fetch = [&](int c) {
    const int t0 = start(c);
    if (tma) {
      if (threadIdx.x == 0) {
        mbar_arrive_expect_tx(&m.arrived, ((STATE ? 1 : 2) * (P / 32) + R / 32) * kRaw);
#pragma unroll
        for (int k = 0; k < P / 32; ++k) {
          if (!STATE)
            tma_load_4d(base + L::kRawX + k * kRaw, &maps.x[pass], &m.arrived, 32 * k, h, t0, (int)b);
          tma_load_4d(base + L::kRawY + k * kRaw, &maps.y[pass], &m.arrived, 32 * k, h, t0, (int)b);
        }
#pragma unroll
        for (int k = 0; k < R / 32; ++k)
          tma_load_4d(base + L::kRawZ + k * kRaw, &maps.z[pass], &m.arrived, slice * R + 32 * k, h,
                      t0, (int)b);
      }
      return;
    }
    auto rows = [&](int to, const Operand& o, int columns, int from, int width) {
      const int n = min(kC, s.T - t0);
      const float* p = o.p + b * o.bs + t0 * o.ts + (int64_t)h * columns + from;
      for (int i = threadIdx.x; i < kC * width; i += kThreads) {
        const int row = i / width, col = i % width;
        const bool take = row < n && col < columns - from;
        copy4(base + to + (col >> 5) * kRaw + raw_piece(row, (col & 31) >> 2) * 16 + (col & 3) * 4,
              take ? p + row * o.ts + col : o.p, take);
      }
    };
    if (!STATE) rows(L::kRawX, a.x, a.p, 0, P);
    rows(L::kRawY, a.y, a.p, 0, P);
    rows(L::kRawZ, a.z, a.r, slice * R, R);
  };
  if (threadIdx.x == 0) {
    mbar_init(&m.arrived, 1);
    m.abort = 0;
    m.look = -1;
    wxx_tc::fence_barrier_init();
  }
  __syncthreads();
  fetch(c0);

  // the state, in the layout of a product's result: rows row0 + 16 mt + quad (+ 8), columns
  // col0 + 8 nt + 2 t (+ 1)
  const int row0 = P >= 64 ? warp * (P / 4) : (warp & 1) * 16;
  const int col0 = P >= 64 ? 0 : (warp >> 1) * (R / 2);
  float X[L::kRowTiles][L::kColTiles][4];
  auto each = [&](auto f) {             // f(entry, row, column)
#pragma unroll
    for (int mt = 0; mt < L::kRowTiles; ++mt)
#pragma unroll
      for (int nt = 0; nt < L::kColTiles; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          f(X[mt][nt][e], row0 + mt * 16 + quad + (e >> 1) * 8, col0 + nt * 8 + 2 * t + (e & 1));
  };
  {
    const int64_t head = (b * s.H + h) * (int64_t)a.p * a.r;
    const float* from = STATE || !a.from ? nullptr : a.from + head;
    int64_t ps = a.p_stride, rs = a.r_stride;
    if (!STATE && seg > 0) {
      from = g.state + ((pass * (int64_t)(g.count - 1) + seg - 1) * heads + b * s.H + h) * a.p * a.r;
      ps = a.r;
      rs = 1;
    }
    const bool first = !STATE && seg == 0 && !back;          // its own step of the decay
    if (first && marks && marks[0] != 0) from = nullptr;
    each([&](float& v, int p, int c) {
      const int r = slice * R + c;
      v = from && p < a.p && r < a.r ? from[p * ps + r * rs] : 0.f;
      if (first) v = l(v);
    });
  }
  const bool pairs_o = ((reinterpret_cast<uintptr_t>(a.out) & 7) == 0) && (a.r & 1) == 0;
  int run = 0;                          // STATE: the piece's decays, -1: a reset is in it

  // Where this lane reads y (and, across rows, y^T), z and the state for the products: the
  // first 16 rows, the first 16 columns; 16 columns on is an address with 1 << 5 exchanged.
  const uint32_t read_y = base + L::kY + piece<P>((mat >> 1) * 8 + mat_row, mat & 1);
  const uint32_t read_z = base + L::kZ + piece<R>((mat & 1) * 8 + mat_row, mat >> 1);
  const uint32_t read_state = base + L::kState + piece<R>((mat & 1) * 8 + mat_row, mat >> 1);
  // y and z by rows: a lane has 4 of every 32 columns; a pass of a warp takes 4 of its 16
  // rows (64 columns and more: two of them 4 apart, for the banks of the tiles)
  const int piece_of = lane & 7, sub = lane >> 3;
  auto first_row = [&](int W) { return warp * 16 + (W == 32 ? sub : (sub & 1) * 4 + (sub >> 1)); };
  auto next_row = [](int W, int k) { return W == 32 ? 4 * k : (k >> 1) * 8 + (k & 1) * 2; };
  auto row_of = [&](int W, int k) { return first_row(W) + next_row(W, k); };

  // the resets, read a chunk ahead (waited for at the chunk: 394 instead of 368 us forward over 16
  // x 8192 packed tokens of 4 heads of 64) where there are registers for them (four blocks of
  // 32 by 32: 205 us without any over 65536 positions of 8 heads, else 199)
  constexpr bool kMarksAhead = L::kBlocks < 4;
  uint32_t mark[3] = {0, 0, 0};
  auto read_marks = [&](int c) {
    const int t0 = start(c), n = min(kC, s.T - t0);
    mark[0] = lane < n ? __ldg(marks + t0 + lane) : 0;
    mark[1] = lane + 32 < n ? __ldg(marks + t0 + lane + 32) : 0;
    mark[2] = !back && t0 + n < s.T ? __ldg(marks + t0 + n) : 0;
  };
  if (kMarksAhead && marks) read_marks(c0);
  auto turn_over = [&](int c) {         // not AHEAD: this chunk's operands are done with
    if (AHEAD || c + 1 >= c1) return;
    wxx_tc::fence_proxy_async_smem();
    __syncthreads();
    fetch(c + 1);
  };
  for (int c = c0; c < c1; ++c) {
    const int t0 = start(c), n = min(kC, s.T - t0);
    // the resets of the chunk, and of the position after it
    unsigned long long cuts = 0;
    bool next = false;
    if (marks) {
      if (!kMarksAhead) read_marks(c);
      const unsigned lo = __ballot_sync(0xffffffffu, mark[0] != 0);
      const unsigned hi = __ballot_sync(0xffffffffu, mark[1] != 0);
      next = mark[2] != 0;
      cuts = (unsigned long long)hi << 32 | lo;
    }
    const Weights w(cuts, n, t0 + n < s.T, back ? cuts & 1 : next);
    bool odd = false;                   // a row that cannot be scaled
    {
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int mt = 0; mt < L::kRowTiles; ++mt)
#pragma unroll
        for (int nt = 0; nt < L::kColTiles; ++nt) {
          square2(s0, s1, X[mt][nt][0], X[mt][nt][1]);
          square2(s0, s1, X[mt][nt][2], X[mt][nt][3]);
        }
      s0 += s1;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
      if (!(s0 < kAbove * kAbove)) {
        odd = !(s0 < kLong);
        if (lane == 0) m.look = c;
      }
      if (s0 < kShort) {                // a state may be shorter than its square tells
        float top = 0.f;
        each([&](float v, int, int) { top = fmaxf(top, fabsf(v)); });
        s0 = -__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
      }
      if (lane == 0) m.square_state[warp] = s0;
    }
    if (tma)
      mbar_wait(&m.arrived, (c - c0) & 1, &m.abort, err);
    else
      copies_done();
    __syncthreads();       // the operands are here, the last chunk's tiles are read

    bool rare = false;                  // a row's square is out of range, or far from the middle
    float4 y[4][P / 32], z[4][R / 32];
    auto up_of = [](float square) { return square == 0.f ? 0.f : power2(kTop - exponent(square)); };
    float up_y[4], up_z[4];
    auto read = [&](auto width, int raw, auto& v, float* squares, float (&up)[4]) {
      constexpr int W = decltype(width)::value;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int from = (raw_piece(first_row(W), piece_of) * 16 ^ ((k & 1) << (W == 32 ? 6 : 5))) +
                         next_row(W, k) * 128;
#pragma unroll
        for (int i = 0; i < W / 32; ++i)
          v[k][i] = *reinterpret_cast<const float4*>(smem + raw + i * kRaw + from);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < W / 32; ++i) {
          square2(s0, s1, v[k][i].x, v[k][i].y);
          square2(s0, s1, v[k][i].z, v[k][i].w);
        }
        s0 += s1;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
        rare = rare || !(s0 >= kBelow && s0 < kAbove);
        up[k] = up_of(s0);
        if (piece_of == 0) squares[row_of(W, k)] = s0;
      }
    };
    read(std::integral_constant<int, P>{}, L::kRawY, y, m.square_y, up_y);
    read(std::integral_constant<int, R>{}, L::kRawZ, z, m.square_z, up_z);
    // x of this warp's positions, in the layout of a product's left operand (not AHEAD: read
    // again for the products, for the registers)
    float2 x[STATE ? 1 : P / 16][4];
    float square_x[2] = {0.f, 0.f};
    auto x_at = [&](int half, int k, int e) {
      return *reinterpret_cast<const float2*>(
          smem + L::kRawX + (k >> 1) * kRaw +
          ((raw_piece(warp * 16 + quad, t >> 1) * 16 + (t & 1) * 8) ^ ((4 * (k & 1) + 2 * e) << 4)) +
          half * 8 * 128);
    };
    if constexpr (!STATE) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int k = 0; k < P / 16; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 v = x_at(half, k, e);
            if (AHEAD) x[k][half + 2 * e] = v;
            square2(s0, s1, v.x, v.y);
          }
        s0 += s1;
        s0 += __shfl_xor_sync(0xffffffffu, s0, 1);
        s0 += __shfl_xor_sync(0xffffffffu, s0, 2);
        square_x[half] = s0;
        rare = rare || !(s0 >= kShort && s0 < kAbove);
      }
    }
    if (__any_sync(0xffffffffu, rare)) {       // rows of zeros are fine
      if (lane == 0) m.look = c;
      auto look = [&](const float* squares, int W, int row, float v0, float v1, float v2, float v3) {
        const float s0 = squares[row];
        odd = odd || !(s0 < kLong) ||
              (s0 < kShort && (v0 != 0.f || v1 != 0.f || v2 != 0.f || v3 != 0.f));
      };
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int i = 0; i < P / 32; ++i)
          look(m.square_y, P, row_of(P, k), y[k][i].x, y[k][i].y, y[k][i].z, y[k][i].w);
#pragma unroll
        for (int i = 0; i < R / 32; ++i)
          look(m.square_z, R, row_of(R, k), z[k][i].x, z[k][i].y, z[k][i].z, z[k][i].w);
      }
      if constexpr (!STATE) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int k = 0; k < P / 16; ++k) {
            const float2 u = AHEAD ? x[k][half] : x_at(half, k, 0);
            const float2 v = AHEAD ? x[k][half + 2] : x_at(half, k, 1);
            look(square_x, 1, half, u.x, u.y, v.x, v.y);
          }
      }
    }
    odd = __syncthreads_or(odd);        // the squares are here, the operands are read
    if (AHEAD && c + 1 < c1) fetch(c + 1);
    if (kMarksAhead && marks && c + 1 < c1) read_marks(c + 1);
    const int kept_power = w.kept(back);
    const float2 kept = kept_power < 0 ? make_float2(0.f, 0.f) : m.kept[kept_power];
    if (STATE) run = run < 0 || kept_power < 0 ? -1 : run + kept_power;
    const float4 parts = *reinterpret_cast<const float4*>(m.square_state);
    const float square_state = (fmaxf(parts.x, 0.f) + fmaxf(parts.y, 0.f)) +
                               (fmaxf(parts.z, 0.f) + fmaxf(parts.w, 0.f));
    int e_state = exponent(square_state);
    if (square_state == 0.f) {
      const float top = -fminf(fminf(parts.x, parts.y), fminf(parts.z, parts.w));
      e_state = top > 0.f ? max((int)(__float_as_uint(top) >> 23) - 127 + 6, kTop - 127) : kNoState;
    }
    if (m.look == c)
      odd = odd || m.power[kC] < 0x1p-126f || (!STATE && far_apart(m.square_y, m.square_z));
    if (odd) {
      float* state = reinterpret_cast<float*>(smem + L::kTiles);
      unsigned char* cut = smem + L::kTiles + (P * R + kThreads) * 4;
      if (threadIdx.x < kC) cut[threadIdx.x] = cuts >> threadIdx.x & 1;
      each([&](float v, int p, int c) { state[p * R + c] = v; });
      __syncthreads();
      rare_chunk<R, STATE>(state, state + P * R, cut, a, s, n, w.tail, next, l, b, h, t0, slice);
      __syncthreads();
      each([&](float& v, int p, int c) { v = state[p * R + c]; });
      turn_over(c);
      continue;
    }

    // what the rows weigh: lane looks at rows lane and lane + 32
    int most = -1000, most_added = -1000;
    int e_row[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = lane + 32 * k;
      const float sy = m.square_y[j], sz = m.square_z[j];
      e_row[k] = exponent(sy) + exponent(sz);
      if (sy == 0.f || sz == 0.f) e_row[k] = -1000;         // nothing there
      const Decayed u(m.power, w.added(j, back));
      most = max(most, e_row[k]);
      e_row[k] = u.any ? e_row[k] + u.e : -1000;
      most_added = max(most_added, e_row[k]);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    most_added = __reduce_max_sync(0xffffffffu, most_added);
    // a weight in the state that one half number does not hold
    const bool far = __any_sync(0xffffffffu, (e_row[0] > -500 && e_row[0] - most_added < -24) ||
                                                 (e_row[1] > -500 && e_row[1] - most_added < -24));
    if (most < -500) most = 0;
    if (most_added < -500) most_added = 0;
    if (threadIdx.x < kC) {
      // the power of two of l^u goes into the weight, the rest into z's scale
      const int j = threadIdx.x;
      const float sy = m.square_y[j], sz = m.square_z[j];
      const bool any = sy != 0.f && sz != 0.f;
      const int e = exponent(sy) + exponent(sz);
      const Decayed u(m.power, w.added(j, back));
      const float one = !any ? 0.f : __fdividef(a.y_unit * power2(e - most), u.rest);
      m.weight[j] = make_float2(one, one * m.power[back ? j & 15 : 15 - (j & 15)]);
      const int below = any && u.any ? e + u.e - most_added : -1000;
      // 2^below as two halves, each 2^-24 at least (0: less than 2^-38 of the largest)
      const int first = max(below, -24), then = max(below - first, -24);
      m.added[0][j] = below < -38 ? 0 : __half_as_ushort(__float2half_rn(power2(first)));
      m.added[1][j] = __half_as_ushort(__float2half_rn(power2(then)));
      m.document[j] = w.document(j);
    }
    // the tiles: y, and the state (z waits for its scales)
    auto tile = [&](auto width, int to, const auto& v, const float (&ups)[4]) {
      constexpr int W = decltype(width)::value;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float up = ups[k];
#pragma unroll
        for (int i = 0; i < W / 32; ++i) {
          uint2 hi, lo;
          split(v[k][i].x, v[k][i].y, up, hi.x, lo.x);
          split(v[k][i].z, v[k][i].w, up, hi.y, lo.y);
          unsigned char* p = smem + to + next_row(W, k) * W * 2 +
                             ((piece<W>(first_row(W), piece_of >> 1) + (piece_of & 1) * 8) ^
                              ((k & 1) << 5) ^ (i << 6));
          *reinterpret_cast<uint2*>(p) = hi;
          *reinterpret_cast<uint2*>(p + kC * W * 2) = lo;
        }
      }
    };
    tile(std::integral_constant<int, P>{}, L::kY, y, up_y);
    if constexpr (!STATE) {
      if (e_state != kNoState) {
        const float up = power2(kTop - e_state);
#pragma unroll
        for (int mt = 0; mt < L::kRowTiles; ++mt)
#pragma unroll
          for (int nt = 0; nt < L::kColTiles; nt += 2) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              split(X[mt][nt + (e >> 1)][(e & 1) * 2], X[mt][nt + (e >> 1)][(e & 1) * 2 + 1], up, hi[e],
                    lo[e]);
            const uint32_t to = (read_state ^ ((col0 / 16 + nt / 2) << 5)) + (row0 + mt * 16) * R * 2;
            store4<0>(to, hi[0], hi[1], hi[2], hi[3]);
            store4<P * R * 2>(to, lo[0], lo[1], lo[2], lo[3]);
          }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) up_z[k] *= Decayed(m.power, w.added(row_of(R, k), back)).rest;
    tile(std::integral_constant<int, R>{}, L::kZ, z, up_z);
    __syncthreads();

    if constexpr (!STATE) {
      int e_x[2];
      uint32_t xh[P / 16][4], xl[P / 16][4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        e_x[half] = square_x[half] == 0.f ? 0 : exponent(square_x[half]);
        const float up = power2(kTop - e_x[half]);
#pragma unroll
        for (int k = 0; k < P / 16; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 v = AHEAD ? x[k][half + 2 * e] : x_at(half, k, e);
            split(v.x, v.y, up, xh[k][half + 2 * e], xl[k][half + 2 * e]);
          }
      }
      // x y^T for the positions up to (back: from) this warp's own
      float S[kC / 8][4];
      for_each<kC / 16>([&](auto block) {
        constexpr int jb = decltype(block)::value;
        if (back ? jb < warp : jb > warp) return;
        float small[2][4];                // the products with low halves
#pragma unroll
        for (int e = 0; e < 4; ++e)
          S[2 * jb][e] = S[2 * jb + 1][e] = small[0][e] = small[1][e] = 0.f;
#pragma unroll
        for (int k = 0; k < P / 16; ++k) {
          uint32_t bh[4], bl[4];
          load4<jb * 16 * P * 2>(bh, read_y ^ (k << 5));
          load4<jb * 16 * P * 2 + kC * P * 2>(bl, read_y ^ (k << 5));
          product(small[0], xl[k], bh[0], bh[1]);
          product(small[1], xl[k], bh[2], bh[3]);
          product(S[2 * jb], xh[k], bh[0], bh[1]);
          product(S[2 * jb + 1], xh[k], bh[2], bh[3]);
          product(small[0], xh[k], bl[0], bl[1]);
          product(small[1], xh[k], bl[2], bl[3]);
        }
#pragma unroll
        for (int jt = 0; jt < 2; ++jt) {
          float(&v)[4] = S[2 * jb + jt];
          add2(v[0], v[1], v[0], v[1], small[jt][0], small[jt][1]);
          add2(v[2], v[3], v[2], v[3], small[jt][2], small[jt][3]);
        }
      });
      // x X.  A sum in a product loses up to an ulp each time (it is cut off, not rounded), so 128
      // channels take all the small products first, while the sum is small: error 9.5e-7 ->
      // 7.2e-7, 164 -> 170 us over 8 x 1024 tokens of 8 heads of 128.  In place it is also
      // faster (193 -> 188 us backward over 8 x 1024 tokens of 16 heads of 64), ahead, whose
      // error is 7.4e-7 at 64 channels, slower (261 -> 268 forward over 37 x 1024).
      constexpr bool kSmallFirst = P == 128 || !AHEAD;
      float o[R / 8][4];
#pragma unroll
      for (int nt = 0; nt < R / 8; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][e] = 0.f;
      if (e_state != kNoState) {
        for_each<P / 16>([&](auto depth) {
          constexpr int k = decltype(depth)::value;
#pragma unroll
          for (int nb = 0; nb < R / 16; ++nb) {
            uint32_t bh[4], bl[4];
            load4_turned<k * 16 * R * 2>(bh, read_state ^ (nb << 5));
            load4_turned<k * 16 * R * 2 + P * R * 2>(bl, read_state ^ (nb << 5));
            if constexpr (kSmallFirst) {
              product(o[2 * nb], xl[k], bh[0], bh[1]);
              product(o[2 * nb + 1], xl[k], bh[2], bh[3]);
              product(o[2 * nb], xh[k], bl[0], bl[1]);
              product(o[2 * nb + 1], xh[k], bl[2], bl[3]);
            } else {
              products(o[2 * nb], o[2 * nb + 1], xh[k], xl[k], bh, bl);
            }
          }
        });
        for_each<kSmallFirst ? P / 16 : 0>([&](auto depth) {
          constexpr int k = decltype(depth)::value;
#pragma unroll
          for (int nb = 0; nb < R / 16; ++nb) {
            uint32_t bh[4];
            load4_turned<k * 16 * R * 2>(bh, read_state ^ (nb << 5));
            product(o[2 * nb], xh[k], bh[0], bh[1]);
            product(o[2 * nb + 1], xh[k], bh[2], bh[3]);
          }
        });
      }
      // The weights of x y^T, and the rows' largest: l^(i - j) is looked up in the warp's
      // own positions, elsewhere it is a product of three powers of at least 0.
      float most_p[2] = {0.f, 0.f};
#pragma unroll
      for (int jb = 0; jb < kC / 16; ++jb) {
        if (back ? jb < warp : jb > warp) continue;
        const float gap = jb == warp ? 1.f : m.power[16 * abs(warp - jb) - 15];
        const float side[2] = {gap * m.power[back ? 15 - quad : quad],
                               gap * m.power[back ? 7 - quad : quad + 8]};
#pragma unroll
        for (int jt = 0; jt < 2; ++jt) {
          float(&v)[4] = S[2 * jb + jt];
          const int j = jb * 16 + jt * 8 + 2 * t;
          const float4 f = *reinterpret_cast<const float4*>(&m.weight[j]);
          if (jb == warp) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = quad + (e >> 1) * 8, k = jt * 8 + 2 * t + (e & 1);
              const int apart = back ? k - i : i - k;
              v[e] = apart < 0 ? 0.f : v[e] * (m.power[max(apart, 0)] * (e & 1 ? f.z : f.x));
            }
          } else {
            mul2(v[0], v[1], v[0], v[1], f.y, f.w);
            mul2(v[2], v[3], v[2], v[3], f.y, f.w);
            mul2(v[0], v[1], v[0], v[1], side[0], side[0]);
            mul2(v[2], v[3], v[2], v[3], side[1], side[1]);
          }
        }
      }
      if (w.inner) {
#pragma unroll
        for (int jt = 0; jt < kC / 8; ++jt) {
          if (back ? jt / 2 < warp : jt / 2 > warp) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (m.document[warp * 16 + quad + (e >> 1) * 8] != m.document[jt * 8 + 2 * t + (e & 1)])
              S[jt][e] = 0.f;
        }
      }
#pragma unroll
      for (int jt = 0; jt < kC / 8; ++jt) {
        if (back ? jt / 2 < warp : jt / 2 > warp) continue;
        most_p[0] = fmax3(most_p[0], fabsf(S[jt][0]), fabsf(S[jt][1]));
        most_p[1] = fmax3(most_p[1], fabsf(S[jt][2]), fabsf(S[jt][3]));
      }
      // Both sums in one scale: the larger's, whichever part it comes from.
      float up[2];
      float by[2], then[2];
      const int unit = most + a.y_exp;
      const int apart = e_state + 2 * kTop - unit;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = warp * 16 + quad + half * 8;
        most_p[half] = fmaxf(most_p[half], __shfl_xor_sync(0xffffffffu, most_p[half], 1));
        most_p[half] = fmaxf(most_p[half], __shfl_xor_sync(0xffffffffu, most_p[half], 2));
        int e_p = max((int)(__float_as_uint(most_p[half]) >> 23) - 127, -110);
        const Decayed u(m.power, w.reach(i, back));
        if (e_state != kNoState) {
          if (u.any) e_p = max(e_p, apart + u.e - kTop);
          const int e_in = u.e + apart - e_p;
          const float in = !u.any || e_in < -126 ? 0.f : u.rest * power2(e_in);
#pragma unroll
          for (int nt = 0; nt < R / 8; ++nt)
            mul2(o[nt][2 * half], o[nt][2 * half + 1], o[nt][2 * half], o[nt][2 * half + 1], in, in);
        }
        up[half] = kTop - e_p < -126 ? 0.f : power2(kTop - e_p);
        const Scale scale(a.out_unit, e_p + e_x[half] + unit + a.out_exp - 4 * kTop);
        by[half] = scale.first;
        then[half] = scale.then;
      }
      for_each<kC / 16>([&](auto block) {
        constexpr int jb = decltype(block)::value;
        if (back ? jb < warp : jb > warp) return;
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          split(S[2 * jb + (e >> 1)][(e & 1) * 2], S[2 * jb + (e >> 1)][(e & 1) * 2 + 1], up[e & 1],
                ph[e], pl[e]);
#pragma unroll
        for (int nb = 0; nb < R / 16; ++nb) {
          uint32_t bh[4], bl[4];
          load4_turned<jb * 16 * R * 2>(bh, read_z ^ (nb << 5));
          load4_turned<jb * 16 * R * 2 + kC * R * 2>(bl, read_z ^ (nb << 5));
          products(o[2 * nb], o[2 * nb + 1], ph, pl, bh, bl);
        }
      });
      const int room = a.r - slice * R;
      const bool plain = pairs_o && n == kC && room >= R;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int nt = 0; nt < R / 8; ++nt)
          mul2(o[nt][half * 2], o[nt][half * 2 + 1], o[nt][half * 2], o[nt][half * 2 + 1], by[half],
               by[half]);
      if (__any_sync(0xffffffffu, then[0] != 1.f || then[1] != 1.f)) {
#pragma unroll
        for (int nt = 0; nt < R / 8; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][e] *= then[e >> 1];
      }
      float* out = a.out + ((b * s.T + t0 + warp * 16 + quad) * s.H + h) * a.r + slice * R + 2 * t;
      const int64_t eight = (int64_t)8 * s.H * a.r;
      if (plain) {
#pragma unroll
        for (int nt = 0; nt < R / 8; ++nt) {
          *reinterpret_cast<float2*>(out + nt * 8) = make_float2(o[nt][0], o[nt][1]);
          *reinterpret_cast<float2*>(out + eight + nt * 8) = make_float2(o[nt][2], o[nt][3]);
        }
      } else {
#pragma unroll
        for (int nt = 0; nt < R / 8; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (warp * 16 + quad + (e >> 1) * 8 < n && nt * 8 + 2 * t + (e & 1) < room)
              out[(e >> 1) * eight + nt * 8 + (e & 1)] = o[nt][e];
      }
    }
    // the state: what the chunk adds, then in 32 bits
    const Scale by(a.y_unit, most_added + a.y_exp - 2 * kTop);
#pragma unroll
    for (int mt = 0; mt < L::kRowTiles; ++mt) {
      float d[L::kColTiles][4];
#pragma unroll
      for (int nt = 0; nt < L::kColTiles; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) d[nt][e] = 0.f;
      for_each<kC / 16>([&](auto depth) {
        constexpr int k = decltype(depth)::value;
        uint32_t ah[4], al[4];
        const uint32_t from = read_y ^ ((row0 / 16 + mt) << 5);
        load4_turned<k * 16 * P * 2>(ah, from);
        load4_turned<k * 16 * P * 2 + kC * P * 2>(al, from);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int j = k * 16 + half * 8 + 2 * t;
          const uint32_t f = *reinterpret_cast<const uint32_t*>(&m.added[0][j]);
#pragma unroll
          for (int e = 2 * half; e < 2 * half + 2; ++e) {
            ah[e] = times(ah[e], f);
            al[e] = times(al[e], f);
          }
          if (far) {
            const uint32_t f2 = *reinterpret_cast<const uint32_t*>(&m.added[1][j]);
#pragma unroll
            for (int e = 2 * half; e < 2 * half + 2; ++e) {
              ah[e] = times(ah[e], f2);
              al[e] = times(al[e], f2);
            }
          }
        }
#pragma unroll
        for (int nb = 0; nb < L::kColTiles / 2; ++nb) {
          uint32_t bh[4], bl[4];
          const uint32_t zat = read_z ^ ((col0 / 16 + nb) << 5);
          load4_turned<k * 16 * R * 2>(bh, zat);
          load4_turned<k * 16 * R * 2 + kC * R * 2>(bl, zat);
          products(d[2 * nb], d[2 * nb + 1], ah, al, bh, bl);
        }
      });
      if (by.then != 1.f) {
#pragma unroll
        for (int nt = 0; nt < L::kColTiles; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[nt][e] *= by.then;
      }
#pragma unroll
      for (int nt = 0; nt < L::kColTiles; ++nt)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          float(&v)[4] = X[mt][nt];
          float t0, t1;
          mul2(t0, t1, v[e], v[e + 1], kept.x, kept.x);
          fma2(t0, t1, d[nt][e], d[nt][e + 1], by.first, by.first, t0, t1);
          fma2(v[e], v[e + 1], v[e], v[e + 1], kept.y, kept.y, t0, t1);
        }
    }
    turn_over(c);
  }

  if (STATE || (a.last && seg == pieces - 1)) {
    float* to = STATE ? g.state + ((pass * (int64_t)pieces + seg) * heads + b * s.H + h) * a.p * a.r
                      : a.last + (b * s.H + h) * (int64_t)a.p * a.r;
    const int64_t ps = STATE ? a.r : a.p_stride, rs = STATE ? 1 : a.r_stride;
    each([&](float v, int p, int c) {
      const int r = slice * R + c;
      if (p < a.p && r < a.r) to[p * ps + r * rs] = v;
    });
  }
  if (STATE && threadIdx.x == 0) {
    const float run_log = (float)run * s.log_decay[h];
    g.kept[(pass * (int64_t)pieces + seg) * heads + b * s.H + h] =
        run < 0                      ? make_float2(0.f, -1.f)
        : whole_of(run_log) != 0.f ? make_float2(expm1f(run_log), 1.f)
                                     : make_float2(expf(0.5f * run_log), 0.f);
  }
}

// The states before the pieces, from what each piece adds to a state and keeps of it, in
// place: a thread an entry, one piece after the other.  Only a reset ends a NaN or an infinity,
// however little the decays leave of a number.
__global__ void __launch_bounds__(kT)
    join_kernel(const __grid_constant__ Passes passes, const Shape s, const Segments g,
                const int64_t heads, const int64_t total) {
  const int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x;
  if (i >= total) return;
  const int pass = blockIdx.y;
  const Pass& a = passes.at[pass];
  const int64_t size = (int64_t)a.p * a.r, head = i / size;
  const int p = (int)(i % size) / a.r, r = (int)(i % size) % a.r;
  const int64_t b = head / s.H;
  float X = a.from ? a.from[head * size + p * a.p_stride + r * a.r_stride] : 0.f;
  const Decay l(s.log_decay[head % s.H]);
  if (!a.back) X = s.reset && s.reset[b * s.T] != 0 ? 0.f : l(X);
  float* E = g.state + pass * (int64_t)(g.count - 1) * total + i;
  const float2* kept = g.kept + pass * (int64_t)(g.count - 1) * heads + head;
  // a piece's numbers are read before the one before it is written
  float own = *E;
  float2 left = __ldg(kept);
  for (int k = 0; k < g.count - 1; ++k) {
    const bool more = k + 1 < g.count - 1;
    const float next = more ? E[total] : 0.f;
    const float2 next_left = more ? __ldg(kept + heads) : left;
    X = left.y < 0.f             ? own
        : !(fabsf(X) < INFINITY) ? l(X) + own
        : left.y > 0.f           ? X + fmaf(left.x, X, own)
                                 : fmaf(left.x * X, left.x, own);
    *E = X;
    own = next, left = next_left;
    E += total, kept += heads;
  }
}

// One position a sequence: a block per sequence, head and 16 V columns of the state, V columns
// a thread (16 threads a row) and every 16th row.  Bound by the state's read and write; a
// thread's loads of up to 4 rows are under way together.
template <int V>
__global__ void __launch_bounds__(kT)
    step_kernel(float* __restrict__ o, float* __restrict__ state, const float* __restrict__ q,
                int64_t q_ld, const float* __restrict__ k, int64_t k_ld,
                const float* __restrict__ v, int64_t v_ld, const float* __restrict__ log_decay,
                int H, int dk, int dv, float scale) {
  constexpr int kRows = 16, kAhead = 4;
  __shared__ float part[kT / 32][16 * V];
  const int slices = (dv + 16 * V - 1) / (16 * V);
  const int slice = blockIdx.x % slices, h = blockIdx.x / slices % H;
  const int64_t b = blockIdx.x / slices / H;
  const int row = threadIdx.x / 16, c = slice * 16 * V + threadIdx.x % 16 * V;
  float* S = state + (b * H + h) * dk * dv + c;
  const float *qh = q + b * q_ld + h * dk, *kh = k + b * k_ld + h * dk;
  const bool in = c < dv;
  float z[V], sum[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sum[e] = 0.f;
  for (int p0 = row; p0 < dk; p0 += kRows * kAhead) {
    float now[kAhead][V], x[kAhead], y[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int p = p0 + i * kRows;
      const bool here = in && p < dk;
      x[i] = here ? qh[p] : 0.f;
      y[i] = here ? kh[p] : 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) now[i][e] = 0.f;
      if (!here) continue;
      if constexpr (V == 4) {
        const float4 t = *reinterpret_cast<const float4*>(S + (int64_t)p * dv);
        now[i][0] = t.x, now[i][1] = t.y, now[i][2] = t.z, now[i][3] = t.w;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) now[i][e] = S[(int64_t)p * dv + e];
      }
    }
    if (p0 == row) {
#pragma unroll
      for (int e = 0; e < V; ++e) z[e] = in ? v[b * v_ld + h * dv + c + e] : 0.f;
    }
    const Decay l(log_decay[h]);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int p = p0 + i * kRows;
      if (!in || p >= dk) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        now[i][e] = fmaf(y[i], z[e], l(now[i][e]));
        sum[e] = fmaf(x[i], now[i][e], sum[e]);
      }
      if constexpr (V == 4) {
        *reinterpret_cast<float4*>(S + (int64_t)p * dv) =
            make_float4(now[i][0], now[i][1], now[i][2], now[i][3]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) S[(int64_t)p * dv + e] = now[i][e];
      }
    }
  }
  // over a warp's two rows, then over the warps
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 16);
    if ((threadIdx.x & 16) == 0) part[warp][threadIdx.x % 16 * V + e] = sum[e];
  }
  __syncthreads();
  const int r = slice * 16 * V + threadIdx.x;
  if (threadIdx.x < 16 * V && r < dv) {
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < kT / 32; ++w) all += part[w][threadIdx.x];
    o[(b * H + h) * dv + r] = scale * all;
  }
}

int check_sizes(const char* what, int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv) {
  WXX_REQUIRE(B >= 0 && T >= 0 && H >= 0 && dk >= 0 && dv >= 0, "%s: negative size", what);
  WXX_REQUIRE(dk <= 256 && dv <= 256, "%s: heads of %lld and %lld channels (256 at most)", what,
              (long long)dk, (long long)dv);
  WXX_REQUIRE(T < (int64_t(1) << 31) - 256 && H < (int64_t(1) << 22) &&
                  B * H * 16 < (int64_t(1) << 31),
              "%s: too many positions, sequences or heads", what);
  return WXX_OK;
}

int sweep(const Pass& a, const Shape& s, int64_t B) {
  sweep_kernel<<<(unsigned)(B * s.H * ((a.r + 31) / 32)), kT, 0, wxx::stream()>>>(a, s);
  return wxx::after_launch(__FILE__, __LINE__);
}

// Room for a kernel's tiles, asked for once for each.
template <class K>
int allow_smem(K kernel, int bytes) {
  static std::mutex lock;
  static K done[16] = {};           // kernels of this type that have it
  std::lock_guard<std::mutex> hold(lock);
  for (K& k : done) {
    if (k == kernel) return WXX_OK;
    if (k) continue;
    WXX_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    k = kernel;
    return WXX_OK;
  }
  WXX_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return WXX_OK;
}

// How many pieces a row of `chunks` is worked on in, for `rows` rows (sequences, heads, slices
// and passes), and whether with the next chunk's operands ahead, `blocks` blocks on an SM, or
// in place, `more` of them: the least of the outputs' launch and, with more than one piece, the
// states' one (half as long a chunk) and what lies between.  In units of a full SM's time for
// one block's chunk; a start is about a chunk.  Measured, heads of 64, 16 chunks a row, 1, 2 and
// 3 blocks on every SM: ahead 106 and 135 us (and 247: two turns), in place 129, 172 and 188; so
// 384 rows take 243 and 180 us, 592 rows 261 and 369.  In 1 and 2 pieces 128 rows of 16 chunks
// 108 and 116 us; with two of the states' blocks on an SM 64 of 128 chunks in 3, 4 and 8 pieces 463,
// 377 and 380, 16 of 128 in 8, 16 and 32 pieces 175, 123 and 135.
struct Plan {
  int pieces;
  bool ahead;
};
Plan plan_of(int64_t rows, int64_t chunks, int blocks, int more, int of_states) {
  const int64_t sms = wxx::num_sms();
  // n blocks, `fit` on an SM at a time: a full SM takes `full`, a block by itself `alone`
  auto turns = [&](int64_t n, int fit, double alone, double full) {
    const int64_t times = n / (sms * fit), rest = (n - times * sms * fit + sms - 1) / sms;
    const double last = rest == 0   ? 0.
                        : fit == 1 ? full
                                   : alone + (full - alone) * (double)(rest - 1) / (fit - 1);
    return times * full + last;
  };
  auto ahead = [&](int64_t n) { return turns(n, blocks, 0.8 * blocks, blocks); };
  double least = 0;
  Plan best{1, true};
  for (int m = 1; m <= 128 && 2 * m <= chunks + 1; ++m) {
    const int64_t size = (chunks + m - 1) / m;
    if ((chunks + size - 1) / size != m) continue;
    const double states = m > 1 ? turns(rows * (m - 1), of_states, 0.8 * blocks, of_states) * (0.5 * size + 1) + 2.5 : 0.;
    const double a = states + ahead(rows * m) * (size + 1);
    if (m == 1 || a < least) least = a, best = {m, true};
    if (more == blocks) continue;
    const double i = states + turns(rows * m, more, 0.95 * blocks, 0.97 * more) * (size + 1);
    if (i < least) least = i, best = {m, false};
  }
  return best;
}

PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    cudaGetLastError();
  });
  return fn;
}

// A map of boxes of 32 channels of a head by 64 positions, where the copy engine takes the
// operand: a 16-byte aligned base and strides.
bool encode(CUtensorMap* map, const Operand& o, int64_t B, int64_t T, int64_t H, int64_t width) {
  auto enc = get_encode();
  const int64_t bs = B > 1 ? o.bs : T * o.ts;
  if (!enc || (reinterpret_cast<uintptr_t>(o.p) & 15) || (o.ts | bs | width) & 3 || o.ts <= 0 ||
      bs <= 0 || o.ts >= (int64_t(1) << 37) || bs >= (int64_t(1) << 37))
    return false;
  cuuint64_t dims[4] = {(cuuint64_t)width, (cuuint64_t)H, (cuuint64_t)T, (cuuint64_t)B};
  cuuint64_t strides[3] = {(cuuint64_t)width * 4, (cuuint64_t)o.ts * 4, (cuuint64_t)bs * 4};
  cuuint32_t box[4] = {32, 1, kC, 1}, ones[4] = {1, 1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, const_cast<float*>(o.p), dims, strides, box,
             ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// n passes of one padded size in one launch, the rows in pieces where there are too few
// sequences and heads to fill the SMs: first what every piece but the last adds to a state,
// then the states before the pieces, then the outputs.
template <int P, int R>
int chunked(const Passes& passes, int n, const Shape& s, int64_t B) {
  using L = Layout<P, R, false, true>;
  using States = Layout<P, R, true, true>;
  using InPlace = Layout<P, R, false, P != 64 || R != 64>;     // (other sizes: measured no faster)
  const Pass& a = passes.at[0];
  const int slices = (a.r + R - 1) / R;
  const int64_t heads = B * s.H, blocks = heads * slices, chunks = (s.T + kC - 1) / kC;
  const Plan plan = plan_of(blocks * n, chunks, L::kBlocks, InPlace::kBlocks, States::kBlocks);
  Segments g{plan.pieces, 0, nullptr, nullptr};
  g.chunks = (int)((chunks + g.count - 1) / g.count);
  WXX_REQUIRE(blocks * n * g.count < (int64_t(1) << 31), "linear attention: too many sequences");
  Maps maps{};
  bool tma = true;
  for (int i = 0; i < n; ++i) {
    const Pass& p = passes.at[i];
    tma = tma && encode(&maps.x[i], p.x, B, s.T, s.H, p.p) &&
          encode(&maps.y[i], p.y, B, s.T, s.H, p.p) && encode(&maps.z[i], p.z, B, s.T, s.H, p.r);
  }
  constexpr bool kIn = InPlace::kBlocks == L::kBlocks;  // there is no such kernel
  auto kernel = plan.ahead ? chunk_kernel<P, R, false, true> : chunk_kernel<P, R, false, kIn>;
  const int bytes = plan.ahead ? L::kBytes : InPlace::kBytes;
  if (int st = allow_smem(chunk_kernel<P, R, true, true>, States::kBytes)) return st;
  if (int st = allow_smem(kernel, bytes)) return st;
  int* err = wxx::device_error_word();
  void* scratch = nullptr;
  if (g.count > 1) {
    const int64_t states = n * (g.count - 1) * heads;
    if (int st = wxx_malloc(&scratch, (uint64_t)(states * (a.p * a.r + 2)) * sizeof(float)))
      return st;
    g.kept = static_cast<float2*>(scratch);
    g.state = reinterpret_cast<float*>(g.kept + states);
    const unsigned per = (unsigned)(blocks * (g.count - 1));
    chunk_kernel<P, R, true, true><<<per * n, kThreads, States::kBytes, wxx::stream()>>>(passes, maps, tma, s, g,
                                                                            per, err);
    int st = wxx::after_launch(__FILE__, __LINE__);
    if (st == WXX_OK) {
      const int64_t total = heads * a.p * a.r;
      join_kernel<<<dim3((unsigned)((total + kT - 1) / kT), n), kT, 0, wxx::stream()>>>(
          passes, s, g, heads, total);
      st = wxx::after_launch(__FILE__, __LINE__);
    }
    if (st != WXX_OK) {
      wxx_free(scratch);
      return st;
    }
  }
  const unsigned per = (unsigned)(blocks * g.count);
  kernel<<<per * n, kThreads, bytes, wxx::stream()>>>(passes, maps, tma, s, g,
                                                                           per, err);
  const int st = wxx::after_launch(__FILE__, __LINE__);
  if (scratch) wxx_free(scratch);
  return st;
}

int padded(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// Passes of the same sizes side by side.
int run_passes(const Pass* a, int n, const Shape& s, int64_t B) {
  for (int i = 0; i < n;) {
    const int P = padded(a[i].p), R = a[i].r <= 32 ? 32 : 64;
    Passes same;
    int k = 0;
    for (; i < n && k < 3; ++i, ++k) {
      if (padded(a[i].p) != P || (a[i].r <= 32 ? 32 : 64) != R ||
          (a[i].r + 63) / 64 != (a[i - k].r + 63) / 64)
        break;
      same.at[k] = a[i];
      same.at[k].y_unit = unit_of(a[i].y_scale, same.at[k].y_exp);
      same.at[k].out_unit = unit_of(a[i].out_scale, same.at[k].out_exp);
    }
    int st;
    if (P == 256) {
      st = WXX_OK;
      for (int j = 0; j < k && st == WXX_OK; ++j) st = sweep(same.at[j], s, B);
    } else if (R == 32) {
      st = P == 32 ? chunked<32, 32>(same, k, s, B) : P == 64 ? chunked<64, 32>(same, k, s, B)
                                                              : chunked<128, 32>(same, k, s, B);
    } else {
      st = P == 32 ? chunked<32, 64>(same, k, s, B) : P == 64 ? chunked<64, 64>(same, k, s, B)
                                                              : chunked<128, 64>(same, k, s, B);
    }
    if (st != WXX_OK) return st;
  }
  return WXX_OK;
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
  return run_passes(&a, 1, s, B);
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
  return run_passes(passes, 3, s, B);
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
  const bool fours = dv % 4 == 0 && (reinterpret_cast<uintptr_t>(state) & 15) == 0;
  auto kernel = fours ? step_kernel<4> : step_kernel<1>;
  const int64_t wide = fours ? 64 : 16;
  kernel<<<(unsigned)(B * H * ((dv + wide - 1) / wide)), kT, 0, wxx::stream()>>>(
      o, state, q, q_ld, k, k_ld, v, v_ld, log_decay, (int)H, (int)dk, (int)dv, scale);
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}
