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
#include <mutex>
#include <type_traits>

#include "common.cuh"

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
};

struct Shape {
  const float* log_decay;   // (H)
  const uint32_t* reset;    // (B, T) or NULL
  int T, H;
};

constexpr int kT = 256;

// One position's decay of a state, l X.  A decay near 1 is applied as X + (l - 1) X: l alone
// is rounded to 2^-25, which n positions in a row make n 2^-25.
// (An infinite state takes l itself: of the two terms' signs one is the other's opposite.)
struct Decay {
  float l, less, whole;
  __device__ explicit Decay(float log_decay)
      : l(expf(log_decay)), less(log_decay > -0.5f ? expm1f(log_decay) : l),
        whole(log_decay > -0.5f ? 1.f : 0.f) {}
  __device__ __forceinline__ float operator()(float X) const {
    return fabsf(X) < INFINITY ? fmaf(less, X, whole * X) : l * X;
  }
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
// position-by-position matrix) is scaled by a power of two that brings its largest entry
// to 2^13, and a state by one for all of it; the powers are put back in 32 bits.  Entries
// far below their row's largest lose accuracy from 2^-20 of it on (they are good to 2^-38
// of the largest).  (Measured, mma.sync: half 554, tf32 277 TFLOP/s; three products of
// tf32 need no scaling, but would be bound by that rate.)  The state stays in 32-bit
// registers, a chunk's products are added to it in 32 bits.
//
// NaN and infinities cannot take part: 0 times NaN would carry them to earlier positions
// and other documents.  A chunk that holds one, or starts from a state that does, is
// worked through position by position (rare_chunk).

constexpr int kC = 64;                  // positions of a chunk
constexpr int kThreads = 256;           // 8 warps: 4 groups of 16 positions by 2 halves
constexpr int kTop = 13;                // a scaled row's largest entry is in [2^13, 2^14)

__device__ __forceinline__ uint32_t smem_address(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void copy16(uint32_t to, const float* from, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from),
               "r"(take ? 16 : 0));
}
__device__ __forceinline__ void copy4(uint32_t to, const float* from, bool take) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from),
               "r"(take ? 4 : 0));
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void pair_barrier(int group) {      // the two warps of a group
  asm volatile("bar.sync %0, 64;" ::"r"(group + 1) : "memory");
}

__device__ __forceinline__ void load4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void load4_turned(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
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

// The high and low halves of two numbers.
__device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {      // two halves each
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// The exponent of a row's largest entry; rows below 2^-100 are scaled as if at 2^-100.
__device__ __forceinline__ int exponent(float size) {
  return max((int)(__float_as_uint(size) >> 23) - 127, -100);
}
__device__ __forceinline__ float power2(int e) {            // -126 <= e <= 127
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// v -> v f 2^e for any e, f about 1: in two steps of one sign, so that nothing is lost on
// the way.
struct Scale {
  float first, then;
  __device__ Scale(float f, int e) {
    e = min(max(e, -250), 250);
    first = f * power2(e / 2);
    then = power2(e - e / 2);
  }
  __device__ __forceinline__ float operator()(float v) const { return v * first * then; }
};

// Tiles of W half numbers a row for ldmatrix: 16-byte pieces of a row exchanged so that
// the same piece of 8 rows lies in 8 different sets of banks.
template <int W>
__device__ __forceinline__ uint32_t piece(int row, int q) {
  const int turn = W == 32 ? (row >> 1) & 3 : row & 7;
  return (uint32_t)(row * W * 2 + ((q ^ turn) << 4));
}
// Rows of W floats as copied: the even 16-byte pieces, then the odd ones, so that a lane's 8
// neighbouring floats are read without conflicts.
template <int W>
__device__ __forceinline__ int raw_piece(int row, int q) {
  const int at = (q >> 1) + (q & 1) * (W / 8);
  return row * (W / 4) + (W == 32 ? at ^ ((row & 1) << 2) : at);
}

template <int P, int R>
struct Layout {
  static constexpr int kRawY = 0, kRawZ = kRawY + kC * P * 4;
  static constexpr int kTiles = kRawZ + kC * R * 4;
  // high halves, then low halves, of x, y, z and the state
  static constexpr int kX = kTiles, kY = kX + kC * P * 4, kZ = kY + kC * P * 4;
  static constexpr int kState = kZ + kC * R * 4;
  static constexpr int kEnd = kState + P * R * 4;
  // where the two halves of a group exchange their sums: x's tile of these positions, which
  // both have read by then, where it is large enough
  static constexpr bool kShared = P >= R;
  static constexpr int kSums = kShared ? kX : kEnd, kGroup = kShared ? 16 * P * 2 : 16 * R * 4;
  static constexpr int kHalf = kShared ? kC * P * 2 : 16 * R * 2;
  static constexpr int kBytes = kShared ? kEnd : kEnd + 8 * 16 * R * 2;
  static_assert(P * R * 4 <= kState - kTiles, "rare_chunk's state lies in the tiles");
  // the warps' parts of the state: 16 rows by kColTiles tiles of 8 columns
  static constexpr int kRowGroups = P / 16 < 8 ? P / 16 : 8;
  static constexpr int kColGroups = 8 / kRowGroups > R / 16 ? R / 16 : 8 / kRowGroups;
  static constexpr int kColTiles = R / 8 / kColGroups;
  static constexpr int kBlocks = P == 128 ? 1 : P == 32 && R == 32 ? 3 : 2;    // on an SM
};

struct Segments {           // pieces of a row that are worked on side by side
  int count, chunks;        // pieces, chunks of a piece
  float* state;             // (passes, count - 1, B H, p * r): after each piece but the last
  float* kept;              // (passes, count - 1, B H): what a piece does to the state before it
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

// A weight of the state, l^u, as rest 2^e with rest in [1, 2); below 2^-126 there is none.
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

// The parts of shared memory that are not tiles.
struct alignas(16) Small {
  float max_x[kC], max_y[kC], max_z[kC];    // the rows' largest entries
  float max_state[8];                   // of the state, by warp
  // per position j: 2^(exponents of y_j and z_j, below the largest) / what z_j's scale has more,
  // and that times l^(15 - j % 16) (back: l^(j % 16))
  float2 weight[kC];
  uint16_t added[2][kC];                // j's weight in the state, as a product of two halves
  float power[kC + 1];                  // l^n
  int document[kC];
};

// The passes of one launch: sweeps over the same B, T and H whose heads have the same
// padded sizes.
struct Passes {
  Pass at[3];
};

// Position by position, for a chunk with numbers that are not finite: the state in shared
// memory, columns over the lanes, rows over kThreads / R groups of threads.
template <int P, int R, bool STATE>
__device__ void rare_chunk(float* state, float* sums, const Pass& a, const Shape& s,
                           const Weights& w, unsigned long long cuts, bool next_cut, Decay l,
                           int64_t b, int h, int t0, int slice) {
  constexpr int kGroups = kThreads / R;
  const int c = threadIdx.x % R, group = threadIdx.x / R, r = slice * R + c;
  for (int k = 0; k < w.n; ++k) {
    const int i = a.back ? w.n - 1 - k : k;
    const float* x = a.x.p + b * a.x.bs + (t0 + i) * a.x.ts + (int64_t)h * a.p;
    const float* y = a.y.p + b * a.y.bs + (t0 + i) * a.y.ts + (int64_t)h * a.p;
    const float z = r < a.r ? a.z.p[b * a.z.bs + (t0 + i) * a.z.ts + (int64_t)h * a.r + r] : 0.f;
    const bool on = k < w.n - 1 || a.back || w.tail;       // the state goes on from here
    const bool cut = k < w.n - 1 ? (a.back ? cuts >> i & 1 : cuts >> (i + 1) & 1)
                                 : (a.back ? cuts & 1 : next_cut);
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
// the state after the piece is wanted.  Warps w and w + 4 have the same 16 positions: each
// takes every other 16 positions of y and z and half of the state's rows, and they add
// their sums at the end (so no warp has more than two of the four position blocks, and the
// operands' registers are few enough for two blocks on an SM).
template <int P, int R, bool STATE>
__global__ void __launch_bounds__(kThreads, Layout<P, R>::kBlocks)
    chunk_kernel(const __grid_constant__ Passes passes, const Shape s, const Segments g,
                 const unsigned per_pass) {
  using L = Layout<P, R>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Small m;
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
  const int group = warp & 3, half = warp >> 2;
  const int mat = lane >> 3, mat_row = lane & 7;
  const bool back = a.back;
  const Decay l(s.log_decay[h]);
  for (int i = threadIdx.x; i <= kC; i += kThreads)
    m.power[i] = i == 0 ? 1.f : expf((float)i * s.log_decay[h]);

  const int chunks = (s.T + kC - 1) / kC;
  const int c0 = seg * g.chunks, c1 = min(c0 + g.chunks, chunks);
  // pieces and chunks are counted in the direction of the sweep
  auto start = [&](int c) { return (back ? chunks - 1 - c : c) * kC; };
  const uint32_t* marks = s.reset ? s.reset + b * s.T : nullptr;
  auto resets = [&](int c, bool& next) {
    const int t0 = start(c), n = min(kC, s.T - t0);
    next = false;
    if (!marks) return 0ull;
    const unsigned lo = __ballot_sync(0xffffffffu, lane < n && marks[t0 + lane] != 0);
    const unsigned hi = __ballot_sync(0xffffffffu, lane + 32 < n && marks[t0 + lane + 32] != 0);
    next = !back && t0 + n < s.T && marks[t0 + n] != 0;
    return (unsigned long long)hi << 32 | lo;
  };
  auto weights = [&](int c, unsigned long long cuts, bool next) {
    const int t0 = start(c), n = min(kC, s.T - t0);
    return Weights(cuts, n, t0 + n < s.T, back ? cuts & 1 : next);
  };

  // the state, in the layout of a product's result: rows row0 + quad (+ 8), columns col0 + 8 nt
  // + 2 t (+ 1); warps without a part keep zeros
  const int row0 = (warp % L::kRowGroups) * 16;
  const bool has_state = warp / L::kRowGroups < L::kColGroups;
  const int col0 = has_state ? warp / L::kRowGroups * L::kColTiles * 8 : 0;
  float X[L::kColTiles][4], d[L::kColTiles][4];
  {
    const int64_t head = (b * s.H + h) * (int64_t)a.p * a.r;
    const float* from = a.from ? a.from + head : nullptr;
    int64_t ps = a.p_stride, rs = a.r_stride;
    bool drop = !has_state;
    if (STATE) {
      from = nullptr;
    } else if (seg > 0) {
      from = g.state + ((pass * (int64_t)(g.count - 1) + seg - 1) * heads + b * s.H + h) * a.p * a.r;
      ps = a.r;
      rs = 1;
    } else if (!back) {
      drop = drop || (marks && marks[0] != 0);
    }
    const bool first = !STATE && seg == 0 && !back;          // its own step of the decay
#pragma unroll
    for (int nt = 0; nt < L::kColTiles; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int p = row0 + quad + (e >> 1) * 8, r = slice * R + col0 + nt * 8 + 2 * t + (e & 1);
        const float v = from && !drop && p < a.p && r < a.r ? from[p * ps + r * rs] : 0.f;
        X[nt][e] = first ? l(v) : v;
        d[nt][e] = 0.f;
      }
  }

  float* raw_y = reinterpret_cast<float*>(smem + L::kRawY);
  float* raw_z = reinterpret_cast<float*>(smem + L::kRawZ);
  const uint32_t base = smem_address(smem);
  // 16-byte accesses where every row allows them
  auto whole = [&](const Operand& o, int width) {
    return ((reinterpret_cast<uintptr_t>(o.p) & 15) == 0) && ((o.bs | o.ts | width) & 3) == 0;
  };
  const bool wide_x = !STATE && whole(a.x, a.p), wide_y = whole(a.y, a.p), wide_z = whole(a.z, a.r);
  auto fetch_rows = [&](auto width, float* raw, const Operand& o, int columns, int from, int t0,
                        bool wide) {
    constexpr int W = decltype(width)::value;
    const int n = min(kC, s.T - t0);
    const float* p = o.p + b * o.bs + t0 * o.ts + (int64_t)h * columns + from;
    const int here = columns - from;                      // columns from there on
    if (wide) {
#pragma unroll
      for (int k = 0; k < kC * (W / 4) / kThreads; ++k) {
        const int i = threadIdx.x + k * kThreads, row = i / (W / 4), q = i % (W / 4);
        const bool take = row < n && q * 4 < here;
        copy16(smem_address(raw) + raw_piece<W>(row, q) * 16, take ? p + row * o.ts + q * 4 : o.p,
               take);
      }
    } else {
      for (int i = threadIdx.x; i < kC * W; i += kThreads) {
        const int row = i / W, col = i % W;
        const bool take = row < n && col < here;
        copy4(smem_address(raw) + raw_piece<W>(row, col >> 2) * 16 + (col & 3) * 4,
              take ? p + row * o.ts + col : o.p, take);
      }
    }
  };
  auto fetch = [&](int c) {
    fetch_rows(std::integral_constant<int, P>{}, raw_y, a.y, a.p, 0, start(c), wide_y);
    fetch_rows(std::integral_constant<int, R>{}, raw_z, a.z, a.r, slice * R, start(c), wide_z);
  };
  // A lane's share of x, y and z: 8 neighbouring columns of a row, W / 32 rows in turn of the
  // warp's 8.
  auto row_of = [&](int W, int k) { return warp * 8 + k * (256 / W) + lane / (W / 8); };
  constexpr int kPassesX = P / 32, kPassesZ = R / 32;
  float x[STATE ? 1 : kPassesX][8];
  auto fetch_x = [&](int c) {
    const int t0 = start(c), n = min(kC, s.T - t0), col = lane % (P / 8) * 8;
#pragma unroll
    for (int k = 0; k < kPassesX; ++k) {
      const int row = row_of(P, k);
      const float* p = a.x.p + b * a.x.bs + (t0 + row) * a.x.ts + (int64_t)h * a.p + col;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[k][e] = 0.f;
      if (row < n) {
        if (wide_x) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            if (col + 4 * q >= a.p) continue;
            const float4 v = *reinterpret_cast<const float4*>(p + 4 * q);
            x[k][4 * q] = v.x, x[k][4 * q + 1] = v.y, x[k][4 * q + 2] = v.z, x[k][4 * q + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (col + e < a.p) x[k][e] = p[e];
        }
      }
    }
  };
  const bool pairs_o = ((reinterpret_cast<uintptr_t>(a.out) & 7) == 0) && (a.r & 1) == 0;

  fetch(c0);
  if constexpr (!STATE) fetch_x(c0);
  float run = 1.f;                      // STATE: what the piece does to the state before it
  float kept = 1.f, odd = 0.f;          // of the last chunk; odd: 0 unless something is not finite
  Scale by_d(0.f, 0);

  for (int c = c0;; ++c) {
    copies_done();
    // y and z are here, the last chunk's tiles are read
    if (__syncthreads_or(!(odd == 0.f))) {
      bool next;
      const unsigned long long cuts = resets(c - 1, next);
      float* state = reinterpret_cast<float*>(smem + L::kTiles);
      auto each = [&](auto f) {
#pragma unroll
        for (int nt = 0; nt < L::kColTiles; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            f(X[nt][e], state[(row0 + quad + (e >> 1) * 8) * R + col0 + nt * 8 + 2 * t + (e & 1)]);
      };
      if (has_state) each([](float& v, float& to) { to = v; });
      __syncthreads();
      rare_chunk<P, R, STATE>(state, state + P * R, a, s, weights(c - 1, cuts, next), cuts, next, l,
                              b, h, start(c - 1), slice);
      __syncthreads();
      if (has_state) each([](float& v, float& to) { v = to; });
      __syncthreads();
    } else if (c > c0) {
#pragma unroll
      for (int nt = 0; nt < L::kColTiles; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) X[nt][e] = fmaf(kept, X[nt][e], by_d(d[nt][e]));
    }
    if (c == c1) break;
    odd = 0.f;
    bool next;
    const unsigned long long cuts = resets(c, next);
    const Weights w = weights(c, cuts, next);
    const int t0 = start(c), n = w.n;

    if (!STATE) {                       // the state's largest entry
      float most = 0.f;
#pragma unroll
      for (int nt = 0; nt < L::kColTiles; ++nt)
#pragma unroll
        for (int e = 0; e < 4; e += 2)
          most = fmax3(most, fabsf(X[nt][e]), fabsf(X[nt][e + 1]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (lane == 0) m.max_state[warp] = most;
    }
    // the rows' largest entries
    auto largest = [&](auto width, const float (&v)[8], int row, float* max_row) {
      constexpr int kLanes = decltype(width)::value / 8;
      float most = fmax3(fabsf(v[0]), fabsf(v[1]), fabsf(v[2]));
      most = fmax3(most, fabsf(v[3]), fabsf(v[4]));
      most = fmax3(most, fabsf(v[5]), fabsf(v[6]));
      most = fmaxf(most, fabsf(v[7]));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1)
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (lane % kLanes == 0) max_row[row] = most;
    };
    float y[kPassesX][8], z[kPassesZ][8];
    auto read = [&](auto width, const float* raw, float (&v)[8], int row) {
      constexpr int W = decltype(width)::value;
      const int q = lane % (W / 8);
      const float4 u0 = reinterpret_cast<const float4*>(raw)[raw_piece<W>(row, 2 * q)];
      const float4 u1 = reinterpret_cast<const float4*>(raw)[raw_piece<W>(row, 2 * q + 1)];
      v[0] = u0.x, v[1] = u0.y, v[2] = u0.z, v[3] = u0.w;
      v[4] = u1.x, v[5] = u1.y, v[6] = u1.z, v[7] = u1.w;
    };
#pragma unroll
    for (int k = 0; k < kPassesX; ++k)
      read(std::integral_constant<int, P>{}, raw_y, y[k], row_of(P, k));
#pragma unroll
    for (int k = 0; k < kPassesZ; ++k)
      read(std::integral_constant<int, R>{}, raw_z, z[k], row_of(R, k));
#pragma unroll
    for (int k = 0; k < kPassesX; ++k)
      largest(std::integral_constant<int, P>{}, y[k], row_of(P, k), m.max_y);
#pragma unroll
    for (int k = 0; k < kPassesZ; ++k)
      largest(std::integral_constant<int, R>{}, z[k], row_of(R, k), m.max_z);
    if constexpr (!STATE) {
#pragma unroll
      for (int k = 0; k < kPassesX; ++k)
        largest(std::integral_constant<int, P>{}, x[k], row_of(P, k), m.max_x);
    }
    __syncthreads();

    // what the rows weigh: lane looks at rows lane and lane + 32
    int most = -1000, most_added = -1000;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = lane + 32 * k;
      const float my = m.max_y[j], mz = m.max_z[j];
      if (my == 0.f || mz == 0.f) continue;               // nothing there
      const int e = exponent(my) + exponent(mz);
      const Decayed u(m.power, w.added(j, back));
      most = max(most, e);
      if (u.any) most_added = max(most_added, e + u.e);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    most_added = __reduce_max_sync(0xffffffffu, most_added);
    if (most == -1000) most = 0;
    if (most_added == -1000) most_added = 0;
    if (threadIdx.x < kC) {
      // the power of two of l^u goes into the weight, the rest into z's scale
      const int j = threadIdx.x, e = exponent(m.max_y[j]) + exponent(m.max_z[j]);
      const Decayed u(m.power, w.added(j, back));
      const float one = e - most < -126 ? 0.f : a.y_scale * power2(min(e - most, 0)) / u.rest;
      m.weight[j] = make_float2(one, one * m.power[back ? j & 15 : 15 - (j & 15)]);
      const int below = u.any ? min(e + u.e - most_added, 0) : -1000;
      // 2^below as two halves, each 2^-24 at least (0: less than 2^-38 of the largest)
      const int first = max(below, -24), then = max(below - first, -24);
      m.added[0][j] = below < -38 ? 0 : __half_as_ushort(__float2half_rn(power2(first)));
      m.added[1][j] = __half_as_ushort(__float2half_rn(power2(then)));
      m.document[j] = w.document(j);
    }
    const bool far = __any_sync(0xffffffffu, [&] {        // a weight below one half number
      bool any = false;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int j = lane + 32 * k;
        const Decayed u(m.power, w.added(j, back));
        const int below = exponent(m.max_y[j]) + exponent(m.max_z[j]) + u.e - most_added;
        any = any || (u.any && below < -24);
      }
      return any;
    }());
    // the tiles
    auto tile = [&](auto width, int to, const float (&v)[8], int row, float up) {
      constexpr int W = decltype(width)::value;
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) split(up * v[2 * i], up * v[2 * i + 1], hi[i], lo[i]);
      unsigned char* p = smem + to + piece<W>(row, lane % (W / 8));
      *reinterpret_cast<uint4*>(p) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(p + kC * W * 2) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    };
    float max_state = 0.f;
    int e_state = 0;
    if constexpr (!STATE) {
#pragma unroll
      for (int i = 0; i < 8; ++i) max_state = fmaxf(max_state, m.max_state[i]);
      e_state = exponent(max_state);
      if (has_state && max_state > 0.f) {
        const float up = power2(kTop - e_state);
#pragma unroll
        for (int nt = 0; nt < L::kColTiles; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t hi, lo;
            split(up * X[nt][e * 2], up * X[nt][e * 2 + 1], hi, lo);
            unsigned char* p = smem + L::kState + piece<R>(row0 + quad + e * 8, col0 / 8 + nt) + 4 * t;
            *reinterpret_cast<uint32_t*>(p) = hi;
            *reinterpret_cast<uint32_t*>(p + P * R * 2) = lo;
          }
      }
#pragma unroll
      for (int k = 0; k < kPassesX; ++k) {
        const int row = row_of(P, k);
        tile(std::integral_constant<int, P>{}, L::kX, x[k], row, power2(kTop - exponent(m.max_x[row])));
      }
    }
#pragma unroll
    for (int k = 0; k < kPassesX; ++k) {
      const int row = row_of(P, k);
      tile(std::integral_constant<int, P>{}, L::kY, y[k], row, power2(kTop - exponent(m.max_y[row])));
    }
#pragma unroll
    for (int k = 0; k < kPassesZ; ++k) {
      const int row = row_of(R, k);
      tile(std::integral_constant<int, R>{}, L::kZ, z[k], row,
           Decayed(m.power, w.added(row, back)).rest * power2(kTop - exponent(m.max_z[row])));
    }
    __syncthreads();
    if (c + 1 < c1) fetch(c + 1);

    if constexpr (!STATE) {
      uint32_t xh[P / 16][4], xl[P / 16][4];
#pragma unroll
      for (int k = 0; k < P / 16; ++k) {
        const uint32_t from =
            base + L::kX + piece<P>(group * 16 + (mat & 1) * 8 + mat_row, 2 * k + (mat >> 1));
        load4(xh[k], from);
        load4(xl[k], from + kC * P * 2);
      }
      // x y^T for every other 16 positions up to (back: from) this group's own
      float S[2][2][4];
      float most_p[2] = {0.f, 0.f};
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int jb = half + 2 * q;
        if (back ? jb < group : jb > group) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) S[q][0][e] = S[q][1][e] = 0.f;
#pragma unroll
        for (int k = 0; k < P / 16; ++k) {
          uint32_t bh[4], bl[4];
          const uint32_t from =
              base + L::kY + piece<P>(jb * 16 + (mat >> 1) * 8 + mat_row, 2 * k + (mat & 1));
          load4(bh, from);
          load4(bl, from + kC * P * 2);
          products(S[q][0], S[q][1], xh[k], xl[k], bh, bl);
        }
        // its weights, and the rows' largest: l^(i - j) is looked up in the group's own
        // positions, elsewhere it is a product of three powers of at least 0
        const float gap = jb == group ? 1.f : m.power[16 * abs(group - jb) - 15];
        const float side[2] = {gap * m.power[back ? 15 - quad : quad],
                               gap * m.power[back ? 7 - quad : quad + 8]};
#pragma unroll
        for (int jt = 0; jt < 2; ++jt) {
          const int j = jb * 16 + jt * 8 + 2 * t;
          const float4 v = *reinterpret_cast<const float4*>(&m.weight[j]);
          const float one[2] = {v.x, v.z}, other[2] = {v.y, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float value = S[q][jt][e];
            if (jb == group) {
              const int i = quad + (e >> 1) * 8, k = jt * 8 + 2 * t + (e & 1);
              const int apart = back ? k - i : i - k;
              value = apart < 0 ? 0.f : value * (m.power[max(apart, 0)] * one[e & 1]);
            } else {
              value *= side[e >> 1] * other[e & 1];
            }
            if (w.inner && m.document[group * 16 + quad + (e >> 1) * 8] != m.document[j + (e & 1)])
              value = 0.f;
            S[q][jt][e] = value;
          }
          most_p[0] = fmax3(most_p[0], fabsf(S[q][jt][0]), fabsf(S[q][jt][1]));
          most_p[1] = fmax3(most_p[1], fabsf(S[q][jt][2]), fabsf(S[q][jt][3]));
        }
      }
      // x X over this half of the state's rows
      float o[R / 8][4];
#pragma unroll
      for (int nt = 0; nt < R / 8; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][e] = 0.f;
      if (max_state > 0.f) {
#pragma unroll
        for (int k = 0; k < P / 32; ++k) {
          const int kk = half * (P / 32) + k;
          uint32_t ah[4], al[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ah[e] = half ? xh[P / 32 + k][e] : xh[k][e];
            al[e] = half ? xl[P / 32 + k][e] : xl[k][e];
          }
#pragma unroll
          for (int nb = 0; nb < R / 16; ++nb) {
            uint32_t bh[4], bl[4];
            const uint32_t from = base + L::kState +
                                  piece<R>(kk * 16 + (mat & 1) * 8 + mat_row, 2 * nb + (mat >> 1));
            load4_turned(bh, from);
            load4_turned(bl, from + P * R * 2);
            products(o[2 * nb], o[2 * nb + 1], ah, al, bh, bl);
          }
        }
      }
      // Both sums in one scale: the larger's, whichever part it comes from.
      Scale by[2] = {Scale(0.f, 0), Scale(0.f, 0)};
      float up[2];
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const int i = group * 16 + quad + side * 8, u = w.reach(i, back);
        most_p[side] = fmaxf(most_p[side], __shfl_xor_sync(0xffffffffu, most_p[side], 1));
        most_p[side] = fmaxf(most_p[side], __shfl_xor_sync(0xffffffffu, most_p[side], 2));
        int e_p = exponent(most_p[side]);
        const float decay = u < 0 ? 0.f : m.power[u];
        const int apart = e_state + 2 * kTop - most;
        if (max_state > 0.f && decay > 0.f) e_p = max(e_p, apart + exponent(decay) - kTop);
        const Scale in(decay, apart - e_p);
#pragma unroll
        for (int nt = 0; nt < R / 8; ++nt) {
          o[nt][2 * side] = in(o[nt][2 * side]);
          o[nt][2 * side + 1] = in(o[nt][2 * side + 1]);
        }
        up[side] = kTop - e_p < -126 ? 0.f : power2(kTop - e_p);
        by[side] = Scale(a.out_scale, e_p + exponent(m.max_x[i]) + most - 4 * kTop);
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int jb = half + 2 * q;
        if (back ? jb < group : jb > group) continue;
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float f = up[e & 1];
          split(f * S[q][e >> 1][(e & 1) * 2], f * S[q][e >> 1][(e & 1) * 2 + 1], ph[e], pl[e]);
        }
#pragma unroll
        for (int nb = 0; nb < R / 16; ++nb) {
          uint32_t bh[4], bl[4];
          const uint32_t from =
              base + L::kZ + piece<R>(jb * 16 + (mat & 1) * 8 + mat_row, 2 * nb + (mat >> 1));
          load4_turned(bh, from);
          load4_turned(bl, from + kC * R * 2);
          products(o[2 * nb], o[2 * nb + 1], ph, pl, bh, bl);
        }
      }
#pragma unroll
      for (int nt = 0; nt < R / 8; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][e] = by[e >> 1](o[nt][e]);
      // each half of the group writes half of the columns
      pair_barrier(group);                                // both have read x's tile
      auto finish = [&](auto which) {
        constexpr int kMine = decltype(which)::value * (R / 16), kOther = R / 16 - kMine;
        float2* sums = reinterpret_cast<float2*>(smem + L::kSums + group * L::kGroup);
        constexpr int kApart = L::kHalf / (int)sizeof(float2);
#pragma unroll
        for (int k = 0; k < R / 16; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            sums[decltype(which)::value * kApart + (2 * k + e) * 32 + lane] =
                make_float2(o[kOther + k][2 * e], o[kOther + k][2 * e + 1]);
        pair_barrier(group);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = group * 16 + quad + e * 8;
          float* out = a.out + ((b * s.T + t0 + i) * s.H + h) * a.r + slice * R;
#pragma unroll
          for (int k = 0; k < R / 16; ++k) {
            const float2 more = sums[(1 - decltype(which)::value) * kApart + (2 * k + e) * 32 + lane];
            const float v0 = o[kMine + k][2 * e] + more.x, v1 = o[kMine + k][2 * e + 1] + more.y;
            const int r = (kMine + k) * 8 + 2 * t, room = a.r - slice * R;
            odd = fmaf(v0, 0.f, odd);
            odd = fmaf(v1, 0.f, odd);
            if (i >= n) continue;
            if (pairs_o) {
              if (r < room) *reinterpret_cast<float2*>(out + r) = make_float2(v0, v1);
            } else {
              if (r < room) out[r] = v0;
              if (r + 1 < room) out[r + 1] = v1;
            }
          }
        }
      };
      if (half == 0)
        finish(std::integral_constant<int, 0>{});
      else
        finish(std::integral_constant<int, 1>{});
      if (c + 1 < c1) fetch_x(c + 1);
    }
    // what the chunk adds to the state
#pragma unroll
    for (int nt = 0; nt < L::kColTiles; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) d[nt][e] = 0.f;
    if (has_state) {
#pragma unroll
      for (int k = 0; k < kC / 16; ++k) {
        uint32_t ah[4], al[4];
        const uint32_t from =
            base + L::kY + piece<P>(k * 16 + (mat >> 1) * 8 + mat_row, row0 / 8 + (mat & 1));
        load4_turned(ah, from);
        load4_turned(al, from + kC * P * 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = k * 16 + (e >> 1) * 8 + 2 * t;
          const uint32_t f = *reinterpret_cast<const uint32_t*>(&m.added[0][j]);
          ah[e] = times(ah[e], f);
          al[e] = times(al[e], f);
          if (far) {
            const uint32_t f2 = *reinterpret_cast<const uint32_t*>(&m.added[1][j]);
            ah[e] = times(ah[e], f2);
            al[e] = times(al[e], f2);
          }
        }
#pragma unroll
        for (int nb = 0; nb < L::kColTiles / 2; ++nb) {
          uint32_t bh[4], bl[4];
          const uint32_t zat = base + L::kZ + piece<R>(k * 16 + (mat & 1) * 8 + mat_row,
                                                       col0 / 8 + 2 * nb + (mat >> 1));
          load4_turned(bh, zat);
          load4_turned(bl, zat + kC * R * 2);
          products(d[2 * nb], d[2 * nb + 1], ah, al, bh, bl);
        }
      }
    }
    by_d = Scale(a.y_scale, most_added - 2 * kTop);
    const int u = w.kept(back);
    kept = u < 0 ? 0.f : m.power[u];
    if (STATE) run *= kept;
#pragma unroll
    for (int nt = 0; nt < L::kColTiles; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) odd = fmaf(d[nt][e], 0.f, fmaf(X[nt][e], 0.f, odd));
  }

  const bool keep = has_state && (STATE || (a.last && seg == pieces - 1));
  float* to = STATE ? g.state + ((pass * (int64_t)pieces + seg) * heads + b * s.H + h) * a.p * a.r
                    : a.last + (b * s.H + h) * (int64_t)a.p * a.r;
  const int64_t ps = STATE ? a.r : a.p_stride, rs = STATE ? 1 : a.r_stride;
#pragma unroll
  for (int nt = 0; nt < L::kColTiles; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int p = row0 + quad + (e >> 1) * 8, r = slice * R + col0 + nt * 8 + 2 * t + (e & 1);
      if (keep && p < a.p && r < a.r) to[p * ps + r * rs] = X[nt][e];
    }
  if (STATE && threadIdx.x == 0)
    g.kept[(pass * (int64_t)pieces + seg) * heads + b * s.H + h] = run;
}

// The states before the pieces, from what each piece adds to a state and keeps of it, in
// place: a thread an entry, one piece after the other.
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
  if (!a.back)
    X = s.reset && s.reset[b * s.T] != 0 ? 0.f : Decay(s.log_decay[head % s.H])(X);
  for (int k = 0; k < g.count - 1; ++k) {
    float* E = g.state + (pass * (int64_t)(g.count - 1) + k) * total + i;
    const float kept = g.kept[(pass * (int64_t)(g.count - 1) + k) * heads + head];
    X = kept == 0.f ? *E : fmaf(kept, X, *E);
    *E = X;
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
  sweep_kernel<32><<<(unsigned)(B * s.H * ((a.r + 31) / 32)), kT, 0, wxx::stream()>>>(a, s);
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
  return WXX_OK;
}

// n passes of one padded size in one launch, the rows in pieces where there are too few
// sequences and heads to fill the SMs: first what every piece but the last adds to a state,
// then the states before the pieces, then the outputs.
template <int P, int R>
int chunked(const Passes& passes, int n, const Shape& s, int64_t B) {
  using L = Layout<P, R>;
  const Pass& a = passes.at[0];
  int slices = 0;
  for (int i = 0; i < n; ++i) slices = std::max(slices, (passes.at[i].r + R - 1) / R);
  const int64_t heads = B * s.H, blocks = heads * slices, chunks = (s.T + kC - 1) / kC;
  const int64_t resident = (int64_t)wxx::num_sms() * L::kBlocks;
  Segments g{1, (int)chunks, nullptr, nullptr};
  const int64_t most = resident / (blocks * n);
  if (most >= 2) {
    int64_t size = (chunks + most - 1) / most;
    if (size < 4) size = 4;
    g.count = (int)((chunks + size - 1) / size);
    g.chunks = (int)size;
  }
  if (int st = allow_smem(chunk_kernel<P, R, true>, L::kBytes)) return st;
  if (int st = allow_smem(chunk_kernel<P, R, false>, L::kBytes)) return st;
  void* scratch = nullptr;
  if (g.count > 1) {
    const int64_t states = n * (g.count - 1) * heads;
    if (int st = wxx_malloc(&scratch, (uint64_t)(states * (a.p * a.r + 1)) * sizeof(float)))
      return st;
    g.state = static_cast<float*>(scratch);
    g.kept = g.state + states * a.p * a.r;
    const unsigned per = (unsigned)(blocks * (g.count - 1));
    chunk_kernel<P, R, true><<<per * n, kThreads, L::kBytes, wxx::stream()>>>(passes, s, g, per);
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
  chunk_kernel<P, R, false><<<per * n, kThreads, L::kBytes, wxx::stream()>>>(passes, s, g, per);
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
