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
#include "tc_gemm.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <mutex>

WXX_EXPORT int wxx_malloc(void** out, uint64_t nbytes);
WXX_EXPORT int wxx_free(void* p);

namespace {

using wxx_tc::mbar_arrive_expect_tx;
using wxx_tc::mbar_init;
using wxx_tc::mbar_wait;
using wxx_tc::smem_u32;
using wxx_tc::tma_load_3d;

constexpr int kT = 256;
constexpr int kSteps = 16;          // positions of a thread
constexpr int kWarps = 8;           // pieces of a tile, at most
constexpr int kTile = kWarps * kSteps * 32;                // floats of a tile's operand
// Blocks resident on an SM.  Four of the forward's leave 64 registers a thread (two
// are spilled).  Measured with four and with three, the gates being weighed in every
// channel: 70 and 72 us over (32, 1024, 1024) with a gate per 64 channels, 18.5 and 20.5
// over (64, 128, 1024); but 60 and 54 over (1, 65536, 256), whose groups are longer, and
// 21 and 20 without the copy engine.  (Five, which only a gate of 32 channels leaves
// registers for: 71 us against 62 over (32, 1024, 1024).)
constexpr int forward_blocks(bool tma, int seg) { return tma && seg == 1 ? 4 : 3; }
constexpr int kBackwardBlocks = 2;
constexpr int kWaitLimit = 1 << 21; // polls of a published word (about a second)

// A gate's weights a = sigmoid(g) and z = 1 - a are, in one order or the other (z is
// the smaller where g >= 0), small = e / (1 + e) and large = 1 / (1 + e) with e =
// exp(-|g|) <= 1, so that nothing overflows.  Each is good to a few ulp of itself: e = 2^y
// 2^r, y = -|g| log2 e rounded (alone it would cost e y half ulps, 60 at |g| = 80) and r
// what the product and the constant lost, so little that 2^r is 1 + r log 2; 1 + e is
// what the approximate reciprocal takes to an ulp.  From |g| = 88 on small is 0, and gates
// past 104 are taken as that, so that y and r are finite.  For two gates (of
// neighbouring positions), so that the additions and products go in pairs.
struct Halves {
  float small, large;
};
__device__ __forceinline__ float far(float g) {
  float t;
  asm("min.NaN.f32 %0, %1, 0f42D00000;" : "=f"(t) : "f"(fabsf(g)));   // 104
  return t;
}
__device__ __forceinline__ void halves2(float g0, float g1, Halves& w0, Halves& w1) {
  constexpr float kC = -1.4426950408889634f;                          // -log2 e, and what is
  constexpr float kLow = (float)(-1.4426950408889634 - (double)kC);   // left of it
  constexpr float kLog2 = 0.6931471805599453f;
  const float t0 = far(g0), t1 = far(g1);
  float y0, y1, r0, r1, e0, e1, s0, s1;
  mul2(y0, y1, t0, t1, kC, kC);
  fma2(r0, r1, t0, t1, kC, kC, -y0, -y1);
  fma2(r0, r1, t0, t1, kLow, kLow, r0, r1);
  fma2(r0, r1, r0, r1, kLog2, kLog2, 1.0f, 1.0f);
  mul2(e0, e1, fast_exp2(y0), fast_exp2(y1), r0, r1);
  add2(s0, s1, e0, e1, 1.0f, 1.0f);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(w0.large) : "f"(s0));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(w1.large) : "f"(s1));
  mul2(w0.small, w1.small, e0, e1, w0.large, w1.large);
}

struct Weights {
  float a, z;
};
__device__ __forceinline__ Weights weights_of(float g, Halves w) {
  return g >= 0.f ? Weights{w.large, w.small} : Weights{w.small, w.large};
}

// Both weights in one number: the smaller, with the sign set where that is a (which may
// be 0).  The other is 1 less it.
__device__ __forceinline__ float pack(float g, Halves w) { return g >= 0.f ? w.small : -w.small; }
__device__ __forceinline__ Weights unpack(float v) {
  const float small = fabsf(v), large = 1.0f - small;
  return __float_as_int(v) >= 0 ? Weights{large, small} : Weights{small, large};
}

// A gate as the smaller of its weights, which says how much of the other value is
// mixed in, and whether the state is the one that is kept.
struct Gate {
  float w;
  bool keep;
};
__device__ __forceinline__ Gate gate_of(float g, Halves w) { return {w.small, g >= 0.f}; }
__device__ __forceinline__ Gate gate_of(Weights w) {
  return {w.z < w.a ? w.z : w.a, w.z < w.a};     // a NaN gives one
}

// a h + z x as the larger-weighted of the two plus the smaller weight times
// their difference: a constant gate's fixed point stays where it is (a and z,
// each rounded, do not add up to 1: at z = 1e-3 that error is multiplied by
// 1000), and a saturated gate keeps or replaces h exactly.
__device__ __forceinline__ float mix(Gate g, float h, float x) {
  const float base = g.keep ? h : x, other = g.keep ? x : h;
  return fmaf(g.w, other - base, base);
}
// The same where the difference may be more than the type holds: an infinity, or
// values of about 1e38 and opposite signs.
__device__ __forceinline__ float mix_any(Gate g, float h, float x) {
  const float base = g.keep ? h : x, other = g.keep ? x : h, apart = other - base;
  return fabsf(apart) < INFINITY ? fmaf(g.w, apart, base)
                                 : fmaf(g.w, other, (1.0f - g.w) * base);
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

struct Yes {
  static constexpr bool value = true;
};
struct No {
  static constexpr bool value = false;
};

struct Operand {            // (B, T, ...) with unit stride inside
  const float* p;
  int64_t bs, ts;
  bool pairs;               // an even number of channels, every row 8-byte aligned
};
Operand operand(const float* p, int64_t bs, int64_t ts, int64_t channels) {
  return {p, bs, ts, (reinterpret_cast<uintptr_t>(p) & 7) == 0 && ((bs | ts | channels) & 1) == 0};
}

// n / d for n < 2^31 as a product: d <= 2^s, m = ceil(2^(31 + s) / d) < 2^32.
struct Divider {
  unsigned m, s, d;
  static Divider of(unsigned d) {
    unsigned s = 0;
    while ((1ull << s) < d) ++s;
    return {(unsigned)(((1ull << (31 + s)) + d - 1) / d), 31 + s, d};
  }
  __device__ __forceinline__ unsigned operator()(unsigned n) const {
    return (unsigned)(((unsigned long long)n * m) >> s);
  }
};

// The tiles of a scan and their scratch.  Every published number travels in one
// 64-bit word with the launch's tag in the upper half, so a reader needs no fence,
// and what an earlier launch left says nothing: the scratch is kept from call to
// call and never cleared (clearing it took 2 us of the GPU and 4 of the host).
struct Counters {
  unsigned ticket, done;      // tiles handed out, blocks that have ended
  unsigned launches;          // the tag is one more (2^32 launches before it returns)
};
struct Chain {
  Counters* counters;
  ulonglong2* tile;           // {A, b} of a tile, 32 channels
  unsigned long long* group;  // the state after each group of tiles
  Divider blocks;             // blocks of 32 channels, all sequences
  Divider row_blocks;         // of one sequence
  int tiles;                  // tiles of a row
  unsigned total;             // tiles of all rows
  Divider per;                // channels of a gate
  int gates;                  // gates that 32 channels can have, at most
  int* err;
};

__device__ __forceinline__ unsigned long long tagged(float v, unsigned tag) {
  return (unsigned long long)tag << 32 | __float_as_uint(v);
}
__device__ __forceinline__ void publish(unsigned long long* p, float v, unsigned tag) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(tagged(v, tag)) : "memory");
}
__device__ __forceinline__ void publish(ulonglong2* p, Stretch s, unsigned tag) {
  asm volatile("st.relaxed.gpu.global.v2.u64 [%0], {%1, %2};" ::"l"(p), "l"(tagged(s.A, tag)),
               "l"(tagged(s.b, tag))
               : "memory");
}
__device__ __forceinline__ bool peek(const unsigned long long* p, float& v, unsigned tag) {
  unsigned long long u;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(u) : "l"(p) : "memory");
  v = __uint_as_float((unsigned)u);
  return (unsigned)(u >> 32) == tag;
}
__device__ __forceinline__ bool peek(const ulonglong2* p, Stretch& s, unsigned tag) {
  unsigned long long u, v;
  asm volatile("ld.relaxed.gpu.global.v2.u64 {%0, %1}, [%2];" : "=l"(u), "=l"(v) : "l"(p) : "memory");
  s.A = __uint_as_float((unsigned)u);
  s.b = __uint_as_float((unsigned)v);
  return (unsigned)(u >> 32) == tag && (unsigned)(v >> 32) == tag;
}
// Polls end when every lane has its words, or give up: at the limit (error word
// set) or as soon as another block has given up.
__device__ __forceinline__ bool poll_over(bool ready, int& n, int* err) {
  if (__all_sync(0xffffffffu, ready)) return true;
  ++n;
  if (n >= kWaitLimit) {
    wxx_device_fail(err, WXX_DEV_ERR_MBAR_TIMEOUT);
    return true;
  }
  return (n & 1023) == 0 && *reinterpret_cast<volatile int*>(err) == WXX_DEV_ERR_MBAR_TIMEOUT;
}

struct Joint {                    // shared memory of a block
  Stretch piece[2][kWarps][32];   // by turns: a warp may start the next tile early
  Stretch before[kWarps][32];
  float group[32];
  uint64_t full;                  // barrier: a tile's inputs have come
  unsigned next, tag;
  int abort[2];                   // a wait for them has given up, by turns
};

// A block works through tiles, the next one's inputs on their way while this
// one is joined and written.  Where tiles wait for one another they are handed
// out by a ticket in the order of the join, and every block takes its own in that
// order, so whoever a block waits for is already being worked on.
__device__ __forceinline__ unsigned take_ticket(const Chain& c) {
  return atomicAdd(&c.counters->ticket, 1u);
}
// A block's end (one thread): the last block leaves the counters for the next launch.
__device__ __forceinline__ void block_ends(const Chain& c) {
  if (atomicAdd(&c.counters->done, 1u) + 1 < gridDim.x) return;
  c.counters->ticket = 0;
  c.counters->done = 0;
  ++c.counters->launches;
}

// Where a thread's piece lies: lane = one of 32 channels, warp = a piece of
// kSteps positions.  Tiles, channels and positions are numbered in 32 bits (the
// host checks that they fit) and divided by products: 64-bit divisions cost as
// much as the piece itself.
struct Place {
  unsigned q, b, j;           // channel block (all sequences), sequence, place in the row
  int d, i, row, t0, left;    // channel, place of the piece, its row in the tile, its first
};                            // position, positions there are
__device__ __forceinline__ Place place_of(const Chain& c, unsigned id, bool backwards, int T,
                                          int D) {
  Place p;
  const int warps = blockDim.x >> 5;
  p.j = c.blocks(id);
  p.q = id - p.j * c.blocks.d;
  p.b = c.row_blocks(p.q);
  p.d = (int)(p.q - p.b * c.row_blocks.d) * 32 + (threadIdx.x & 31);
  p.i = threadIdx.x >> 5;
  p.row = (backwards ? warps - 1 - p.i : p.i) * kSteps;
  p.t0 = (backwards ? c.tiles - 1 - (int)p.j : (int)p.j) * warps * kSteps + p.row;
  p.left = p.d < D ? max(0, min(kSteps, T - p.t0)) : 0;
  return p;
}

// A tile's inputs come to shared memory as [position][32 channels].  With kTma
// one thread asks for a box of each operand (what lies outside the tensor reads as
// zero); rows that are not 16-byte aligned are copied by the threads, float by
// float or in pairs, and so is a gate of several channels, as [position][gates].
__device__ __forceinline__ void copy_float(float* dst, const float* src, bool here) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(here ? 4 : 0)
               : "memory");
}
// The barrier takes this thread's arrival when its copies are done.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// This warp's piece of an operand, `back` positions earlier (zero before position 0,
// after the last and past the last channel).  Where rows and channels come in pairs of
// floats, half the lanes copy a position each, two channels at a time: (16, 4096, 250)
// 53 + 91 us, 59 + 103 float by float.
__device__ __forceinline__ void copy_piece(float* tile, const Operand& o, const Place& p,
                                           int back, int T, int D) {
  const int lane = threadIdx.x & 31;
  if (o.pairs) {
    const int half = lane >> 4, in_row = 2 * (lane & 15), d = p.d - lane + in_row;
    float* dst = tile + (p.row + half) * 32 + in_row;
    int t = p.t0 + half;
    const float* src = o.p + p.b * o.bs + (int64_t)(t - back) * o.ts + d;
#pragma unroll 4
    for (int k = 0; k < kSteps; k += 2) {
      const bool here = t < T && t >= back && d < D;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(dst + k * 32)),
                   "l"(here ? src : o.p), "r"(here ? 8 : 0)
                   : "memory");
      t += 2;
      src += 2 * o.ts;
    }
    return;
  }
  float* dst = tile + p.row * 32 + lane;
  const float* src = o.p + p.b * o.bs + (p.t0 - back) * o.ts + p.d;
#pragma unroll 4
  for (int k = 0; k < kSteps; ++k) {
    const bool here = k < p.left && p.t0 + k >= back;
    copy_float(dst + k * 32, here ? src : o.p, here);
    src += o.ts;
  }
}
// Two threads a position; the block's first gate is gate 0 of the tile.
__device__ __forceinline__ int first_gate(const Chain& c, const Place& p) {
  return c.per(p.d - (threadIdx.x & 31));
}
__device__ __forceinline__ void copy_gates(float* tile, const Operand& g, const Chain& c,
                                           const Place& p, int T, int D) {
  const int d0 = p.d - (threadIdx.x & 31), first = first_gate(c, p);
  const int n = c.per(min(d0 + 31, D - 1)) - first + 1;
  const int row = threadIdx.x >> 1, t = p.t0 - p.row + row;
  const float* src = g.p + p.b * g.bs + t * g.ts + first;
  for (int k = threadIdx.x & 1; k < n; k += 2)
    copy_float(tile + row * c.gates + k, t < T ? src + k : g.p, t < T);
}

// A gate for all of a warp's channels: the first threads each load the gate of one
// position of the tile (past the last: keep the state) and, by the time the tile is
// begun, have put its weights into shared memory, where a pair of positions is one
// read, and for the forward the products of a over its piece (a piece is 16 lanes).
// Their arrival is part of the tile's barrier.  Weighed in every channel, (32, 1024,
// 1024) with a gate per 64 channels took 70 us forward, so 60.
__device__ __forceinline__ float warp_gate(const Operand& g, const Chain& c, const Place& p,
                                           int T) {
  const int row = threadIdx.x, t = p.t0 - p.row + row;
  if (row >= (int)(blockDim.x >> 5) * kSteps || t >= T) return INFINITY;
  return g.p[p.b * g.bs + t * g.ts + first_gate(c, p)];
}
__device__ __forceinline__ void weigh(float2* tile, float* upto, float gate, uint64_t* bar) {
  const int rows = (blockDim.x >> 5) * kSteps, row = threadIdx.x;
  if ((row & ~31) >= rows) return;
  Halves half, same;
  halves2(gate, gate, half, same);
  const Weights w = weights_of(gate, half);
  if (upto) {
    static_assert(kSteps == 16, "a piece is half a warp");
    float A = w.a;
#pragma unroll
    for (int o = 1; o < kSteps; o <<= 1) {
      const float before = __shfl_up_sync(0xffffffffu, A, o, kSteps);
      if ((row & (kSteps - 1)) >= o) A *= before;
    }
    if (row < rows) upto[row] = A;
  }
  if (row >= rows) return;
  tile[row] = make_float2(w.a, w.z);
  wxx_tc::mbar_arrive(bar);
}
// The weights of positions k and k + 1 of a warp's piece.
__device__ __forceinline__ void weighed(const float2* piece, int k, Weights& w0, Weights& w1) {
  const float4 v = *reinterpret_cast<const float4*>(piece + k);
  w0 = {v.x, v.y};
  w1 = {v.z, v.w};
}

// Joins the pieces of a tile (warp i of the order holds piece `mine`) with
// everything before it.  j: the tile's place in its row, q: its channel block.
// Returns the state before this warp's piece.  The order of the additions
// depends on j alone: the state after the group before, the tiles of the same group
// so far (kWarps segments of kSeg tiles, one looked at by each warp), the pieces.
// fetch_next is called once, when every warp has taken its inputs from shared
// memory.
template <int kSeg, class F>
__device__ __forceinline__ float join_tile(const Chain& c, Joint& s, int turn, const Place& p,
                                           Stretch mine, float start, F fetch_next) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, i = p.i;
  auto& piece = s.piece[turn];
  piece[i][lane] = mine;
  __syncthreads();
  if (c.tiles > 1 && i == 0) {
    Stretch all = mine;
    for (int k = 1; k < warps; ++k) all = join(all, piece[k][lane]);
    publish(c.tile + ((int64_t)p.q * c.tiles + p.j) * 32 + lane, all, s.tag);
  }
  fetch_next();
  float h = start;
  if (c.tiles > 1) {
    constexpr int kGroup = kSeg * kWarps;
    const int r = p.j % kGroup, g = p.j / kGroup;
    const int64_t groups = (c.tiles + kGroup - 1) / kGroup;
    const ulonglong2* row = c.tile + ((int64_t)p.q * c.tiles + g * kGroup + i * kSeg) * 32 + lane;
    // segment i: tiles i kSeg .. of the group, those before r
    Stretch seg[kSeg];
    int n = 0;
    while (true) {
      bool ready = true;
#pragma unroll
      for (int k = 0; k < kSeg; ++k) {
        seg[k] = {1.0f, 0.0f};
        if (i * kSeg + k < r) ready = peek(row + k * 32, seg[k], s.tag) && ready;
      }
      if (poll_over(ready, n, c.err)) break;
    }
    Stretch before = seg[0];
#pragma unroll
    for (int k = 1; k < kSeg; ++k) before = join(before, seg[k]);
    s.before[i][lane] = before;
    if (i == 0) {
      if (g > 0) {
        n = 0;
        while (!poll_over(peek(c.group + (p.q * groups + g - 1) * 32 + lane, h, s.tag), n, c.err)) {
        }
      }
      s.group[lane] = h;
    }
    __syncthreads();
    h = s.group[lane];
#pragma unroll
    for (int k = 0; k < kWarps; ++k) h = through(s.before[k][lane], h);
    for (int k = 0; k < i; ++k) h = through(piece[k][lane], h);
    if (i == warps - 1 && r == kGroup - 1)
      publish(c.group + (p.q * groups + g) * 32 + lane, through(mine, h), s.tag);
    return h;
  }
  for (int k = 0; k < i; ++k) h = through(piece[k][lane], h);
  return h;
}

// The document starts of this warp's piece: lane k's word is position k's.
__device__ __forceinline__ uint32_t reset_word(const uint32_t* __restrict__ reset, const Place& p,
                                               int T) {
  const int lane = threadIdx.x & 31;
  return reset && lane < kSteps && p.t0 + lane < T ? reset[(int64_t)p.b * T + p.t0 + lane] : 0u;
}

// A block's way through its tiles, the same in both directions.  fetch asks for
// a tile's inputs, ready is called before the wait for them, work with a tile when they
// are there; it calls back (with the place of the next) once it has taken them.
template <bool kBackwards, class Fetch, class Ready, class Work>
__device__ __forceinline__ void through_tiles(const Chain& c, Joint& s, unsigned arrivals,
                                              const uint32_t* reset, int T, int D, Fetch fetch,
                                              Ready ready, Work work) {
  if (threadIdx.x == 0) {
    mbar_init(&s.full, arrivals);
    wxx_tc::fence_barrier_init();
    s.abort[0] = s.abort[1] = 0;
    if (c.tiles > 1) {
      s.tag = *reinterpret_cast<volatile unsigned*>(&c.counters->launches) + 1;
      s.next = take_ticket(c);
    }
  }
  __syncthreads();
  unsigned id = c.tiles == 1 ? blockIdx.x : s.next;
  if (id >= c.total) {
    if (c.tiles > 1 && threadIdx.x == 0) block_ends(c);
    return;
  }
  Place p = place_of(c, id, kBackwards, T, D);
  fetch(p);
  uint32_t starts = reset_word(reset, p, T);
  __syncthreads();             // s.next has been read
  int turn = 0;
  for (;; turn ^= 1) {
    if (c.tiles > 1 && threadIdx.x == 0) s.next = take_ticket(c);
    const unsigned cut = __ballot_sync(0xffffffffu, starts != 0);
    ready(turn);
    mbar_wait(&s.full, turn, &s.abort[turn], c.err);
    Place after = p;
    work(p, cut, turn, [&] {
      // after a wait that gave up nothing more is asked for: the tile's numbers
      // are wrong, the error word says so, and no copy is in flight but its own
      id = s.abort[turn] ? c.total : c.tiles == 1 ? id + gridDim.x : s.next;
      if (id >= c.total) return;
      after = place_of(c, id, kBackwards, T, D);
      fetch(after);
      starts = reset_word(reset, after, T);
    });
    if (id >= c.total) break;
    p = after;
  }
  // a last wait for the copies of a tile that did not come, before the block's
  // shared memory goes to another
  if (s.abort[turn]) {
    int given_up = 0;
    mbar_wait(&s.full, turn, &given_up, c.err);
  }
  if (c.tiles > 1 && threadIdx.x == 0) block_ends(c);
}

__device__ __forceinline__ float* aligned_smem(float* p) {
  return reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(p) + 127) & ~uintptr_t(127));
}

// A tile is 32 channels by up to kWarps pieces of kSteps positions.  A piece's
// inputs come through shared memory into registers and stay there while the
// state before it is found, so each is read once and h is written once, 12 bytes
// a position.  A piece is run from a zero state: what it gives at every position,
// and the product of the weights up to there, which then takes the state that the
// join gives.  A warp whose piece is whole and holds no reset (nearly all) runs
// without the tests for them, and runs it again with them where it comes out
// infinite or NaN: a difference of two values may have passed the largest number
// (asking costs 1 us at (1, 65536, 256) at most).
//
// A row of 8192 positions has 64 tiles, so (16, 8192, 256) gives 8192 tiles for 592
// blocks: 77 us, 5.2 TB/s of its 403 MB, the join's looks at other tiles and the
// latency of a tile's steps taking what a plain copy would not (without any join 5 us
// less).  (1, 65536, 256) has 8 rows of tiles side by side and waits for its hops: 55 us,
// 3.7 TB/s.  Measured against 79 and 54 us and not kept: two channels a lane (80 and 61 us; a third of the
// instructions less, but fewer warps to hide latencies), a second buffer of inputs
// (85 us: the tiles it holds back are the ones that others wait for), pieces of 8 (95
// us) and 32 positions (76 us forward, but 151 backward, 14 more, and the length is one
// for both), groups of groups (83 and 66 us), a look at the tiles before while the own
// one is still being put together (85 and 63 us: it is repeated more often, and the own
// tile is published later).
template <bool kTma, int kSeg, bool kWarpGate>
__global__ void __launch_bounds__(kT, forward_blocks(kTma, kSeg))
    recurrence_forward_kernel(float* __restrict__ h, float* __restrict__ h_last,
                              const __grid_constant__ CUtensorMap map_x,
                              const __grid_constant__ CUtensorMap map_g, Operand x, Operand g,
                              const float* __restrict__ h0, const uint32_t* __restrict__ reset,
                              int T, int D, Chain c) {
  extern __shared__ float s_raw[];
  __shared__ Joint s;
  float *s_x = aligned_smem(s_raw), *s_g = s_x + kTile;
  // kWarpGate, by turns: the weights of a tile's positions, the products of a in a piece
  constexpr int kRows = kWarps * kSteps;
  float2* s_w = reinterpret_cast<float2*>(s_g);
  float* s_A = s_g + 4 * kRows;
  float gate = 0.f;                 // kWarpGate: of this thread's position of the next tile
  const bool own_gate = !kWarpGate && c.per.d == 1;
  const unsigned box = (blockDim.x >> 5) * kSteps * 32 * sizeof(float);
  auto fetch = [&](const Place& p) {
    if (kTma && threadIdx.x == 0) {
      mbar_arrive_expect_tx(&s.full, own_gate ? 2 * box : box);
      tma_load_3d(smem_u32(s_x), &map_x, &s.full, p.d, p.t0 - p.row, p.b);
      if (own_gate) tma_load_3d(smem_u32(s_g), &map_g, &s.full, p.d, p.t0 - p.row, p.b);
    }
    if (!kTma) copy_piece(s_x, x, p, 0, T, D);
    if (!kTma && own_gate) copy_piece(s_g, g, p, 0, T, D);
    if (kWarpGate) gate = warp_gate(g, c, p, T);
    else if (!own_gate) copy_gates(s_g, g, c, p, T, D);
    if (!kTma || !(kWarpGate || own_gate)) copies_arrive(&s.full);
  };
  auto ready = [&](int turn) {
    if (kWarpGate) weigh(s_w + turn * kRows, s_A + turn * kRows, gate, &s.full);
  };
  const unsigned arrivals = (kTma ? 1 : 0) + (!kTma || !(kWarpGate || own_gate) ? blockDim.x : 0) +
                            (kWarpGate ? blockDim.x / 2 : 0);
  through_tiles<false>(c, s, arrivals, reset, T, D, fetch, ready, [&](const Place& p, unsigned cut,
                                                                      int turn, auto next) {
    const bool whole = __all_sync(0xffffffffu, p.left == kSteps && cut == 0);
    const int stride = own_gate ? 32 : c.gates;
    const float* sx = s_x + p.row * 32 + (threadIdx.x & 31);
    const float* sg = s_g + p.row * stride +
                      (own_gate ? (int)(threadIdx.x & 31)
                                : (int)c.per(min(p.d, D - 1)) - first_gate(c, p));
    const float2* sw = s_w + turn * kRows + p.row;
    const float* sA = s_A + turn * kRows + p.row;
    Stretch upto[kSteps];            // the piece's positions up to each (kWarpGate: A is sA's)
    Stretch mine = {1.0f, 0.0f};
    auto first_run = [&](auto plain) {
      constexpr bool kPlain = decltype(plain)::value;
      mine = {1.0f, 0.0f};
#pragma unroll
      for (int k0 = 0; k0 < kSteps; k0 += 2) {
        Gate gates[2];
        float a[2];
        if (kWarpGate) {
          Weights w[2];
          weighed(sw, k0, w[0], w[1]);
#pragma unroll
          for (int e = 0; e < 2; ++e) gates[e] = gate_of(w[e]);
        } else {
          float g[2];
          Halves w[2];
#pragma unroll
          for (int k = 0; k < 2; ++k)            // past the end: keep the state
            g[k] = kPlain || k0 + k < p.left ? sg[(k0 + k) * stride] : INFINITY;
          halves2(g[0], g[1], w[0], w[1]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            gates[e] = gate_of(g[e], w[e]);
            a[e] = weights_of(g[e], w[e]).a;
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int k = k0 + e;
          if (!kPlain && (cut >> k & 1)) mine = {-0.0f, 0.0f};
          const float now = kPlain || k < p.left ? sx[k * 32] : 0.f;
          mine.b = kPlain ? mix(gates[e], mine.b, now) : mix_any(gates[e], mine.b, now);
          if (!kWarpGate) mine.A *= a[e];
          upto[k] = mine;
        }
      }
      if (kWarpGate && kPlain) mine.A = sA[kSteps - 1];
      if (kWarpGate && !kPlain) mine.A = cut ? -0.0f : sA[kSteps - 1];
    };
    if (whole) first_run(Yes{});
    if (__any_sync(0xffffffffu, !whole || !(fabsf(mine.b) < INFINITY))) first_run(No{});
    const int64_t state = (int64_t)p.b * D + p.d;
    const float v = join_tile<kSeg>(c, s, turn, p, mine, h0 && p.d < D && p.j < kSeg * kWarps ? h0[state] : 0.f, next);
    float* hp = h + ((int64_t)p.b * T + p.t0) * D + p.d;
    auto second_run = [&](auto plain) {
      constexpr bool kPlain = decltype(plain)::value;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        if (kWarpGate) {
          upto[k].A = sA[k];
          if (!kPlain && (cut & ((2u << k) - 1))) upto[k].A = -0.0f;
        }
        const float now = kPlain ? fmaf(upto[k].A, v, upto[k].b) : through(upto[k], v);
        if (kPlain || k < p.left) *hp = now;
        if (k == (kPlain ? kSteps : p.left) - 1 && p.t0 + k == T - 1) h_last[state] = now;
        hp += D;
      }
    };
    if (whole) second_run(Yes{}); else second_run(No{});
  });
}

// The same tiles with time reversed: c_t = a_t r_t (dh_t + c_{t+1}) is what
// position t hands to t - 1.  Reads dh, x, gate, h, writes dx, dgate: 24 bytes a
// position; (16, 8192, 256) takes 135 us, 5.9 TB/s of its 805 MB (138 us with documents;
// without any join 2 us less).  DG: where the gate's gradient goes -- 1: sums over the
// `per` lanes of a head (a power of two below 32; the first of them writes), 32: sums over
// the warp, one per block of 32 channels; 0: every channel's own.
template <bool kTma, int kSeg, int DG>
__global__ void __launch_bounds__(kT, kBackwardBlocks)
    recurrence_backward_kernel(float* __restrict__ dx, float* __restrict__ dg,
                               float* __restrict__ dh0,
                               const __grid_constant__ CUtensorMap map_x,
                               const __grid_constant__ CUtensorMap map_g,
                               const __grid_constant__ CUtensorMap map_d,
                               const __grid_constant__ CUtensorMap map_h, Operand x, Operand g,
                               Operand dh, Operand h, const float* __restrict__ dlast,
                               const float* __restrict__ h0, const uint32_t* __restrict__ reset,
                               int T, int D, Chain c) {
  extern __shared__ float s_raw[];
  __shared__ Joint s;
  float *s_x = aligned_smem(s_raw), *s_d = s_x + kTile, *s_h = s_d + kTile, *s_g = s_h + kTile;
  // kWarpGate, by turns: the weights of a tile's positions
  constexpr int kRows = kWarps * kSteps;
  float2* s_w = reinterpret_cast<float2*>(s_g);
  constexpr bool kWarpGate = DG == 32;
  float gate = 0.f;                 // kWarpGate: of this thread's position of the next tile
  const bool own_gate = !kWarpGate && c.per.d == 1;
  const unsigned box = (blockDim.x >> 5) * kSteps * 32 * sizeof(float);
  auto fetch = [&](const Place& p) {
    if (kTma && threadIdx.x == 0) {
      const int t0 = p.t0 - p.row;
      mbar_arrive_expect_tx(&s.full, own_gate ? 4 * box : 3 * box);
      tma_load_3d(smem_u32(s_x), &map_x, &s.full, p.d, t0, p.b);
      tma_load_3d(smem_u32(s_d), &map_d, &s.full, p.d, t0, p.b);
      tma_load_3d(smem_u32(s_h), &map_h, &s.full, p.d, t0 - 1, p.b);
      if (own_gate) tma_load_3d(smem_u32(s_g), &map_g, &s.full, p.d, t0, p.b);
    }
    if (!kTma) {
      copy_piece(s_x, x, p, 0, T, D);
      copy_piece(s_d, dh, p, 0, T, D);
      copy_piece(s_h, h, p, 1, T, D);
      if (own_gate) copy_piece(s_g, g, p, 0, T, D);
    }
    if (kWarpGate) gate = warp_gate(g, c, p, T);
    else if (!own_gate) copy_gates(s_g, g, c, p, T, D);
    if (!kTma || !(kWarpGate || own_gate)) copies_arrive(&s.full);
  };
  auto ready = [&](int turn) {
    if (kWarpGate) weigh(s_w + turn * kRows, nullptr, gate, &s.full);
  };
  const unsigned arrivals = (kTma ? 1 : 0) + (!kTma || !(kWarpGate || own_gate) ? blockDim.x : 0) +
                            (kWarpGate ? blockDim.x / 2 : 0);
  const int lanes = DG == 1 ? c.per.d : DG == 32 ? 32 : 1, heads = DG == 0 ? D : D / lanes;
  through_tiles<true>(c, s, arrivals, reset, T, D, fetch, ready, [&](const Place& p, unsigned cut,
                                                                     int turn, auto next) {
    const bool whole = __all_sync(0xffffffffu, p.left == kSteps && cut == 0 && p.t0 > 0);
    const int stride = own_gate ? 32 : c.gates, at = p.row * 32 + (threadIdx.x & 31);
    const float* sg = s_g + p.row * stride +
                      (own_gate ? (int)(threadIdx.x & 31)
                                : (int)c.per(min(p.d, D - 1)) - first_gate(c, p));
    const int64_t state = (int64_t)p.b * D + p.d;
    const float2* sw = s_w + turn * kRows + p.row;
    // the total gradient from a zero carry, the weights, dgate per unit of the total
    float G[kSteps], gates[kSteps], u[kSteps];
    Stretch mine = {1.0f, 0.0f};
    auto first_run = [&](auto plain) {
      constexpr bool kPlain = decltype(plain)::value;
#pragma unroll
      for (int k0 = kSteps - 2; k0 >= 0; k0 -= 2) {
        float slope[2];
        Weights w[2];
        if (kWarpGate) {
          weighed(sw, k0, w[0], w[1]);
        } else {
          float g[2];
          Halves half[2];
#pragma unroll
          for (int k = 0; k < 2; ++k)
            g[k] = kPlain || k0 + k < p.left ? sg[(k0 + k) * stride] : INFINITY;
          halves2(g[0], g[1], half[0], half[1]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            w[e] = weights_of(g[e], half[e]);
            gates[k0 + e] = pack(g[e], half[e]);
          }
        }
        mul2(slope[0], slope[1], w[0].a, w[1].a, w[0].z, w[1].z);    // d a / d gate
#pragma unroll
        for (int e = 1; e >= 0; --e) {
          const int k = k0 + e;
          const bool here = kPlain || k < p.left;
          float before = s_h[at + k * 32];
          if (!kPlain && p.t0 + k == 0) before = h0 && here ? h0[state] : 0.f;
          if (!kPlain && (cut >> k & 1)) before = 0.f;
          u[k] = (before - s_x[at + k * 32]) * slope[e];
          G[k] = mine.b + (here ? s_d[at + k * 32] : 0.f);
          mine.b = w[e].a * G[k];
          mine.A *= w[e].a;
          if (!kPlain && (cut >> k & 1)) mine = {-0.0f, 0.0f};
        }
      }
    };
    if (whole) first_run(Yes{}); else first_run(No{});
    const float v = join_tile<kSeg>(c, s, turn, p, mine, dlast && p.d < D && p.j < kSeg * kWarps ? dlast[state] : 0.f,
                        next);
    const int64_t last = (int64_t)p.b * T + p.t0 + kSteps - 1;
    float* xo = dx + last * D + p.d;
    float* go = DG == 0 ? dg + last * D + p.d : nullptr;
    // What the join gives reaches position k through the weights after it.  They are
    // good to a few ulp of themselves here too: where the only gradient comes from later
    // positions (that of the last state, say), all there is goes through them.
    float carried = v;
    auto second_run = [&](auto plain) {
      constexpr bool kPlain = decltype(plain)::value;
#pragma unroll
      for (int k = kSteps - 1; k >= 0; --k) {
        Weights w;
        if (kWarpGate) {
          const float2 both = sw[k];
          w = {both.x, both.y};
        } else {
          w = unpack(gates[k]);
        }
        const float total = G[k] + carried;
        if (kPlain || k < p.left) *xo = w.z * total;
        u[k] *= total;
        if (DG == 0 && (kPlain || k < p.left)) *go = u[k];
        carried *= w.a;
        if (!kPlain && (cut >> k & 1)) carried = 0.f;
        xo -= D;
        if (DG == 0) go -= D;
      }
    };
    if (whole) second_run(Yes{}); else second_run(No{});
    if (DG == 1) {
      // 16 sums over the lanes of a head: every exchange halves the sums that a lane
      // still carries (14 exchanges over 8 lanes where one sum at a time takes 48);
      // positions past the end are 0, their weight z a being so
      const int lane = threadIdx.x & 31;
      int first = 0, n_mine = kSteps;          // the lane's positions
#pragma unroll
      for (int n = kSteps / 2, step = 1; n > 0; n >>= 1, ++step) {
        const int o = lanes >> step;
        if (o == 0) break;
        const bool upper = lane & o;
#pragma unroll
        for (int k = 0; k < n; ++k) {
          const float keep = upper ? u[k + n] : u[k], send = upper ? u[k] : u[k + n];
          u[k] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
        first += upper ? n : 0;
        n_mine = n;
      }
      float* out = dg + ((int64_t)p.b * T + p.t0 + first) * heads + p.d / lanes;
#pragma unroll
      for (int k = 0; k < kSteps / 2; ++k) {
        if (k < n_mine && first + k < p.left) *out = u[k];
        out += heads;
      }
    }
    if (DG == 32) {
      // the same over the whole warp: 16 exchanges where one sum at a time takes 80
      const int lane = threadIdx.x & 31;
#pragma unroll
      for (int n = kSteps / 2, o = 16; n > 0; n >>= 1, o >>= 1)
#pragma unroll
        for (int k = 0; k < n; ++k) {
          const bool upper = lane & o;
          const float keep = upper ? u[k + n] : u[k], send = upper ? u[k] : u[k + n];
          u[k] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      const float sum = u[0] + __shfl_xor_sync(0xffffffffu, u[0], 1);
      const int k = lane >> 1, left = __shfl_sync(0xffffffffu, p.left, 0);
      if ((lane & 1) == 0 && k < left)
        dg[((int64_t)p.b * T + p.t0 + k) * heads + (p.d - lane) / 32] = sum;
    }
    if (dh0 && p.left && p.t0 == 0) dh0[state] = mine.b + carried;
  });
}

// out[i] = the sum of in[i parts .. (i + 1) parts - 1], in that order.
__global__ void sum_parts_kernel(float* __restrict__ out, const float* __restrict__ in, int64_t n,
                                 int parts) {
  for (int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x; i < n; i += (int64_t)gridDim.x * kT) {
    const float* p = in + i * parts;
    float v = p[0];
    for (int k = 1; k < parts; ++k) v += p[k];
    out[i] = v;
  }
}

// The same for many parts: a warp has an output.  Backward over (4, 4096, 1000) with a
// thread and with a warp an output: 87 and 96 us with 50 parts, 93 and 84 with 100, 90 and
// 75 with 250, 150 and 77 with 1000; over (1, 1024, 1000) 17 and 13 us with 100, 24 and 12
// with 250.
constexpr int kManyParts = 100;
__global__ void sum_many_parts_kernel(float* __restrict__ out, const float* __restrict__ in,
                                      int64_t n, int parts) {
  const int lane = threadIdx.x & 31, warps = kT / 32;
  for (int64_t i = (int64_t)blockIdx.x * warps + (threadIdx.x >> 5); i < n;
       i += (int64_t)gridDim.x * warps) {
    float v = 0.f;
    for (int k = lane; k < parts; k += 32) v += in[i * parts + k];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) out[i] = v;
  }
}

// One position: 16 bytes a channel; (32, 1024) takes 3 us, a launch's own time.
__global__ void recurrence_step_kernel(float* __restrict__ state, const float* __restrict__ x,
                                       int64_t x_ld, const float* __restrict__ g, int64_t g_ld,
                                       int64_t n, unsigned D, unsigned per) {
  for (int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * kT) {
    const unsigned b = (unsigned)i / D, d = (unsigned)i - b * D;
    const float gate = g[b * g_ld + d / per];
    Halves w, same;
    halves2(gate, gate, w, same);
    state[i] = mix_any(gate_of(gate, w), state[i], x[b * x_ld + d]);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 get_encode_scan() {
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

// A map of boxes of 32 channels by `steps` positions over an operand, where the
// copy engine takes it: 16-byte aligned base and strides, time inside batch.
bool encode_operand(CUtensorMap* map, const Operand& o, int64_t B, int64_t T, int64_t D,
                    unsigned steps) {
  auto enc = get_encode_scan();
  const int64_t bs = B > 1 ? o.bs : T * o.ts;
  if (!enc || (reinterpret_cast<uintptr_t>(o.p) & 15) || o.ts % 4 || bs % 4 || o.ts < D ||
      bs < T * o.ts || bs >= (int64_t(1) << 37))
    return false;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)T, (cuuint64_t)B};
  cuuint64_t strides[2] = {(cuuint64_t)o.ts * 4, (cuuint64_t)bs * 4};
  cuuint32_t box[3] = {32, steps, 1}, ones[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float*>(o.p), dims, strides, box,
             ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int check_sizes(const char* what, int64_t B, int64_t T, int64_t D, int64_t H) {
  WXX_REQUIRE(B >= 0 && T >= 0 && D >= 0 && H >= 0, "%s: negative size", what);
  WXX_REQUIRE(D == 0 || (H > 0 && D % H == 0), "%s: %lld channels are not a multiple of %lld heads",
              what, (long long)D, (long long)H);
  // positions, channels and rows are numbered in 32 bits (offsets are not)
  WXX_REQUIRE(B < (int64_t(1) << 31) && T < (int64_t(1) << 31) - 256 &&
                  D < (int64_t(1) << 31) - 32 && B * D < (int64_t(1) << 31),
              "%s: time or batch times channels is 2^31 or more", what);
  return WXX_OK;
}

// Tiles of a group.  Looking at more tiles costs every tile, a hop between groups
// (about 1.5 us) costs the row.  The rows are joined side by side, so the hops of
// groups of 8 are hidden where the tiles of 8 positions of all rows take longer than
// one: from about 24 blocks of 32 channels.  Forward in groups of 8 against 32: 72 and
// 53 us with 8 blocks of 512 tiles, 40 and 39 us with 16 of 192, 46 and 47 us with 32 of
// 128, 78 and 84 us with 128 of 64.
constexpr int kShortSeg = 1, kLongSeg = 4;
bool long_rows(const Chain& c) { return c.blocks.d < 24; }
int group_tiles(const Chain& c) { return kWarps * (long_rows(c) ? kLongSeg : kShortSeg); }

// Held from the choice of a scan's scratch to its launch: another host thread's
// larger scan would free the scratch in between.
std::mutex g_scan;

// Scratch of at least `bytes` (under g_scan).  Each stream keeps its own, zero when it
// is new, so scans on two streams do not meet; streams are told apart by their id,
// which no later stream has again, as it may a handle.  A recorded launch may be
// replayed beside either, so it has scratch of its own in the recording, cleared
// before it; so has a launch on a stream past the sixteenth.  *own is such scratch,
// for the caller to free.
int scan_scratch(size_t bytes, char** p, void** own) {
  struct Kept {
    unsigned long long stream;
    char* p;
    size_t size;
  };
  static Kept kept[16];
  static int n = 0;
  cudaStream_t stream = wxx::stream();
  *own = nullptr;
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  WXX_CUDA_CHECK(cudaStreamIsCapturing(stream, &cs));
  Kept* mine = nullptr;
  if (cs == cudaStreamCaptureStatusNone) {
    unsigned long long id = 0;
    WXX_CUDA_CHECK(cudaStreamGetId(stream, &id));
    for (int i = 0; i < n && !mine; ++i)
      if (kept[i].stream == id) mine = &kept[i];
    if (!mine && n < 16) {
      mine = &kept[n++];
      *mine = {id, nullptr, 0};
    }
  }
  if (!mine) {
    if (int st = wxx_malloc(own, bytes)) return st;
    *p = static_cast<char*>(*own);
    cudaError_t e = cudaMemsetAsync(*p, 0, bytes, stream);
    if (e == cudaSuccess) return WXX_OK;
    wxx_free(*own);
    *own = nullptr;
    wxx::set_error("clearing a scan's scratch failed: %s", cudaGetErrorString(e));
    return WXX_E_CUDA;
  }
  if (mine->size < bytes) {
    size_t size = 1 << 20;
    while (size < bytes) size <<= 1;
    char* old = mine->p;
    mine->p = nullptr;
    mine->size = 0;
    if (old) WXX_CUDA_CHECK(cudaFreeAsync(old, stream));
    char* fresh = nullptr;
    WXX_CUDA_CHECK(cudaMallocAsync(reinterpret_cast<void**>(&fresh), size, stream));
    cudaError_t e = cudaMemsetAsync(fresh, 0, size, stream);
    if (e != cudaSuccess) {
      cudaFreeAsync(fresh, stream);
      wxx::set_error("clearing a scan's scratch failed: %s", cudaGetErrorString(e));
      return WXX_E_CUDA;
    }
    mine->p = fresh;
    mine->size = size;
  }
  *p = mine->p;
  return WXX_OK;
}

unsigned scan_grid(const Chain& c, int resident) {
  const unsigned most = (unsigned)(wxx::num_sms() * resident);
  return c.total < most ? c.total : most;
}

// Threads and tiles of a scan, and its scratch (*own is freed by the caller).
int plan_scan(const char* what, int64_t B, int64_t T, int64_t D, int64_t H, Chain& c,
              unsigned& threads, void** own) {
  const int64_t pieces = (T + kSteps - 1) / kSteps;
  const int64_t warps = pieces < kWarps ? pieces : kWarps;
  c = Chain{};
  c.tiles = (int)((pieces + warps - 1) / warps);
  c.row_blocks = Divider::of((unsigned)((D + 31) / 32));
  c.per = Divider::of((unsigned)(D / H));
  c.gates = c.per.d >= 32 ? 2 : 31 / c.per.d + 2;
  c.err = wxx::device_error_word();
  *own = nullptr;
  threads = (unsigned)(warps * 32);
  const int64_t blocks = B * c.row_blocks.d, total = blocks * c.tiles;
  WXX_REQUIRE(total < (int64_t(1) << 31), "%s: too many elements", what);
  c.blocks = Divider::of((unsigned)blocks);
  c.total = (unsigned)total;
  if (c.tiles == 1) return WXX_OK;
  const int64_t size = group_tiles(c), groups = (c.tiles + size - 1) / size;
  const size_t tile_bytes = (size_t)total * 32 * sizeof(ulonglong2);
  char* p;
  if (int st = scan_scratch(256 + tile_bytes + (size_t)(blocks * groups) * 32 * 8, &p, own))
    return st;
  c.counters = reinterpret_cast<Counters*>(p);
  c.tile = reinterpret_cast<ulonglong2*>(p + 256);
  c.group = reinterpret_cast<unsigned long long*>(p + 256 + tile_bytes);
  return WXX_OK;
}

// Room for the kernel's tiles, asked for once for each kernel.
template <class K>
int allow_smem(K kernel, int bytes) {
  static K done[16] = {};           // kernels of this type that have it
  for (K& k : done) {
    if (k == kernel) return WXX_OK;
    if (k) continue;
    WXX_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    k = kernel;
    return WXX_OK;
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
  const Operand ox = operand(x, x_bs, x_ts, D), og = operand(gate, g_bs, g_ts, H);
  std::lock_guard<std::mutex> lock(g_scan);
  Chain c;
  unsigned threads;
  void* scratch;
  if (int st = plan_scan("wxx_gated_recurrence", B, T, D, H, c, threads, &scratch)) return st;
  constexpr int kBytes = 2 * kTile * sizeof(float) + 128;
  CUtensorMap mx{}, mg{};
  const unsigned steps = threads / 32 * kSteps;
  const bool tma = encode_operand(&mx, ox, B, T, D, steps) &&
                   (c.per.d > 1 || encode_operand(&mg, og, B, T, D, steps));
  auto launch = [&](auto kernel, int resident) {
    if (int st = allow_smem(kernel, kBytes)) return st;
    kernel<<<scan_grid(c, resident), threads, kBytes, wxx::stream()>>>(
        h, h_last, mx, mg, ox, og, h0, reset, (int)T, (int)D, c);
    return wxx::after_launch(__FILE__, __LINE__);
  };
  auto pick = [&](auto t, auto seg) {
    constexpr bool kTma = decltype(t)::value;
    constexpr int kSeg = decltype(seg)::value ? kLongSeg : kShortSeg;
    constexpr int kBlocks = forward_blocks(kTma, kSeg);
    return c.per.d % 32 == 0 ? launch(recurrence_forward_kernel<kTma, kSeg, true>, kBlocks)
                             : launch(recurrence_forward_kernel<kTma, kSeg, false>, kBlocks);
  };
  const int st = long_rows(c) ? (tma ? pick(Yes{}, Yes{}) : pick(No{}, Yes{}))
                              : (tma ? pick(Yes{}, No{}) : pick(No{}, No{}));
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
  if (B * D == 0) {                   // a gate of no channels: the sum over none
    if (B * T * H > 0)
      WXX_CUDA_CHECK(cudaMemsetAsync(dgate, 0, (size_t)(B * T * H) * sizeof(float),
                                     wxx::stream()));
    return WXX_OK;
  }
  if (T == 0) return dh0 ? copy_state(dh0, dlast, B * D) : WXX_OK;
  // The gate's gradient is summed over a head's channels in the kernel where
  // they lie in one warp's 32 neighbours, by partial sums per 32 channels where
  // they are several warps', and from every channel's own otherwise.
  const int64_t per = D / H;
  const bool warp = per % 32 == 0, lanes = per < 32 && (per & (per - 1)) == 0;
  const bool inside = lanes || per == 32;
  const int64_t parts = warp ? per / 32 : per;
  const Operand ox = operand(x, x_bs, x_ts, D), og = operand(gate, g_bs, g_ts, H),
                od = operand(dh, T * D, D, D), oh = operand(h, T * D, D, D);
  std::lock_guard<std::mutex> lock(g_scan);
  Chain c;
  unsigned threads;
  void *scratch = nullptr, *wide = nullptr;
  float* sums = dgate;
  if (!inside) {
    if (int st = wxx_malloc(&wide, (uint64_t)(B * T * H * parts) * sizeof(float))) return st;
    sums = static_cast<float*>(wide);
  }
  int st = plan_scan("wxx_gated_recurrence_backward", B, T, D, H, c, threads, &scratch);
  if (st == WXX_OK) {
    constexpr int kBytes = 4 * kTile * sizeof(float) + 128;
    CUtensorMap mx{}, mg{}, md{}, mh{};
    const unsigned steps = threads / 32 * kSteps;
    const bool tma = encode_operand(&mx, ox, B, T, D, steps) &&
                     encode_operand(&md, od, B, T, D, steps) &&
                     encode_operand(&mh, oh, B, T, D, steps) &&
                     (c.per.d > 1 || encode_operand(&mg, og, B, T, D, steps));
    auto launch = [&](auto kernel) {
      if (int e = allow_smem(kernel, kBytes)) return e;
      kernel<<<scan_grid(c, kBackwardBlocks), threads, kBytes, wxx::stream()>>>(
          dx, sums, dh0, mx, mg, md, mh, ox, og, od, oh, dlast, h0, reset, (int)T, (int)D, c);
      return wxx::after_launch(__FILE__, __LINE__);
    };
    auto pick = [&](auto t, auto seg) {
      constexpr bool kTma = decltype(t)::value;
      constexpr int kSeg = decltype(seg)::value ? kLongSeg : kShortSeg;
      return warp                  ? launch(recurrence_backward_kernel<kTma, kSeg, 32>)
             : lanes && per > 1    ? launch(recurrence_backward_kernel<kTma, kSeg, 1>)
                                   : launch(recurrence_backward_kernel<kTma, kSeg, 0>);
    };
    st = long_rows(c) ? (tma ? pick(Yes{}, Yes{}) : pick(No{}, Yes{}))
                      : (tma ? pick(Yes{}, No{}) : pick(No{}, No{}));
    if (st == WXX_OK && wide) {
      const int64_t n = B * T * H;
      if (parts < kManyParts)
        sum_parts_kernel<<<wxx::grid_for(n, kT), kT, 0, wxx::stream()>>>(dgate, sums, n,
                                                                         (int)parts);
      else
        sum_many_parts_kernel<<<wxx::grid_for(n, kT / 32), kT, 0, wxx::stream()>>>(dgate, sums, n,
                                                                                   (int)parts);
      st = wxx::after_launch(__FILE__, __LINE__);
    }
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
  recurrence_step_kernel<<<wxx::grid_for(n, kT), kT, 0, wxx::stream()>>>(
      state, x, x_ld, gate, g_ld, n, (unsigned)D, (unsigned)(D / H));
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}
