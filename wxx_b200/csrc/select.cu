// Selection over logits: the k largest of each row, and one step of beam
// search (selection over beams and vocabulary, and the reordering of the
// beams' states in place).
//
// Order.  Values are compared as numbers (-0 equals +0), equal values by the
// lower index first.  wxx_topk puts NaN above every number; beam search gives
// a beam whose log-probabilities are NaN the score -inf.

#include <cuda_runtime.h>
#include <cooperative_groups.h>
#include <stdint.h>

#include <type_traits>

#include "common.cuh"

namespace {

constexpr int kT = 256;
constexpr int kMaxTopk = 256;
constexpr int kMaxBeams = 16;
constexpr int kMaxStates = 128;
constexpr int kCandidates = 2048;     // of a row, in shared memory
constexpr int kClusterBlocks = 8;     // blocks that share a batch item's rows

// The order-preserving bits of a value (-0 counts as +0); nan_key is what a NaN
// counts as.
constexpr uint32_t kNanHighest = 0xfffffffeu;            // above +inf
constexpr uint32_t kNanLowest = 0x007fffffu;             // the key of -inf
__device__ __forceinline__ uint32_t value_key(float v, uint32_t nan_key) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  const uint32_t k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return v != v ? nan_key : k;
}
// A (value, index) pair as one number that is larger for the better pair: the
// value's key above the inverted index.  0 is below every pair.
__device__ __forceinline__ uint64_t pair_key(float v, uint32_t i, uint32_t nan_key) {
  return ((uint64_t)value_key(v, nan_key) << 32) | (uint32_t)~i;
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return ~(uint32_t)k; }

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

struct Select {                       // shared memory of a row's selection
  uint64_t pair[kCandidates];
  unsigned hist[256];
  float tau[32];
  float sum[32], top[32];
  unsigned count, digit, rest;
};

// A row split over THREADS threads: 16-byte groups in the aligned middle, thread
// t taking groups t, t + THREADS, ..., and up to six single entries at its ends,
// one each for the first threads.
struct Row {
  const float* p;
  const float4* mid;
  int V, head, groups, single;        // single: this thread's single entry, -1 for none
  __device__ Row(const float* row, int n) : p(row), V(n) {
    head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / 4);
    groups = (n - head) / 4;
    mid = reinterpret_cast<const float4*>(row + head);
    const int tail = n - head - 4 * groups, t = threadIdx.x;
    single = t < head ? t : t < head + tail ? n - tail + (t - head) : -1;
  }
  template <int THREADS, class F>
  __device__ __forceinline__ void each(F f) const {
    if (single >= 0) f(p[single], single);
    for (int i = threadIdx.x; i < groups; i += THREADS) {
      const float4 v = mid[i];
      const int at = head + 4 * i;
      f(v.x, at);
      f(v.y, at + 1);
      f(v.z, at + 2);
      f(v.w, at + 3);
    }
  }
};

// The r-th largest (from 1) of key(entry) over the row's entries that `among`
// lets in, by 8-bit digits from the top; rest: how many of the entries equal to it
// are needed to make up r.
template <int THREADS, class Key, class Among>
__device__ uint32_t nth_key(const Row& row, Select& s, unsigned r, unsigned& rest, Key key,
                            Among among) {
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += THREADS) s.hist[i] = 0;
    __syncthreads();
    row.each<THREADS>([&](float v, int i) {
      const uint32_t k = key(v, i);
      if (among(v, i) && (k & mask) == prefix) atomicAdd(&s.hist[k >> shift & 255u], 1u);
    });
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned above = 0;
      int d = 255;
      while (d > 0 && above + s.hist[d] < r) above += s.hist[d--];
      s.digit = d;
      s.rest = r - above;
    }
    __syncthreads();
    prefix |= s.digit << shift;
    mask |= 255u << shift;
    r = s.rest;
    __syncthreads();
  }
  rest = r;
  return prefix;
}

// Puts the row's K best pairs, and perhaps more of its best, into s.pair and
// returns how many (K <= V).  With SUM, top and sum come to hold the row's largest
// number and the sum of exp(v - top).
//
// One pass over the row gives every thread its largest entry.  The ceil(K / warps)
// th largest of a warp's, the smallest of that over the warps, is a value that at
// least K entries reach, and few more do: about 3 K of 50304 at K = 64 and 32
// warps.  The threads whose largest reaches it read their entries again (from
// L2) and keep those that do.  Where too many do (long runs of one value, or large
// ones crowded into a few threads), the exact K-th pair is found digit by digit.
template <int THREADS, uint32_t NAN_KEY, bool SUM>
__device__ int best_pairs(const Row& row, int K, Select& s, float& top, float& sum) {
  constexpr int kWarps = THREADS / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float m = row.single >= 0 ? row.p[row.single] : -INFINITY;
  if (NAN_KEY == kNanLowest && m != m) m = -INFINITY;
  float part = 0.f;
  if (SUM && row.single >= 0 && row.p[row.single] != -INFINITY) part = expf(row.p[row.single] - m);
  auto larger = [](float a, float b) {
    return NAN_KEY == kNanHighest ? max_nan(a, b) : fmaxf(a, b);
  };
#pragma unroll 4
  for (int i = threadIdx.x; i < row.groups; i += THREADS) {
    const float4 v = row.mid[i];
    const float n = larger(larger(m, v.x), larger(larger(v.y, v.z), v.w));
    if (SUM && n != -INFINITY) {
      if (n > m) part *= fast_exp2((m - n) * 1.4426950408889634f);
      part += (fast_exp2((v.x - n) * 1.4426950408889634f) +
               fast_exp2((v.y - n) * 1.4426950408889634f)) +
              (fast_exp2((v.z - n) * 1.4426950408889634f) +
               fast_exp2((v.w - n) * 1.4426950408889634f));
    } else if (SUM) {
      part += (v.x + v.y) + (v.z + v.w) == -INFINITY ? 0.f : NAN;   // nothing but -inf, or NaN
    }
    m = n;
  }
  // the warp's lanes in descending order of their largest entries
  float o = m != m ? INFINITY : m;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, o, j);
      const bool first = (lane & j) == 0, down = (lane & k) == 0;
      o = first == down ? fmaxf(o, other) : fminf(o, other);
    }
  const float reach = __shfl_sync(0xffffffffu, o, (K + kWarps - 1) / kWarps - 1);
  if (SUM) {
    const float w = __shfl_sync(0xffffffffu, o, 0);
    part *= m == -INFINITY || m == w ? 1.0f : expf(m - w);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) part += __shfl_xor_sync(0xffffffffu, part, k);
    if (lane == 0) {
      s.top[warp] = w;
      s.sum[warp] = part;
    }
  }
  if (lane == 0) s.tau[warp] = reach;
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  float tau = INFINITY;
  for (int w = 0; w < kWarps; ++w) tau = fminf(tau, s.tau[w]);
  if (SUM) {
    top = -INFINITY;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s.top[w]);
    sum = 0.f;
    for (int w = 0; w < kWarps; ++w)
      sum += s.top[w] == top ? s.sum[w] : s.sum[w] * expf(s.top[w] - top);
  }
  auto keep = [&](float v, int i) {
    const unsigned at = atomicAdd(&s.count, 1u);
    if (at < kCandidates) s.pair[at] = pair_key(v, i, NAN_KEY);
  };
  // all pairs of a short row, else those that reach tau (NaN counts as reaching
  // where it is the highest; where it is the lowest, tau = -inf is left to the
  // digits, which know where it stands)
  const bool all = row.V <= kCandidates && tau == -INFINITY;
  const bool plain = all || tau > -INFINITY || NAN_KEY == kNanHighest;
  if (plain && (all || !(m < tau)))
    row.each<THREADS>([&](float v, int i) {
      if (all || (NAN_KEY == kNanHighest ? !(v < tau) : v >= tau)) keep(v, i);
    });
  __syncthreads();
  const unsigned n = s.count;
  if (plain && n <= kCandidates) return (int)n;
  __syncthreads();
  unsigned rest, none;
  const uint32_t cut = nth_key<THREADS>(
      row, s, K, rest, [](float v, int) { return value_key(v, NAN_KEY); },
      [](float, int) { return true; });
  const uint32_t last = ~nth_key<THREADS>(
      row, s, rest, none, [](float, int i) { return ~(uint32_t)i; },
      [&](float v, int) { return value_key(v, NAN_KEY) == cut; });
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  row.each<THREADS>([&](float v, int i) {
    const uint32_t k = value_key(v, NAN_KEY);
    if (k > cut || (k == cut && (uint32_t)i <= last)) keep(v, i);
  });
  __syncthreads();
  return K;
}

// Calls put(rank, pair) for the K best of the n pairs in s.pair (all different).
// Up to 256 of them are counted against each other; more are sorted, a pair a
// thread, where there are threads for that.
template <int THREADS, class F>
__device__ void in_order(Select& s, int n, int K, F put) {
  const int t = threadIdx.x;
  if (n <= 256 || n > THREADS) {
    for (int i = t; i < n; i += THREADS) {
      const uint64_t mine = s.pair[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += s.pair[j] > mine;
      if (rank < K) put(rank, mine);
    }
    return;
  }
  int size = 512;
  while (size < n) size <<= 1;
  uint64_t mine = t < n ? s.pair[t] : 0;
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      uint64_t other;
      if (j >= 32) {
        __syncthreads();
        if (t < size) s.pair[t] = mine;
        __syncthreads();
        other = t < size ? s.pair[t ^ j] : 0;
      } else {
        other = __shfl_xor_sync(0xffffffffu, mine, j);
      }
      const bool first = (t & j) == 0, down = (t & k) == 0;
      mine = (first == down) == (mine > other) ? mine : other;
    }
  if (t < K) put(t, mine);
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS, 2048 / THREADS)
    topk_kernel(float* __restrict__ values, uint32_t* __restrict__ ids,
                const float* __restrict__ x, int64_t ld, int V, int K) {
  __shared__ Select s;
  const int64_t at = blockIdx.x;
  const Row row(x + at * ld, V);
  float top, sum;
  const int n = best_pairs<THREADS, kNanHighest, false>(row, K, s, top, sum);
  in_order<THREADS>(s, n, K, [&](int rank, uint64_t pair) {
    const uint32_t i = key_index(pair);
    ids[at * K + rank] = i;
    values[at * K + rank] = row.p[i];
  });
}

// One selection step.  A cluster takes a batch item; its rows, or `parts` pieces
// of each where there are few, go to its blocks in turn.  Each leaves the piece's
// best W pairs, its largest logit and its sum of exponentials in shared memory,
// and the first block merges them all:
//   score = scores[w] + ((z - top_w) - log sum_w)
struct Piece {
  uint64_t pair[kMaxBeams];           // 0: no pair
  float top, sum;
};
struct Merge {
  Select s;
  Piece piece[2];                     // pieces rank, rank + blocks
  uint64_t first[kMaxBeams * kMaxBeams], second[kMaxBeams * kMaxBeams];
  float top[kMaxBeams], log_sum[kMaxBeams];
};

template <int THREADS>
__global__ void __launch_bounds__(THREADS)
    beam_select_kernel(float* __restrict__ new_scores, uint32_t* __restrict__ parents,
                       uint32_t* __restrict__ new_tokens, uint32_t* __restrict__ new_finished,
                       const float* __restrict__ logits, int64_t ld,
                       const float* __restrict__ scores, const uint32_t* __restrict__ finished,
                       int W, int V, int parts, uint32_t stop) {
  __shared__ Merge s;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), blocks = cluster.num_blocks();
  const int64_t b = blockIdx.x / blocks;
  const int t = threadIdx.x, pieces = W * parts;
  // a piece's length, a multiple of 4 so that all start where the first does
  const int length = parts == 1 ? V : ((V + parts - 1) / parts + 3) / 4 * 4;
  for (int q = rank, turn = 0; q < pieces; q += blocks, ++turn) {
    Piece& piece = s.piece[turn];
    const int w = q / parts, from = (q - w * parts) * length;
    const int n = min(length, V - from), K = min(W, n);
    if (t < W) piece.pair[t] = 0;
    __syncthreads();
    if (finished && finished[b * W + w]) continue;
    const Row row(logits + (b * W + w) * ld + from, n);
    float top, sum;
    const int found = best_pairs<THREADS, kNanLowest, true>(row, K, s.s, top, sum);
    in_order<THREADS>(s.s, found, K, [&](int r, uint64_t pair) {
      piece.pair[r] = pair - (uint32_t)from;        // the inverted index of the row
    });
    if (t == 0) {
      piece.top = top;
      piece.sum = sum;
    }
    __syncthreads();
  }
  cluster.sync();
  if (rank == 0) {
    auto piece_of = [&](int q) -> const Piece* {
      return cluster.map_shared_rank(&s.piece[q / blocks], q % blocks);
    };
    if (t < W) {
      float top = -INFINITY, sum = 0.f;
      if (!(finished && finished[b * W + t])) {
        for (int k = 0; k < parts; ++k) top = fmaxf(top, piece_of(t * parts + k)->top);
        for (int k = 0; k < parts; ++k) {
          const Piece* p = piece_of(t * parts + k);
          sum += p->top == top ? p->sum : p->sum * expf(p->top - top);
        }
      }
      s.top[t] = top;
      s.log_sum[t] = logf(sum);
    }
    __syncthreads();
    // Every beam's W best pairs of all its pieces compete: by score, then the lower
    // beam, then the better pair of it.
    const int n = pieces * W;
    for (int i = t; i < n; i += THREADS) {
      const int q = i / W, r = i - q * W, w = q / parts;
      const float score = scores[b * W + w];
      uint64_t pair = piece_of(q)->pair[r];
      float c = -INFINITY;
      if (finished && finished[b * W + w]) {
        if (q == w * parts && r == 0) {
          c = score;
          pair = 1;
        }
      } else if (pair) {
        const float z = logits[(b * W + w) * ld + key_index(pair)];
        c = score + ((z - s.top[w]) - s.log_sum[w]);
      }
      s.first[i] = (uint64_t)value_key(c, kNanLowest) << 32 | (uint32_t)(kMaxBeams - w);
      s.second[i] = pair;
    }
    __syncthreads();
    for (int i = t; i < n; i += THREADS) {
      const uint64_t f = s.first[i], g = s.second[i];
      int place = 0;
      for (int j = 0; j < n; ++j) {
        const uint64_t fj = s.first[j], gj = s.second[j];
        place += fj > f || (fj == f && (gj > g || (gj == g && j < i)));
      }
      if (place >= W) continue;
      const int w = i / W / parts;
      const bool done = finished && finished[b * W + w];
      const uint32_t token = done ? stop : g ? key_index(g) : 0u;
      const uint32_t k = (uint32_t)(f >> 32);
      const int64_t o = b * W + place;
      new_scores[o] = __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
      parents[o] = w;
      new_tokens[o] = token;
      if (new_finished) new_finished[o] = done || token == stop;
    }
  }
  cluster.sync();                     // the pieces stay until they have been read
}

struct StateTable {
  int n;
  uint32_t* p[kMaxStates];
  int64_t row[kMaxStates];     // words of a row
  int64_t unit[kMaxStates];    // words of one position (0: the whole row moves)
};

// Every thread owns a place in the rows of a batch item: it reads it from every
// beam that someone else follows, then writes it to the followers, so the move is
// in place and a beam is read once however many follow it.  Beams that follow
// themselves are not touched.  MAX: beams, at most; four words at a time where the
// rows are 16-byte aligned.
template <int MAX>
__global__ void __launch_bounds__(kT)
    beam_reorder_kernel(const __grid_constant__ StateTable tab,
                        const uint32_t* __restrict__ parents,
                        const uint32_t* __restrict__ cur_len, int W, int* err) {
  __shared__ unsigned s_followers[MAX];
  const int64_t b = blockIdx.y;
  const int s = blockIdx.z, t = threadIdx.x;
  const int64_t row = tab.row[s];
  int64_t n = row;
  if (cur_len && tab.unit[s]) {
    const int64_t used = (int64_t)*cur_len * tab.unit[s];
    n = used < n ? used : n;
  }
  if (t < 32) {
    const uint32_t parent = t < W ? parents[b * W + t] : (uint32_t)t;
    if (t < W && parent >= (uint32_t)W) wxx_device_fail(err, WXX_DEV_ERR_BAD_INDEX);
    for (int p = 0; p < MAX; ++p) {
      const unsigned who = __ballot_sync(0xffffffffu, t < W && parent == (uint32_t)p && t != p);
      if (t == 0) s_followers[p] = who;
    }
  }
  __syncthreads();
  unsigned followers[MAX];
  unsigned any = 0;
#pragma unroll
  for (int p = 0; p < MAX; ++p) any |= followers[p] = s_followers[p];
  if (!any) return;
  uint32_t* base = tab.p[s] + b * W * row;
  auto move = [&](auto* at, int64_t step, int64_t i) {
    auto* column = at + i;
    std::remove_reference_t<decltype(*at)> v[MAX];
#pragma unroll
    for (int p = 0; p < MAX; ++p)
      if (followers[p]) v[p] = column[p * step];
#pragma unroll
    for (int p = 0; p < MAX; ++p)
      for (unsigned who = followers[p]; who; who &= who - 1)
        column[(__ffs(who) - 1) * step] = v[p];
  };
  int64_t done = 0;
  if (row % 4 == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0) {
    for (int64_t i = (int64_t)blockIdx.x * kT + t; i < n / 4; i += (int64_t)gridDim.x * kT)
      move(reinterpret_cast<uint4*>(base), row / 4, i);
    done = n / 4 * 4;
  }
  for (int64_t i = done + (int64_t)blockIdx.x * kT + t; i < n; i += (int64_t)gridDim.x * kT)
    move(base, row, i);
}

}  // namespace

// values and ids (N, K): the K largest of each row of x (N, V; row stride ld)
// in descending order.
WXX_EXPORT int wxx_topk(float* values, uint32_t* ids, const float* x, int64_t ld, int64_t N,
                        int64_t V, int K) {
  WXX_REQUIRE_INIT();
  WXX_REQUIRE(N >= 0 && N < (int64_t(1) << 31) && V >= 1 && V < (int64_t(1) << 31),
              "wxx_topk: bad sizes");
  WXX_REQUIRE(K >= 1 && K <= kMaxTopk && K <= V, "wxx_topk: k = %d outside [1, min(%lld, %d)]", K,
              (long long)V, kMaxTopk);
  if (N == 0) return WXX_OK;
  // 256 threads see a short row in a few loads; a long one, or a K that would take
  // many of each warp's entries, is worth 1024
  if (V <= 4096 && K <= 64)
    topk_kernel<256><<<(unsigned)N, 256, 0, wxx::stream()>>>(values, ids, x, ld, (int)V, K);
  else
    topk_kernel<1024><<<(unsigned)N, 1024, 0, wxx::stream()>>>(values, ids, x, ld, (int)V, K);
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}

// One selection step of beam search over logits (B W, V; row stride ld) and the
// beams' scores (B, W): new_scores, parents and tokens (B, W).  finished (B, W)
// and new_finished go together (NULL: no stop token): a finished beam is
// carried on by the stop token alone, at no cost.
WXX_EXPORT int wxx_beam_select(float* new_scores, uint32_t* parents, uint32_t* tokens,
                               uint32_t* new_finished, const float* logits, int64_t ld,
                               const float* scores, const uint32_t* finished, int64_t B, int W,
                               int64_t V, uint32_t stop) {
  WXX_REQUIRE_INIT();
  WXX_REQUIRE(W >= 1 && W <= kMaxBeams, "wxx_beam_select: %d beams outside [1, %d]", W, kMaxBeams);
  WXX_REQUIRE(B >= 0 && B * W < (int64_t(1) << 31) && V >= 1 && V < (int64_t(1) << 31),
              "wxx_beam_select: bad sizes");
  WXX_REQUIRE((finished == nullptr) == (new_finished == nullptr),
              "wxx_beam_select: finished and new_finished go together");
  if (B == 0) return WXX_OK;
  // long rows of few beams are split so that the cluster's blocks all have a piece
  const bool wide = V > 4096;
  const int parts = wide && W < kClusterBlocks ? kClusterBlocks / W : 1;
  const int blocks = W * parts < kClusterBlocks ? W * parts : kClusterBlocks;
  WXX_REQUIRE(B * blocks < (int64_t(1) << 31), "wxx_beam_select: too many rows");
  auto launch = [&](auto kernel, int threads) -> int {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * blocks));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = wxx::stream();
    cudaLaunchAttribute at = {};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim = {(unsigned)blocks, 1, 1};
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    WXX_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, new_scores, parents, tokens, new_finished,
                                      logits, ld, scores, finished, W, (int)V, parts, stop));
    WXX_LAUNCH_CHECK();
    return WXX_OK;
  };
  return wide ? launch(beam_select_kernel<1024>, 1024) : launch(beam_select_kernel<256>, 256);
}

// Moves the rows of n state tensors in place: row b W + w of each takes what
// row b W + parents[b, w] had.  state[i] (device pointers in a host array) has
// B W rows of row[i] 4-byte words; with cur_len (one device word) only the first
// *cur_len * unit[i] words of a row move (unit[i] = 0: all of them).
WXX_EXPORT int wxx_beam_reorder(int n, uint32_t* const* state, const int64_t* row,
                                const int64_t* unit, const uint32_t* parents, int64_t B, int W,
                                const uint32_t* cur_len) {
  WXX_REQUIRE_INIT();
  WXX_REQUIRE(W >= 1 && W <= kMaxBeams, "wxx_beam_reorder: %d beams outside [1, %d]", W, kMaxBeams);
  WXX_REQUIRE(n >= 0 && B >= 0 && B < 65536, "wxx_beam_reorder: bad sizes");
  if (B == 0) return WXX_OK;
  int i = 0;
  while (i < n) {
    StateTable tab;
    tab.n = 0;
    int64_t longest = 0;
    for (; i < n && tab.n < kMaxStates; ++i) {
      WXX_REQUIRE(row[i] >= 0 && unit[i] >= 0, "wxx_beam_reorder: state %d has a negative size", i);
      if (row[i] == 0) continue;
      WXX_REQUIRE(state[i] != nullptr, "wxx_beam_reorder: state %d is NULL", i);
      tab.p[tab.n] = state[i];
      tab.row[tab.n] = row[i];
      tab.unit[tab.n] = unit[i];
      ++tab.n;
      longest = longest < row[i] ? row[i] : longest;
    }
    if (tab.n == 0) continue;
    // about eight blocks an SM in all, more where a row gives each thread work
    const int64_t groups = (longest / 4 + kT - 1) / kT, rest = B * tab.n;
    int64_t blocks = (wxx::num_sms() * 32 + rest - 1) / rest;
    blocks = blocks < groups ? blocks : groups;
    const dim3 grid((unsigned)(blocks < 1 ? 1 : blocks), (unsigned)B, (unsigned)tab.n);
    auto kernel = W <= 4 ? beam_reorder_kernel<4> : W <= 8 ? beam_reorder_kernel<8>
                                                          : beam_reorder_kernel<16>;
    kernel<<<grid, kT, 0, wxx::stream()>>>(tab, parents, cur_len, W, wxx::device_error_word());
    WXX_LAUNCH_CHECK();
  }
  return WXX_OK;
}
