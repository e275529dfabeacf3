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
#include <utility>

#include "common.cuh"
#include "rows.cuh"

namespace {

using wxx_rows::Row;
using wxx_rows::warp_sum;

constexpr int kT = 256;
constexpr int kMaxTopk = 256;
constexpr int kMaxBeams = 16;
constexpr int kMaxStates = 128;
constexpr int kCandidates = 2048;     // of a row, in shared memory
constexpr int kClusterBlocks = 8;     // blocks that share a batch item's rows, at most

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
__device__ __forceinline__ float key_float(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ float key_value(uint64_t k) { return key_float((uint32_t)(k >> 32)); }

// The largest of three; a NaN wins where it is the highest and loses where it is
// the lowest.
template <uint32_t NAN_KEY>
__device__ __forceinline__ float largest(float a, float b, float c) {
  float d;
  if (NAN_KEY == kNanHighest)
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  else
    d = fmax3(a, b, c);
  return d;
}

// The lanes' values in descending order.
__device__ __forceinline__ uint32_t descending(uint32_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, v, j);
      const bool first = (lane & j) == 0, down = (lane & k) == 0;
      v = first == down ? max(v, other) : min(v, other);
    }
  return v;
}

struct Select {                       // shared memory of a row's selection
  uint64_t pair[kCandidates];
  unsigned hist[256];
  uint32_t reach[32];
  float sum[32], top[32];
  int warp[32];
  unsigned char looks[32][32];
  float tau;
  unsigned digit, rest;
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

// Puts the pairs of the entries that wanted() lets in into s.pair, in an order that
// depends on the row alone, and returns how many there are (the first kCandidates
// are kept); threads with look = false have none.  A warp goes through the 16-byte
// groups of its looking threads with all its lanes, marks what is wanted, and reads
// the marked entries again once the marks are counted over the block (a counter in
// shared memory that every pair takes a turn at cost 12,000 cycles for 228 pairs).
template <int THREADS, uint32_t NAN_KEY, class Wanted>
__device__ int collect(const Row& row, Select& s, bool look, Wanted wanted) {
  constexpr int kWarps = THREADS / 32, kAhead = 4, kRounds = 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned looking = __ballot_sync(0xffffffffu, look);
  const int n = __popc(looking);
  if (look) s.looks[warp][__popc(looking & ((1u << lane) - 1))] = (unsigned char)lane;
  __syncwarp();
  const int each = (row.groups + THREADS - 1) / THREADS;     // groups of a thread
  const bool lone = look && row.single >= 0 && wanted(row.p[row.single], row.single);
  // the group of this lane in round r, or past the end
  auto group_of = [&](int r) {
    const int i = r * 32 + lane, g = n ? i / n : each;
    return g < each ? warp * 32 + s.looks[warp][i - g * n] + g * THREADS : row.groups;
  };
  int total = 0;
  for (int r0 = 0; r0 < max(each, 1); r0 += kRounds) {       // each * 32 groups at most
    unsigned long long marks = 0;
#pragma unroll
    for (int k0 = 0; k0 < kRounds; k0 += kAhead) {
      if ((r0 + k0) * 32 >= n * each) break;
      float4 v[kAhead];
      int g[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        g[k] = (r0 + k0 + k) * 32 < n * each ? group_of(r0 + k0 + k) : row.groups;
        if (g[k] < row.groups) v[k] = row.mid[g[k]];
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int at = row.head + 4 * g[k];
        if (g[k] >= row.groups) continue;
        const unsigned four = (unsigned)wanted(v[k].x, at) | (unsigned)wanted(v[k].y, at + 1) << 1 |
                              (unsigned)wanted(v[k].z, at + 2) << 2 |
                              (unsigned)wanted(v[k].w, at + 3) << 3;
        marks |= (unsigned long long)four << 4 * (k0 + k);
      }
    }
    const int mine = __popcll(marks) + (int)(lone && r0 == 0);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int before = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += before;
    }
    __syncthreads();                  // s.warp has been read
    if (lane == 31) s.warp[warp] = upto;
    __syncthreads();
    const int w = lane < kWarps ? s.warp[lane] : 0;
    int at = total + upto - mine + __reduce_add_sync(0xffffffffu, lane < warp ? w : 0);
    total += __reduce_add_sync(0xffffffffu, w);
    if (lone && r0 == 0) {
      if (at < kCandidates) s.pair[at] = pair_key(row.p[row.single], row.single, NAN_KEY);
      ++at;
    }
    for (; marks; marks &= marks - 1, ++at) {
      const int k = __ffsll(marks) - 1;
      const int i = row.head + 4 * group_of(r0 + (k >> 2)) + (k & 3);
      if (at < kCandidates) s.pair[at] = pair_key(row.p[i], i, NAN_KEY);
    }
  }
  __syncthreads();
  return total;
}

// The warps' largest entries and sums of exponentials, and their join (the row's).
__device__ __forceinline__ void warp_sums(Select& s, float warp_top, float m, float part) {
  part = warp_sum(part * (m == -INFINITY || m == warp_top ? 1.0f : expf(m - warp_top)));
  if ((threadIdx.x & 31) == 0) {
    s.top[threadIdx.x >> 5] = warp_top;
    s.sum[threadIdx.x >> 5] = part;
  }
}
template <int WARPS>
__device__ __forceinline__ void join_sums(Select& s, float& top, float& sum) {
  const int lane = threadIdx.x & 31;
  const float w = lane < WARPS ? s.top[lane] : -INFINITY;
  top = key_float(__reduce_max_sync(0xffffffffu, value_key(w, kNanLowest)));
  sum = warp_sum(lane < WARPS ? s.sum[lane] * (w == top ? 1.0f : expf(w - top)) : 0.f);
}

// Puts the row's K best pairs, and perhaps more of its best, into s.pair and
// returns how many (K <= V).  With SUM, top and sum come to hold the row's largest
// number and the sum of exp(v - top).
//
// One pass over the row gives every thread its largest entry.  Of the jth largest
// of each warp's, the mth largest over the warps is a value tau that at least
// j m >= K entries reach, and few more do where m is about 2/3 of the warps: about
// 125 entries at K = 64 (with j = K / warps and the smallest over the warps it was
// 228).  The threads whose largest reaches tau read their entries again (from L2)
// and keep those that do.  Where too many do (long runs of one value, or large ones
// crowded into a few threads), the exact K-th pair is found digit by digit.
template <int THREADS, uint32_t NAN_KEY, bool SUM>
__device__ int best_pairs(const Row& row, int K, Select& s, float& top, float& sum) {
  constexpr int kWarps = THREADS / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float m = row.single >= 0 ? row.p[row.single] : -INFINITY;
  if (NAN_KEY == kNanLowest && m != m) m = -INFINITY;
  float part = 0.f;
  if (SUM && row.single >= 0 && row.p[row.single] != -INFINITY) part = expf(row.p[row.single] - m);
  // four groups at a time: their largest against the thread's so far, one rescaling
  // of its sum of exponentials
  constexpr int kAhead = 4;
  for (int i = threadIdx.x; i < row.groups; i += kAhead * THREADS) {
    float4 v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      v[k] = i + k * THREADS < row.groups
                 ? row.mid[i + k * THREADS]
                 : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    float n = m;
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      n = largest<NAN_KEY>(largest<NAN_KEY>(n, v[k].x, v[k].y), v[k].z, v[k].w);
    if (SUM) {
      // exp(v - n) is 2^y with y = (v - n) log2 e rounded: y half ulps lost, but a term weighs
      // its probability, over which the mean of y is log2 V at most, so the sum loses less
      // than by being added up.
      // Nothing but -inf (and perhaps NaN) so far: shifted by any number, they are 0.
      const float shift = n == -INFINITY ? 0.f : n;
      if (n > m) part *= fast_exp2((m - n) * 1.4426950408889634f);
      float e = 0.f;
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        e += (fast_exp2((v[k].x - shift) * 1.4426950408889634f) +
              fast_exp2((v[k].y - shift) * 1.4426950408889634f)) +
             (fast_exp2((v[k].z - shift) * 1.4426950408889634f) +
              fast_exp2((v[k].w - shift) * 1.4426950408889634f));
      part += e;
    }
    m = n;
  }
  // the nth largest of the warp's lanes (of their largest entries)
  uint32_t o = value_key(m, NAN_KEY);
  // (of the warps that have entries; tau is -inf where they are too few)
  const int active = min(kWarps, (row.groups + 31) / 32), most = max(1, active * 2 / 3);
  const int nth = min(32, (K + most - 1) / most);
  const int mth = (K + nth - 1) / nth;         // <= warps: K <= 32 warps
  uint32_t reach = __reduce_max_sync(0xffffffffu, o);
  if (SUM) warp_sums(s, key_float(reach), m, part);
  if (nth <= 4) {
    for (int k = 1; k < nth; ++k) {      // without the lane that had it
      if (lane == __ffs(__ballot_sync(0xffffffffu, o == reach)) - 1) o = 0;
      reach = __reduce_max_sync(0xffffffffu, o);
    }
  } else {
    reach = __shfl_sync(0xffffffffu, descending(o), nth - 1);
  }
  if (lane == 0) s.reach[warp] = reach;
  __syncthreads();
  if (warp == 0) {
    const uint32_t order = descending(lane < kWarps ? s.reach[lane] : 0u);
    if (lane == mth - 1) s.tau = key_float(order);
  }
  if (SUM) join_sums<kWarps>(s, top, sum);
  __syncthreads();
  const float tau = s.tau;
  // all pairs of a short row, else those that reach tau (NaN counts as reaching
  // where it is the highest; where it is the lowest, tau = -inf is left to the
  // digits, which know where it stands)
  const bool all = row.V <= kCandidates && tau == -INFINITY;
  if (all || tau > -INFINITY || NAN_KEY == kNanHighest) {
    const int n = collect<THREADS, NAN_KEY>(row, s, all || !(m < tau), [&](float v, int) {
      return all || (NAN_KEY == kNanHighest ? !(v < tau) : v >= tau);
    });
    if (n <= kCandidates) return n;
  }
  unsigned rest, none;
  const uint32_t cut = nth_key<THREADS>(
      row, s, K, rest, [](float v, int) { return value_key(v, NAN_KEY); },
      [](float, int) { return true; });
  const uint32_t last = ~nth_key<THREADS>(
      row, s, rest, none, [](float, int i) { return ~(uint32_t)i; },
      [&](float v, int) { return value_key(v, NAN_KEY) == cut; });
  return collect<THREADS, NAN_KEY>(row, s, true, [&](float v, int i) {
    const uint32_t k = value_key(v, NAN_KEY);
    return k > cut || (k == cut && (uint32_t)i <= last);
  });
}

// Sorts the first SIZE pairs (0 past n) in descending order, one a thread, by the
// first SIZE threads of the block; returns this thread's.
template <int SIZE>
__device__ __forceinline__ uint64_t sorted_pair(Select& s, int n) {
  const int t = threadIdx.x;
  uint64_t mine = t < n ? s.pair[t] : 0;
#pragma unroll
  for (int k = 2; k <= SIZE; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      uint64_t other;
      if (j >= 32) {
        asm volatile("bar.sync 1, %0;" ::"n"(SIZE) : "memory");
        s.pair[t] = mine;
        asm volatile("bar.sync 1, %0;" ::"n"(SIZE) : "memory");
        other = s.pair[t ^ j];
      } else {
        other = __shfl_xor_sync(0xffffffffu, mine, j);
      }
      const bool first = (t & j) == 0, down = (t & k) == 0;
      mine = (first == down) == (mine > other) ? mine : other;
    }
  return mine;
}

// Calls put(rank, pair) for the K best of the n pairs in s.pair, all different.
// Up to 64 of them are counted against each other, a few neighbouring threads
// sharing a pair's count; more are sorted, a pair a thread (n^2 / 32 reads of
// shared memory by a warp against log^2 n / 2 exchanges), or counted where threads
// are too few.
template <int THREADS, class F>
__device__ __forceinline__ void in_order(Select& s, int n, int K, F put) {
  const int t = threadIdx.x;
  if (n <= 64 || n > THREADS) {
    int share = 1;
    while (share < 32 && n * share * 2 <= THREADS) share <<= 1;
    const int lane = t & (share - 1);
    for (int at = 0; at < n; at += THREADS / share) {
      const int i = at + t / share;
      const uint64_t mine = i < n ? s.pair[i] : 0;
      int rank = 0;
#pragma unroll 4
      for (int j = lane; j < n; j += share) rank += s.pair[j] > mine;
      for (int o = 1; o < share; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
      if (i < n && lane == 0 && rank < K) put(rank, mine);
    }
    return;
  }
  uint64_t mine = 0;
  if (n <= 128) {
    if (t < 128) mine = sorted_pair<128>(s, n);
  } else if (n <= 256) {
    if (t < 256) mine = sorted_pair<256>(s, n);
  } else if (THREADS > 256) {
    if (n <= 512) {
      if (t < 512) mine = sorted_pair<512>(s, n);
    } else {
      mine = sorted_pair<THREADS>(s, n);
    }
  }
  if (t < K) put(t, mine);
}

// A block a row.  4 bytes an entry: the top 64 of 4096 x 50304 in 154 us, 5.4 TB/s.
// Two blocks of 1024 threads share an SM, one streams its row while the other picks;
// what is left of the time is where both pick (asking L2 for a later block's row in
// the meantime took 28 us longer).
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
    const uint32_t i = key_index(pair), v = (uint32_t)(pair >> 32);
    ids[at * K + rank] = i;
    // a key gives its value back, but for the sign of zero and a NaN's bits
    values[at * K + rank] = v == 0x80000000u || v == kNanHighest ? row.p[i] : key_float(v);
  });
}

// A warp a row, for short rows: its entries' keys stay in registers, entry 32 j + lane
// in key[j].  Of every lane's NTH largest, the mth largest over the lanes is a key
// that at least NTH m >= K entries reach.  From there the cut is raised by bisection
// towards the largest key: over the registers while more reach it than shared memory
// holds, then over those pairs until few more than K are left, which are counted
// against each other.  A ballot counts entries in the order of their indices, so of
// entries that a cut cannot tell apart the first are taken.
// Bound by its instructions (about 700 a row of 1024 at K = 32) and, with few rows, by
// their latency; there is no barrier: the top 32 of 1024 x 1024 take 6 us, of which the
// launch is 3, of 4096 x 1024 10 us (16.8 MB, 1.6 TB/s).
constexpr int kRowWarps = 4;

template <int M>
__device__ __forceinline__ int reaching(const uint32_t (&key)[M], uint32_t cut) {
  int n = 0;
#pragma unroll
  for (int j = 0; j < M; ++j) n += key[j] >= cut;
  return __reduce_add_sync(0xffffffffu, n);
}

// Raises the cut, which `left` >= K keys reach, until at most `most` do or it is the
// K-th key itself.
template <int M>
__device__ __forceinline__ void raise(const uint32_t (&key)[M], int K, int most, uint32_t& cut,
                                      uint32_t& high, int& left) {
  while (left > most && cut < high) {
    const uint32_t middle = cut + (high - cut + 1) / 2;
    const int n = reaching(key, middle);
    if (n >= K) {
      cut = middle;
      left = n;
    } else {
      high = middle - 1;
    }
  }
}

// put(j, place) for the keys that reach the cut or, where they are more than `most`,
// for the K first of them (the cut is the K-th key then).  Returns how many.
template <int M, class Put>
__device__ __forceinline__ int take(const uint32_t (&key)[M], int K, int most, uint32_t cut,
                                    int left, Put put) {
  const unsigned lower = (1u << (threadIdx.x & 31)) - 1;
  int n = 0;
  if (left <= most) {
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const unsigned who = __ballot_sync(0xffffffffu, key[j] >= cut);
      if (key[j] >= cut) put(j, n + __popc(who & lower));
      n += __popc(who);
    }
    return n;
  }
  int ties = K - reaching(key, cut + 1);
#pragma unroll
  for (int j = 0; j < M; ++j) {
    const unsigned same = __ballot_sync(0xffffffffu, key[j] == cut);
    const bool wanted = key[j] > cut || (key[j] == cut && __popc(same & lower) < ties);
    const unsigned who = __ballot_sync(0xffffffffu, wanted);
    if (wanted) put(j, n + __popc(who & lower));
    ties -= __popc(same);
    n += __popc(who);
  }
  return n;
}

template <int ITEMS, int NTH>
__global__ void __launch_bounds__(kRowWarps * 32)
    topk_rows_kernel(float* __restrict__ values, uint32_t* __restrict__ ids,
                     const float* __restrict__ x, int64_t ld, int64_t N, int V, int K) {
  constexpr int kMost = 40 * NTH;     // pairs to count: a quarter more than the largest K
  constexpr int kPairs = NTH == 8 ? 512 : 256;
  __shared__ uint64_t s_pair[kRowWarps][kPairs];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * kRowWarps + warp;
  if (at >= N) return;
  const float* row = x + at * ld;
  uint64_t* pair = s_pair[warp];
  uint32_t key[ITEMS];                // 0: no entry
  {
    float v[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) v[j] = 32 * j + lane < V ? row[32 * j + lane] : 0.f;
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      key[j] = 32 * j + lane < V ? value_key(v[j], kNanHighest) : 0u;
  }
  uint32_t best[NTH] = {};
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    uint32_t rest = key[j];
#pragma unroll
    for (int i = 0; i < NTH; ++i) {
      const uint32_t larger = max(best[i], rest);
      rest = min(best[i], rest);
      best[i] = larger;
    }
  }
  const int m = (K + NTH - 1) / NTH;
  uint32_t cut = m == 32 ? __reduce_min_sync(0xffffffffu, best[NTH - 1])
                         : __shfl_sync(0xffffffffu, descending(best[NTH - 1]), m - 1);
  uint32_t high = __reduce_max_sync(0xffffffffu, best[0]);
  cut = max(cut, 1u);
  int n = reaching(key, cut);
  raise(key, K, kPairs, cut, high, n);
  n = take(key, K, kPairs, cut, n, [&](int j, int place) {
    pair[place] = (uint64_t)key[j] << 32 | (uint32_t)~(32 * j + lane);
  });
  __syncwarp();
  constexpr int kOwn = (kMost + 31) / 32;
  uint64_t own[kPairs / 32];
  if (n > kMost) {
    uint32_t part[kPairs / 32];
#pragma unroll
    for (int i = 0; i < kPairs / 32; ++i) {
      own[i] = 32 * i + lane < n ? pair[32 * i + lane] : 0;
      part[i] = (uint32_t)(own[i] >> 32);
    }
    __syncwarp();                     // all have been read
    raise(part, K, kMost, cut, high, n);
    n = take(part, K, kMost, cut, n, [&](int i, int place) { pair[place] = own[i]; });
    __syncwarp();
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) own[i] = 32 * i + lane < n ? pair[32 * i + lane] : 0;
  int rank[kOwn] = {};
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const uint64_t other = pair[j];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) rank[i] += other > own[i];
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    if (own[i] == 0 || rank[i] >= K) continue;
    const uint32_t entry = key_index(own[i]), k = (uint32_t)(own[i] >> 32);
    ids[at * K + rank[i]] = entry;
    values[at * K + rank[i]] = k == 0x80000000u || k == kNanHighest ? row[entry] : key_float(k);
  }
}

template <int ITEMS>
void topk_rows(float* values, uint32_t* ids, const float* x, int64_t ld, int64_t N, int V, int K) {
  auto kernel = K <= 32    ? topk_rows_kernel<ITEMS, 1>
                : K <= 64  ? topk_rows_kernel<ITEMS, 2>
                : K <= 128 ? topk_rows_kernel<ITEMS, 4>
                           : topk_rows_kernel<ITEMS, 8>;
  kernel<<<(unsigned)((N + kRowWarps - 1) / kRowWarps), kRowWarps * 32, 0, wxx::stream()>>>(
      values, ids, x, ld, N, V, K);
}

// One selection step.  A cluster takes a batch item; its rows, or `parts` pieces
// of each where there are few, go to its blocks in turn.  Each sends the piece's
// best W pairs, its largest logit and its sum of exponentials to the first block,
// which merges them all:
//   score = scores[w] + ((z - top_w) - log sum_w)
// One item of 4 beams over 1024 tokens takes 6 us: start of a cluster, one pass, the
// merge, all latencies; 8 items of 8 beams over 50304 tokens (12.9 MB) 12 us.
constexpr int kMostPieces = kMaxBeams > kClusterBlocks ? kMaxBeams : kClusterBlocks;
static_assert(kMostPieces * kMaxBeams <= 256, "a thread a proposal");
struct Merge {
  uint64_t pair[kMostPieces * kMaxBeams];       // 0: no pair
  float top[kMostPieces], sum[kMostPieces];
  uint64_t key[kMostPieces * kMaxBeams];
};

template <int THREADS>
__global__ void __launch_bounds__(THREADS)
    beam_select_kernel(float* __restrict__ new_scores, uint32_t* __restrict__ parents,
                       uint32_t* __restrict__ new_tokens, uint32_t* __restrict__ new_finished,
                       const float* __restrict__ logits, int64_t ld,
                       const float* __restrict__ scores, const uint32_t* __restrict__ finished,
                       int W, int V, int parts, uint32_t stop) {
  __shared__ Select s;
  __shared__ Merge s_merge;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  auto started = cluster.barrier_arrive();
  bool met = false;                  // the cluster's blocks have all started
  auto meet = [&] {
    if (!met) cluster.barrier_wait(std::move(started));
    met = true;
  };
  const int rank = cluster.block_rank(), blocks = cluster.num_blocks();
  const int64_t b = blockIdx.x / blocks;
  const int t = threadIdx.x, pieces = W * parts, n = pieces * W;
  Merge* merge = cluster.map_shared_rank(&s_merge, 0);
  // a thread of the merge: proposal r of piece t / W
  const int my_piece = t / W, my_beam = my_piece / parts, my_rank = t - my_piece * W;
  const bool mine = rank == 0 && t < n;
  const float score = mine ? scores[b * W + my_beam] : 0.f;
  const bool done = mine && finished && finished[b * W + my_beam];
  // a piece's length, a multiple of 4 so that all start where the first does
  const int length = parts == 1 ? V : ((V + parts - 1) / parts + 3) / 4 * 4;
  for (int q = rank; q < pieces; q += blocks) {
    const int w = q / parts, from = (q - w * parts) * length;
    const int len = min(length, V - from), K = min(W, len);
    if (finished && finished[b * W + w]) continue;
    const Row row(logits + (b * W + w) * ld + from, len);
    float top, sum;
    const int found = best_pairs<THREADS, kNanLowest, true>(row, K, s, top, sum);
    meet();
    in_order<THREADS>(s, found, K, [&](int r, uint64_t pair) {
      merge->pair[q * W + r] = pair - (uint32_t)from;          // the inverted index of the row
    });
    if (t < W && t >= K) merge->pair[q * W + t] = 0;
    if (t == 0) {
      merge->top[q] = top;
      merge->sum[q] = sum;
    }
    __syncthreads();                 // s is used again
  }
  meet();
  cluster.sync();
  if (rank != 0) return;
  // Every beam's W best pairs of all its pieces compete: by score, then the lower
  // beam, then the better pair of it.
  uint64_t pair = 0;
  uint64_t key = 0;                  // no proposal
  if (mine) {
    float c = -INFINITY;
    int place = my_rank;             // among the beam's
    if (done) {
      c = my_piece == my_beam * parts && my_rank == 0 ? score : -INFINITY;
    } else {
      pair = s_merge.pair[t];
      const int first = my_beam * parts;
      float top = -INFINITY, sum = 0.f;
      for (int k = first; k < first + parts; ++k) top = fmaxf(top, s_merge.top[k]);
      for (int k = first; k < first + parts; ++k)
        sum += s_merge.sum[k] * (s_merge.top[k] == top ? 1.0f : expf(s_merge.top[k] - top));
      if (pair) c = score + ((key_value(pair) - top) - logf(sum));
      if (parts > 1) {
        place = 0;
        for (int k = first * W; k < (first + parts) * W; ++k) place += s_merge.pair[k] > pair;
      }
    }
    if (place < W && !(done && my_piece != my_beam * parts))
      key = (uint64_t)value_key(c, kNanLowest) << 32 | (uint32_t)(kMaxBeams - my_beam) << 8 |
            (uint32_t)(255 - place);
    s_merge.key[t] = key;
  }
  __syncthreads();
  if (!mine || key == 0) return;
  int place = 0;
#pragma unroll 8
  for (int j = 0; j < n; ++j) place += s_merge.key[j] > key;
  if (place >= W) return;
  const uint32_t token = done ? stop : pair ? key_index(pair) : 0u;
  const int64_t o = b * W + place;
  new_scores[o] = key_value(key);
  parents[o] = my_beam;
  new_tokens[o] = token;
  if (new_finished) new_finished[o] = done || token == stop;
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
// rows are 16-byte aligned.  Bound by memory: 8 items of 8 beams with four caches of 700
// x 1024 floats (about 1.1 GB read and written) in 165 us, 6.5 TB/s.  Of more than 8 beams a
// thread holds twice as many (140 registers, one block an SM) and is further from it: 4
// items of 16 beams (1.18 GB) 221 us, 5.3 TB/s, 6 of 9 (0.95 GB) 218 us, 4.4 TB/s.
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
    uint32_t parent = t < W ? parents[b * W + t] : (uint32_t)t;
    if (t < W && parent >= (uint32_t)W) {        // also where it is below MAX
      wxx_device_fail(err, WXX_DEV_ERR_BAD_INDEX);
      parent = (uint32_t)t;
    }
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

// The rows' next tokens behind their first *cur_len ids; the block that writes them
// all advances the length.
__global__ void beam_append_kernel(uint32_t* __restrict__ ids, int64_t ld, int64_t rows,
                                   const uint32_t* __restrict__ tokens, uint32_t* cur_len,
                                   uint32_t most, int* err) {
  const uint32_t n = *cur_len;
  __syncthreads();
  if (n >= most) {
    if (threadIdx.x == 0) wxx_device_fail(err, WXX_DEV_ERR_BAD_INDEX);
    return;
  }
  for (int64_t r = threadIdx.x; r < rows; r += blockDim.x) ids[r * ld + n] = tokens[r];
  if (threadIdx.x == 0) *cur_len = n + 1;
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
  // A warp a row against a block a row: 4096 rows of 1024 at K = 8, 32 and 128 8, 10 and
  // 25 us and 37, 33 and 74 us, of 2048 12, 16 and 31 and 27, 33 and 74 us, 16 of 2048 6, 6
  // and 10 and 6, 6 and 8 us.
  // Small blocks hide one another's steps, but more rows are then under way and what
  // is read again no longer comes from L2, and a large K takes most entries of few
  // threads.  256, 512 and 1024 threads, 100 M entries: rows of 4096 at K = 32 179, 322
  // and 631 us, of 16384 at K = 64 101, 109 and 152 and at K = 128 411, 156 and 191, of
  // 24576 at K = 64 122, 91 and 119, of 32768 133, 84 and 98, of 50304 137, 106 and 84; at
  // K = 256 rows of 4096 take 10569, 4570 and 997.  (A memory bound pass takes 64.)
  if (V <= 256)
    topk_rows<8>(values, ids, x, ld, N, (int)V, K);
  else if (V <= 512)
    topk_rows<16>(values, ids, x, ld, N, (int)V, K);
  else if (V <= 1024)
    topk_rows<32>(values, ids, x, ld, N, (int)V, K);
  else if (V <= 2048)
    topk_rows<64>(values, ids, x, ld, N, (int)V, K);
  else if (V <= 16384 && K <= 64)
    topk_kernel<256><<<(unsigned)N, 256, 0, wxx::stream()>>>(values, ids, x, ld, (int)V, K);
  else if (V <= 32768 && K <= 128)
    topk_kernel<512><<<(unsigned)N, 512, 0, wxx::stream()>>>(values, ids, x, ld, (int)V, K);
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
  // Where rows are long and few, those of fewer beams than the cluster has blocks are
  // split, and blocks have 512 threads.  1 item of 4 beams over 50304 tokens took 10 us
  // (12 us with a block of 256 threads a row), 8 of 8 beams 12 us (14 us); 32 of 4
  // beams, more than one block an SM, 14 us with a block of 256 a row and 23 us split.
  // (With clusters of 16 blocks, which are not portable, 8 of 8 beams took 9 us more.)
  const bool few = V > 16384 && B * (W < kClusterBlocks ? kClusterBlocks / W * W : kClusterBlocks)
                                    <= wxx::num_sms();
  const int parts = few && W < kClusterBlocks ? kClusterBlocks / W : 1;
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
  return few ? launch(beam_select_kernel<512>, 512) : launch(beam_select_kernel<256>, 256);
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

// ids[r, *cur_len] = tokens[r] for the rows of ids (rows, most; row stride ld), then
// *cur_len += 1.  A full table is left as it is and sets the device error word.
WXX_EXPORT int wxx_beam_append(uint32_t* ids, int64_t ld, int64_t rows, const uint32_t* tokens,
                               uint32_t* cur_len, int64_t most) {
  WXX_REQUIRE_INIT();
  WXX_REQUIRE(rows >= 0 && most >= 0 && most < (int64_t(1) << 32) && ld >= most,
              "wxx_beam_append: bad sizes");
  if (rows == 0) return WXX_OK;
  beam_append_kernel<<<1, kT, 0, wxx::stream()>>>(ids, ld, rows, tokens, cur_len, (uint32_t)most,
                                                  wxx::device_error_word());
  WXX_LAUNCH_CHECK();
  return WXX_OK;
}
