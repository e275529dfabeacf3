// Selection over logits: the k largest of each row, and one step of beam
// search (selection over beams and vocabulary, and the reordering of the
// beams' states in place).
//
// Order.  Values are compared as numbers (-0 equals +0), equal values by the
// lower index first.  wxx_topk puts NaN above every number; beam search gives
// a beam whose log-probabilities are NaN the score -inf.

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

WXX_EXPORT int wxx_malloc(void** out, uint64_t nbytes);
WXX_EXPORT int wxx_free(void* p);

namespace {

constexpr int kT = 256;
constexpr int kMaxTopk = 256;
constexpr int kMaxBeams = 16;
constexpr int kMaxStates = 128;

// A (value, index) pair as one number that is larger for the better pair:
// the value's order-preserving bits above the inverted index.  nan_key is what
// a NaN counts as.
__device__ __forceinline__ uint64_t pair_key(float v, uint32_t i, uint32_t nan_key) {
  const uint32_t u = __float_as_uint(v + 0.0f);          // -0 becomes +0
  uint32_t k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  if (v != v) k = nan_key;
  return ((uint64_t)k << 32) | (uint32_t)~i;
}
constexpr uint32_t kNanHighest = 0xfffffffeu;             // above +inf, and no pair is all ones
constexpr uint32_t kNanLowest = 0x007fffffu;             // the key of -inf

__device__ __forceinline__ uint32_t key_index(uint64_t k) { return ~(uint32_t)k; }

__device__ __forceinline__ uint64_t block_max_key(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < kT / 32; ++w) v = red[w] > v ? red[w] : v;
  __syncthreads();
  return v;
}

// The best pair of the row that is below `under`.
__device__ uint64_t next_best(const float* __restrict__ row, int V, uint64_t under,
                              uint32_t nan_key, uint64_t* red) {
  uint64_t best = 0;
  for (int c = threadIdx.x; c < V; c += kT) {
    const uint64_t k = pair_key(row[c], c, nan_key);
    if (k < under && k > best) best = k;
  }
  return block_max_key(best, red);
}

__global__ void __launch_bounds__(kT)
    topk_kernel(float* __restrict__ values, uint32_t* __restrict__ ids,
                const float* __restrict__ x, int64_t ld, int V, int K) {
  __shared__ uint64_t red[kT / 32];
  const int64_t row = blockIdx.x;
  const float* z = x + row * ld;
  uint64_t under = ~0ull;
  for (int k = 0; k < K; ++k) {
    under = next_best(z, V, under, kNanHighest, red);
    if (threadIdx.x == 0) {
      const uint32_t i = key_index(under);
      ids[row * K + k] = i;
      values[row * K + k] = z[i];
    }
  }
}

// Candidates of one beam: its W best tokens by logit with their scores.
__global__ void __launch_bounds__(kT)
    beam_rows_kernel(float* __restrict__ cand, uint32_t* __restrict__ tokens,
                     const float* __restrict__ logits, int64_t ld,
                     const float* __restrict__ scores, const uint32_t* __restrict__ finished,
                     int W, int V, uint32_t stop) {
  __shared__ uint64_t red[kT / 32];
  __shared__ float s_sum[kT / 32];
  const int64_t row = blockIdx.x;
  const float* z = logits + row * ld;
  const float score = scores[row];
  if (finished && finished[row]) {
    if (threadIdx.x < W) {
      cand[row * W + threadIdx.x] = threadIdx.x == 0 && score == score ? score : -INFINITY;
      tokens[row * W + threadIdx.x] = stop;
    }
    return;
  }
  uint64_t under = next_best(z, V, ~0ull, kNanLowest, red);
  const float m = z[key_index(under)];
  float s = 0.f;
  for (int c = threadIdx.x; c < V; c += kT) s += expf(z[c] - m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.f;
#pragma unroll
  for (int w = 0; w < kT / 32; ++w) s += s_sum[w];
  const float log_s = logf(s);
  for (int k = 0; k < W; ++k) {
    if (threadIdx.x == 0) {
      const uint32_t i = key_index(under);
      const float c = k < V ? score + ((z[i] - m) - log_s) : -INFINITY;
      cand[row * W + k] = c == c ? c : -INFINITY;
      tokens[row * W + k] = k < V ? i : 0u;
    }
    if (k + 1 < V) under = next_best(z, V, under, kNanLowest, red);
  }
}

// The W best candidates of a batch item, by score, then beam, then rank.
__global__ void beam_merge_kernel(float* __restrict__ new_scores, uint32_t* __restrict__ parents,
                                  uint32_t* __restrict__ new_tokens,
                                  uint32_t* __restrict__ new_finished,
                                  const float* __restrict__ cand,
                                  const uint32_t* __restrict__ tokens,
                                  const uint32_t* __restrict__ finished, int W, uint32_t stop) {
  const int64_t b = blockIdx.x;
  const int i = threadIdx.x, n = W * W;
  if (i >= n) return;
  const float* c = cand + b * n;
  const uint64_t mine = pair_key(c[i], i, kNanLowest);
  int rank = 0;
  for (int j = 0; j < n; ++j) rank += pair_key(c[j], j, kNanLowest) > mine;
  if (rank >= W) return;
  const int64_t o = b * W + rank;
  new_scores[o] = c[i];
  parents[o] = i / W;
  const uint32_t t = tokens[b * n + i];
  new_tokens[o] = t;
  if (new_finished) new_finished[o] = finished[b * W + i / W] != 0 || t == stop;
}

struct StateTable {
  int n;
  uint32_t* p[kMaxStates];
  int64_t row[kMaxStates];     // words of a row
  int64_t unit[kMaxStates];    // words of one position (0: the whole row moves)
};

// Every thread owns a word position of a batch item: it reads it from all the
// beams, then writes it to all, so the move is in place.
__global__ void beam_reorder_kernel(const __grid_constant__ StateTable tab,
                                    const uint32_t* __restrict__ parents,
                                    const uint32_t* __restrict__ cur_len, int W, int* err) {
  const int64_t b = blockIdx.y;
  const int s = blockIdx.z;
  int64_t n = tab.row[s];
  if (cur_len && tab.unit[s]) {
    const int64_t used = (int64_t)*cur_len * tab.unit[s];
    n = used < n ? used : n;
  }
  uint32_t* base = tab.p[s] + b * W * tab.row[s];
  for (int64_t i = (int64_t)blockIdx.x * kT + threadIdx.x; i < n; i += (int64_t)gridDim.x * kT) {
    uint32_t v[kMaxBeams];
    for (int w = 0; w < W; ++w) v[w] = base[w * tab.row[s] + i];
    for (int w = 0; w < W; ++w) {
      const uint32_t p = parents[b * W + w];
      if (p >= (uint32_t)W) {
        wxx_device_fail(err, WXX_DEV_ERR_BAD_INDEX);
        continue;
      }
      base[w * tab.row[s] + i] = v[p];
    }
  }
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
  topk_kernel<<<(unsigned)N, kT, 0, wxx::stream()>>>(values, ids, x, ld, (int)V, K);
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
  void* scratch = nullptr;
  const int64_t n = B * W * W;
  if (int st = wxx_malloc(&scratch, (uint64_t)n * 8)) return st;
  float* cand = static_cast<float*>(scratch);
  uint32_t* toks = reinterpret_cast<uint32_t*>(cand + n);
  beam_rows_kernel<<<(unsigned)(B * W), kT, 0, wxx::stream()>>>(cand, toks, logits, ld, scores,
                                                                finished, W, (int)V, stop);
  int st = wxx::after_launch(__FILE__, __LINE__);
  if (st == WXX_OK) {
    beam_merge_kernel<<<(unsigned)B, 256, 0, wxx::stream()>>>(
        new_scores, parents, tokens, new_finished, cand, toks, finished, W, stop);
    st = wxx::after_launch(__FILE__, __LINE__);
  }
  wxx_free(scratch);
  return st;
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
    int64_t blocks = (longest + kT - 1) / kT;
    if (blocks > 1024) blocks = 1024;
    dim3 grid((unsigned)blocks, (unsigned)B, (unsigned)tab.n);
    beam_reorder_kernel<<<grid, kT, 0, wxx::stream()>>>(tab, parents, cur_len, W,
                                                        wxx::device_error_word());
    WXX_LAUNCH_CHECK();
  }
  return WXX_OK;
}
