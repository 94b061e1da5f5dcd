// The router of a mixture of experts (gfx950): for each token the k largest of
// its logits, their softmax weights, and the tokens' rows ordered by expert;
// and the sum of the experts' rows per token.
//
// Choice: G lanes hold a token's logits, eight each, and take the largest k
// times.  A logit is compared as an integer of the same order (NaN above all,
// both zeros equal), the lowest index first among equals.  -inf masks an
// expert: it is never chosen, and a token with fewer than k experts left has -1
// and weight 0 in the rest.
//
// Order: a stable counting sort of the T k assignments by expert, those without
// one last.  The blocks that choose count their tokens' experts; then as many
// blocks sum the counts before their own and rank their assignments: lanes of a
// wave with the same expert find each other by one ballot per bit of the
// expert's number.  No order depends on atomics (those on integer counts only
// add up).  Few tokens take one block and one launch.
//
// Few tokens are bound by the launch (8 of 32 experts: 4.4 us).  100k tokens of 16
// experts, two choices: 10.0 us to choose and 10.7 to rank, where the bytes of both
// take about 1: the blocks' barriers, and counts and choices that go through memory
// between the two; the gradient 4.0 us.  The sum of 100k tokens' rows and its
// gradient (12.0 and 20.8 us, 96 channels) are bound by memory.
#include "numeric.hpp"

#include <algorithm>

namespace spira_hip {

namespace route {

constexpr int kMaxExperts = 512;
constexpr int kMaxChoices = 16;
constexpr int kTile = 2048;  // most assignments per block
constexpr int kHeld = 8;     // logits per lane

// larger logit, larger key; 0 for nothing left
__device__ __forceinline__ uint32_t sort_key(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.f);  // (-0 is 0)
  if (v != v) return 0xFFFFFFFFu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kMasked = 0x007FFFFFu;  // sort_key(-inf)

template <int G> __device__ __forceinline__ void largest(uint32_t &key, int &index) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    const uint32_t k = __shfl_xor(key, o, 64);
    const int i = __shfl_xor(index, o, 64);
    if (k > key || (k == key && i < index)) {
      key = k;
      index = i;
    }
  }
}

// One token by G lanes: lane `lane` holds the logits of experts lane * kHeld
// and on.  Calls put(j, expert or -1, numerator of its softmax weight) for each
// choice and put(-1, 0, denominator) at the end, on every lane.
template <class T, int G, class Put>
__device__ __forceinline__ void choose(const T *logits, int experts, int k, int renormalize, int lane, Put &&put) {
  float v[kHeld];
  uint32_t key[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld / kVec<T>; ++i) {
    const int at = lane * kHeld + i * kVec<T>;
    const Chunk<T> c = load_chunk(logits + at, experts - at);
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) v[i * kVec<T> + j] = c.v[j];
  }
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const uint32_t s = sort_key(v[i]);
    key[i] = lane * kHeld + i < experts && s > kMasked ? s : 0;
  }
  float top = 0, sum = 0;
  for (int j = 0; j < k; ++j) {
    uint32_t best = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < kHeld; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    int index = lane * kHeld + at;
    largest<G>(best, index);
    float num = 0;
    if (best != 0) {
      // (the key back to its logit)
      const float value = best == 0xFFFFFFFFu
                              ? __builtin_nanf("")
                              : __builtin_bit_cast(float, best & 0x80000000u ? best & 0x7FFFFFFFu : ~best);
      if (j == 0) top = value;
      num = expf(value - top);
    }
    const int e = best != 0 ? index : -1;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (e == lane * kHeld + i) key[i] = 0;
    if (j == 0 && !renormalize) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (e >= 0 && lane * kHeld + i < experts) sum += expf(v[i] - top);
      sum = group_sum<G>(sum);
    }
    if (renormalize) sum += num;
    put(j, e, num);
  }
  put(-1, 0, sum);
}

// the bin of an assignment: its expert, or `experts` without one (also for
// numbers that are none, so that no count leaves its place)
__device__ __forceinline__ int bin_of(int32_t e, int experts) {
  return static_cast<uint32_t>(e) < static_cast<uint32_t>(experts) ? e : experts;
}

// The choices of tokens first to first + count by the block's 256 threads, 256 / G
// at a time, and their number per bin.
template <class T, int G>
__device__ void choose_tokens(const T *logits, int64_t first, int count, int experts, int k, int renormalize,
                              float *weights, int32_t *chosen, int32_t *bins) {
  constexpr int TPB = 256 / G;
  __shared__ float num[TPB][kMaxChoices + 1];
  __shared__ int32_t pick[TPB][kMaxChoices + 1];
  const int lane = threadIdx.x % G, slot = threadIdx.x / G;
  for (int e = threadIdx.x; e <= experts; e += 256) bins[e] = 0;
  for (int t0 = 0; t0 < count; t0 += TPB) {
    __syncthreads();
    if (t0 + slot < count)
      choose<T, G>(logits + (first + t0 + slot) * experts, experts, k, renormalize, lane, [&](int j, int e, float v) {
        if (lane != 0) return;
        num[slot][j < 0 ? kMaxChoices : j] = v;
        if (j >= 0) pick[slot][j] = e;
      });
    __syncthreads();
    const int n = min(TPB, count - t0) * k;
    for (int i = threadIdx.x; i < n; i += 256) {
      const int t = i / k, j = i % k;
      const int32_t e = pick[t][j];
      weights[(first + t0) * k + i] = e >= 0 ? num[t][j] / num[t][kMaxChoices] : 0.f;
      chosen[(first + t0) * k + i] = e;
      atomicAdd(&bins[bin_of(e, experts)], 1);
    }
  }
  __syncthreads();
}

// choices of `tile` tokens a block, and counts[bin, block]
template <class T, int G>
__global__ __launch_bounds__(256) void choose_kernel(const T *logits, int64_t tokens, int tile, int experts, int k,
                                                     int renormalize, float *weights, int32_t *chosen,
                                                     int32_t *counts) {
  __shared__ int32_t bins[kMaxExperts + 1];
  const int64_t first = blockIdx.x * static_cast<int64_t>(tile);
  choose_tokens<T, G>(logits, first, static_cast<int>(std::min<int64_t>(tile, tokens - first)), experts, k, renormalize,
                      weights, chosen, bins);
  for (int e = threadIdx.x; e <= experts; e += 256) counts[e * static_cast<int64_t>(gridDim.x) + blockIdx.x] = bins[e];
}

// inclusive sum over the block's threads (NT), with the block's total
template <int NT> __device__ __forceinline__ int32_t block_scan(int32_t v, int32_t *shared, int32_t &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int32_t u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 63) shared[wave] = v;
  __syncthreads();
  int32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    before += w < wave ? shared[w] : 0;
    total += shared[w];
  }
  return v + before;
}

// one block per bin: its counts to running sums over the blocks, and its total
__global__ __launch_bounds__(256) void running_kernel(int blocks, int32_t *counts, int32_t *totals) {
  __shared__ int32_t shared[4];
  int32_t *c = counts + blockIdx.x * static_cast<int64_t>(blocks);
  int32_t sum = 0;
  for (int first = 0; first < blocks; first += 256) {
    const int i = first + threadIdx.x;
    const int32_t v = i < blocks ? c[i] : 0;
    int32_t total;
    const int32_t upto = block_scan<256>(v, shared, total);
    if (i < blocks) c[i] = sum + upto - v;
    sum += total;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = sum;
}

// lanes of the wave whose value (below 2^bits) is this lane's; `there`: lanes that have one
__device__ __forceinline__ uint64_t same(int value, int bits, bool there) {
  uint64_t m = ballot(there);
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = ballot(value >> b & 1);
    m &= value >> b & 1 ? set : ~set;
  }
  return m;
}

struct Order {
  int experts, k, bits;
  int32_t *offsets, *rows, *slots;
};

// Ranks assignments first to last (at most kTile) of `chosen`; begin(e): the
// first row of bin e for them.  A quarter of them a wave, in order.
template <class Begin>
__device__ void rank_tile(const int32_t *chosen, int64_t first, int64_t last, const Order &o, Begin &&begin) {
  __shared__ int32_t base[4][kMaxExperts + 1];  // next row of each bin, per wave
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int share = static_cast<int>((last - first + 255) / 256) * 64;
  const int64_t from = first + wave * share, to = std::min(from + share, last);
  for (int e = lane; e <= o.experts; e += 64) base[wave][e] = 0;
  __syncthreads();
  int bin[kTile / 256];
#pragma unroll
  for (int i = 0; i < kTile / 256; ++i) {
    const int64_t a = from + i * 64 + lane;
    bin[i] = a < to ? bin_of(chosen[a], o.experts) : o.experts;
    if (a < to) atomicAdd(&base[wave][bin[i]], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= o.experts; e += 256) {
    int32_t at = begin(e);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int32_t c = base[w][e];
      base[w][e] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kTile / 256; ++i) {
    const int64_t a = from + i * 64 + lane;
    const bool there = a < to;
    if (!ballot(there)) break;
    const uint64_t m = same(bin[i], o.bits, there);
    if (there) {
      const int32_t at = base[wave][bin[i]] + lane_prefix(m);
      // (the last lane of each expert, after all have read; a wave's LDS
      // accesses keep their order)
      if ((m >> lane) == 1) base[wave][bin[i]] = at + 1;
      const bool held = bin[i] < o.experts;
      o.rows[at] = held ? static_cast<int32_t>(a / o.k) : -1;
      o.slots[a] = held ? at : -1;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// first[e] = sum of v[0 .. e - 1] for the experts + 1 bins of a block
__device__ __forceinline__ void bins_before(const int32_t *v, int32_t *first, int experts, int32_t *shared) {
  int32_t sum = 0;
  for (int e0 = 0; e0 <= experts; e0 += 256) {
    const int e = e0 + threadIdx.x;
    const int32_t c = e <= experts ? v[e] : 0;
    int32_t total;
    const int32_t upto = block_scan<256>(c, shared, total);
    if (e <= experts) first[e] = sum + upto - c;
    sum += total;
  }
  __syncthreads();
}

// (totals null: the counts are those of the blocks, and each block sums them;
// else running_kernel has)
__global__ __launch_bounds__(256) void rank_kernel(const int32_t *chosen, int64_t n, int tile, int blocks,
                                                   const int32_t *counts, const int32_t *totals, const Order o) {
  __shared__ int32_t total[kMaxExperts + 1], before[kMaxExperts + 1], first[kMaxExperts + 1], shared[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (totals) {
    for (int e = threadIdx.x; e <= o.experts; e += 256) {
      total[e] = totals[e];
      before[e] = n > 0 ? counts[e * static_cast<int64_t>(blocks) + blockIdx.x] : 0;
    }
  } else {
    for (int e = wave; e <= o.experts; e += 4) {
      int32_t all = 0, mine = 0;
      for (int b = lane; b < blocks; b += 64) {
        const int32_t c = counts[e * static_cast<int64_t>(blocks) + b];
        all += c;
        mine += b < static_cast<int>(blockIdx.x) ? c : 0;
      }
#pragma unroll
      for (int s = 32; s > 0; s >>= 1) {
        all += __shfl_xor(all, s, 64);
        mine += __shfl_xor(mine, s, 64);
      }
      if (lane == 0) {
        total[e] = all;
        before[e] = mine;
      }
    }
  }
  __syncthreads();
  bins_before(total, first, o.experts, shared);
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= o.experts; e += 256) o.offsets[e] = first[e];
  const int64_t a = blockIdx.x * static_cast<int64_t>(tile);
  rank_tile(chosen, a, std::min<int64_t>(a + tile, n), o, [&](int e) { return first[e] + before[e]; });
}

// the whole of it by one block
template <class T, int G>
__global__ __launch_bounds__(256) void route_kernel(const T *logits, int tokens, int renormalize, float *weights,
                                                    int32_t *chosen, const Order o) {
  __shared__ int32_t bins[kMaxExperts + 1], first[kMaxExperts + 1], shared[4];
  choose_tokens<T, G>(logits, 0, tokens, o.experts, o.k, renormalize, weights, chosen, bins);
  bins_before(bins, first, o.experts, shared);
  for (int e = threadIdx.x; e <= o.experts; e += 256) o.offsets[e] = first[e];
  // (the choices, written by other threads of the block, are visible behind the barriers)
  rank_tile(chosen, 0, static_cast<int64_t>(tokens) * o.k, o, [&](int e) { return first[e]; });
}

// dlogits.  Over the chosen: w (d - sum d w) at them, 0 elsewhere; over all
// experts: p (d - sum d w), with p made again from the logits.
template <class T, int G>
__global__ __launch_bounds__(256) void choose_backward_kernel(const T *logits, const float *weights,
                                                              const int32_t *chosen, const float *dweights,
                                                              int64_t first, int64_t tokens, int experts, int k,
                                                              int renormalize, T *dlogits) {
  const int lane = threadIdx.x % G;
  const int64_t token = (first + blockIdx.x) * (256 / G) + threadIdx.x / G;
  if (token >= tokens) return;
  float p[kHeld] = {}, d[kHeld] = {};
  float mean = 0;
  for (int j = 0; j < k; ++j) {
    const int e = chosen[token * k + j];
    if (e < 0) continue;
    const float dj = dweights[token * k + j], w = weights[token * k + j];
    mean += dj * w;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (e == lane * kHeld + i) {
        d[i] = dj;
        p[i] = w;
      }
  }
  if (!renormalize) {
    float top = -INFINITY, sum = 0;
#pragma unroll
    for (int i = 0; i < kHeld / kVec<T>; ++i) {
      const int at = lane * kHeld + i * kVec<T>;
      const Chunk<T> c = load_chunk(logits + token * experts + at, experts - at);
#pragma unroll
      for (int j = 0; j < kVec<T>; ++j) p[i * kVec<T> + j] = at + j < experts ? c.v[j] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) top = fmaxf(top, p[i]);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if (top == -INFINITY) top = 0;  // (no expert: every p is 0)
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      p[i] = expf(p[i] - top);
      sum += p[i];
    }
    sum = group_sum<G>(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) p[i] *= inv;
  }
#pragma unroll
  for (int i = 0; i < kHeld / kVec<T>; ++i) {
    const int at = lane * kHeld + i * kVec<T>;
    Chunk<T> c;
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) c.v[j] = p[i * kVec<T> + j] * (d[i * kVec<T> + j] - mean);
    if (renormalize) {
#pragma unroll
      for (int j = 0; j < kVec<T>; ++j)
        if (p[i * kVec<T> + j] == 0.f) c.v[j] = 0.f;
    }
    store_chunk(dlogits + token * experts + at, experts - at, c);
  }
}

// y[t] = sum_j w[t, j] h[slots[t, j]]: a thread per chunk of a token's row.  I: type
// of h, the outputs' or fp32
template <class T, class I>
__global__ __launch_bounds__(256) void combine_kernel(const I *h, int64_t rows, const int32_t *slots,
                                                      const float *weights, int64_t first, int64_t tokens, int k, int c,
                                                      T *y) {
  const int chunks = (c + kVec<T> - 1) / kVec<T>;
  const int64_t i = (first + blockIdx.x) * 256 + threadIdx.x;
  if (i >= tokens * chunks) return;
  const int64_t t = i / chunks;
  const int at = static_cast<int>(i - t * chunks) * kVec<T>;
  Chunk<T> sum{};
  for (int j = 0; j < k; ++j) {
    const int32_t s = slots[t * k + j];
    if (s < 0 || s >= rows) continue;
    const float w = weights ? weights[t * k + j] : 1.f;
    const I *row = h + static_cast<int64_t>(s) * c + at;
#pragma unroll
    for (int p = 0; p < kVec<T>; p += kVec<I>) {
      const Chunk<I> v = load_chunk(row + p, c - at - p);
#pragma unroll
      for (int q = 0; q < kVec<I>; ++q) sum.v[p + q] += w * v.v[q];
    }
  }
  store_chunk(y + t * c + at, c - at, sum);
}

// dh[slots[t, j]] = w dy[t], dw[t, j] = <dy[t], h[slots[t, j]]>: 16 lanes per
// token; then zeros in the rows of no token
template <class T>
__global__ __launch_bounds__(256) void combine_backward_kernel(const T *h, int64_t rows, const int32_t *rows_of,
                                                               const int32_t *slots, const float *weights,
                                                               const T *dy, int64_t first, int64_t tokens, int k,
                                                               int c, int64_t token_blocks, T *dh, float *dweights) {
  constexpr int G = 16;
  const int lane = threadIdx.x % G;
  const int64_t block = first + blockIdx.x;
  if (block >= token_blocks) {
    const int64_t r = (block - token_blocks) * (256 / G) + threadIdx.x / G;
    if (!dh || r >= rows || rows_of[r] >= 0) return;
    for (int at = lane * kVec<T>; at < c; at += G * kVec<T>) store_chunk(dh + r * c + at, c - at, Chunk<T>{});
    return;
  }
  const int64_t t = block * (256 / G) + threadIdx.x / G;
  if (t >= tokens) return;
  for (int j = 0; j < k; ++j) {
    const int32_t s = slots[t * k + j];
    float dot = 0;
    if (s >= 0 && s < rows) {
      const float w = weights[t * k + j];
      for (int at = lane * kVec<T>; at < c; at += G * kVec<T>) {
        Chunk<T> g = load_chunk(dy + t * c + at, c - at);
        if (dweights) {
          const Chunk<T> v = load_chunk(h + static_cast<int64_t>(s) * c + at, c - at);
#pragma unroll
          for (int q = 0; q < kVec<T>; ++q) dot += g.v[q] * v.v[q];
        }
        if (dh) {
#pragma unroll
          for (int q = 0; q < kVec<T>; ++q) g.v[q] *= w;
          store_chunk(dh + static_cast<int64_t>(s) * c + at, c - at, g);
        }
      }
    }
    dot = group_sum<G>(dot);
    if (dweights && lane == 0) dweights[t * k + j] = dot;
  }
}

// f(lanes) for a token of this many experts
template <class F> int with_lanes(int experts, F &&f) {
  using std::integral_constant;
  if (experts <= kHeld) return f(integral_constant<int, 1>{});
  if (experts <= 2 * kHeld) return f(integral_constant<int, 2>{});
  if (experts <= 4 * kHeld) return f(integral_constant<int, 4>{});
  if (experts <= 8 * kHeld) return f(integral_constant<int, 8>{});
  if (experts <= 16 * kHeld) return f(integral_constant<int, 16>{});
  if (experts <= 32 * kHeld) return f(integral_constant<int, 32>{});
  return f(integral_constant<int, 64>{});
}

// Tokens per block: one pass of the block's threads while that leaves the sort
// no more than 256 blocks' counts, then more, up to kTile assignments; all of
// them where four passes of one block do.
static int tile_tokens(int64_t tokens, int experts, int k) {
  int lanes = 1;
  while (lanes * kHeld < experts) lanes *= 2;
  const int pass = std::min(256 / lanes, kTile / k);
  if (tokens <= 4 * pass && tokens * k <= kTile) return static_cast<int>(std::max<int64_t>(tokens, 1));
  const int64_t even = round_up(div_up(tokens, 256), pass);
  return static_cast<int>(std::max<int64_t>(std::min<int64_t>(even, kTile / k / pass * pass), pass));
}

template <class T, class I>
static int launch_combine(const I *h, int64_t rows, const int32_t *slots, const float *weights, int64_t tokens, int k,
                          int c, T *y, hipStream_t stream) {
  return in_slices(div_up(tokens * div_up(c, kVec<T>), 256), [&](int64_t first, dim3 blocks) {
    hipLaunchKernelGGL((combine_kernel<T, I>), blocks, dim3(256), 0, stream, h, rows, slots, weights, first, tokens, k,
                       c, y);
  });
}

static int check(int64_t tokens, int experts, int k) {
  SPIRA_HIP_REQUIRE(experts > 0 && experts <= kMaxExperts, "route: needs 1 to 512 experts");
  SPIRA_HIP_REQUIRE(k > 0 && k <= kMaxChoices && k <= experts, "route: needs 1 to 16 choices, at most the experts");
  SPIRA_HIP_REQUIRE(tokens >= 0 && tokens * k < (int64_t(1) << 31) - kTile, "route: too many tokens");
  return kOk;
}

}  // namespace route

int sum_slots(const float *h, int64_t rows, const int32_t *slots, int64_t tokens, int k, int c, int dtype, void *y,
              hipStream_t stream) {
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return route::launch_combine<T, float>(h, rows, slots, nullptr, tokens, k, c, static_cast<T *>(y), stream);
  });
}

}  // namespace spira_hip

using namespace spira_hip;

extern "C" {

int spira_hip_route_workspace(int64_t tokens, int experts, int k, size_t *bytes) {
  if (int rc = route::check(tokens, experts, k)) return rc;
  const int64_t blocks = div_up(tokens, route::tile_tokens(tokens, experts, k));
  *bytes = static_cast<size_t>((blocks + 1) * (experts + 1)) * sizeof(int32_t);
  return kOk;
}

int spira_hip_route(const void *logits, int64_t tokens, int experts, int k, int dtype, int renormalize, float *weights,
                    int32_t *chosen, int32_t *offsets, int32_t *rows, int32_t *slots, void *workspace,
                    size_t workspace_bytes, hipStream_t stream) {
  if (int rc = route::check(tokens, experts, k)) return rc;
  const int64_t n = tokens * k;
  const int tile = route::tile_tokens(tokens, experts, k);
  const int blocks = static_cast<int>(div_up(tokens, tile));
  SPIRA_HIP_REQUIRE(workspace && workspace_bytes >= static_cast<size_t>((blocks + int64_t(1)) * (experts + 1)) * 4,
                    "route: workspace too small (spira_hip_route_workspace)");
  SPIRA_HIP_REQUIRE(offsets && (n == 0 || (logits && weights && chosen && rows && slots)), "route: null tensor");
  auto *totals = static_cast<int32_t *>(workspace);
  int32_t *counts = totals + experts + 1;
  int bits = 0;
  while ((1 << bits) <= experts) ++bits;
  const route::Order o{experts, k, bits, offsets, rows, slots};
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return route::with_lanes(experts, [&](auto G) -> int {
      constexpr int g = decltype(G)::value;
      const T *l = static_cast<const T *>(logits);
      if (blocks <= 1) {
        hipLaunchKernelGGL((route::route_kernel<T, g>), dim3(1), dim3(256), 0, stream, l, static_cast<int>(tokens),
                           renormalize, weights, chosen, o);
        SPIRA_HIP_LAUNCH_CHECK();
        return kOk;
      }
      hipLaunchKernelGGL((route::choose_kernel<T, g>), dim3(blocks), dim3(256), 0, stream, l, tokens, tile, experts, k,
                         renormalize, weights, chosen, counts);
      SPIRA_HIP_LAUNCH_CHECK();
      // Each block of the second launch reads all counts, a wave a bin: worth it
      // while that is a few microseconds (one launch costs about four).
      const bool summed = (experts + 1) * div_up(blocks, 64) <= 128;
      if (!summed) {
        hipLaunchKernelGGL(route::running_kernel, dim3(experts + 1), dim3(256), 0, stream, blocks, counts, totals);
        SPIRA_HIP_LAUNCH_CHECK();
      }
      hipLaunchKernelGGL(route::rank_kernel, dim3(blocks), dim3(256), 0, stream, chosen, n, tile * k, blocks, counts,
                         summed ? nullptr : totals, o);
      SPIRA_HIP_LAUNCH_CHECK();
      return kOk;
    });
  });
}

int spira_hip_route_backward(const void *logits, int64_t tokens, int experts, int k, int dtype, int renormalize,
                             const float *weights, const int32_t *chosen, const float *dweights, void *dlogits,
                             hipStream_t stream) {
  if (int rc = route::check(tokens, experts, k)) return rc;
  SPIRA_HIP_REQUIRE(tokens == 0 || (logits && weights && chosen && dweights && dlogits), "route_backward: null tensor");
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (tokens == 0) return kOk;
    return route::with_lanes(experts, [&](auto G) -> int {
      constexpr int g = decltype(G)::value;
      return in_slices(div_up(tokens, 256 / g), [&](int64_t first, dim3 blocks) {
        hipLaunchKernelGGL((route::choose_backward_kernel<T, g>), blocks, dim3(256), 0, stream,
                           static_cast<const T *>(logits), weights, chosen, dweights, first, tokens, experts, k,
                           renormalize, static_cast<T *>(dlogits));
      });
    });
  });
}

int spira_hip_combine(const void *h, int64_t num_rows, const int32_t *slots, const float *weights, int64_t tokens,
                      int k, int c, int dtype, void *y, hipStream_t stream) {
  SPIRA_HIP_REQUIRE(tokens >= 0 && num_rows >= 0 && num_rows < (int64_t(1) << 31) && k > 0 && c > 0,
                    "combine: bad sizes");
  SPIRA_HIP_REQUIRE(tokens == 0 || (slots && y && (h || num_rows == 0)), "combine: null tensor");
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return route::launch_combine<T, T>(static_cast<const T *>(h), num_rows, slots, weights, tokens, k, c,
                                       static_cast<T *>(y), stream);
  });
}

int spira_hip_combine_backward(const void *h, int64_t num_rows, const int32_t *rows, const int32_t *slots,
                               const float *weights, const void *dy, int64_t tokens, int k, int c, int dtype, void *dh,
                               float *dweights, hipStream_t stream) {
  SPIRA_HIP_REQUIRE(tokens >= 0 && num_rows >= 0 && num_rows < (int64_t(1) << 31) && k > 0 && c > 0,
                    "combine_backward: bad sizes");
  SPIRA_HIP_REQUIRE((tokens == 0 || (slots && weights && dy)) && (num_rows == 0 || (h && rows)),
                    "combine_backward: null tensor");
  const int64_t token_blocks = div_up(tokens, 16), blocks = token_blocks + (dh ? div_up(num_rows, 16) : 0);
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return in_slices(blocks, [&](int64_t first, dim3 slice) {
      hipLaunchKernelGGL(route::combine_backward_kernel<T>, slice, dim3(256), 0, stream, static_cast<const T *>(h),
                         num_rows, rows, slots, weights, static_cast<const T *>(dy), first, tokens, k, c, token_blocks,
                         static_cast<T *>(dh), dweights);
    });
  });
}

}  // extern "C"
