// The balance loss of a router (gfx950):
//
//   p[t] = softmax(logits[t]) over the experts that are not masked (-inf)
//   P[e] = mean of p[t, e] over the tokens that have an expert
//   f[e] = share of the assignments that went to e
//   L = E sum_e f[e] P[e]            dL/dl[t, e] = E / tokens p[t, e] (f[e] - sum_j p[t, j] f[j])
//
// (1 where the router is even.)  f counts choices and has no gradient.  G lanes
// hold a token's logits, eight each, and add the tokens' p up in registers; the
// blocks' sums are added in order by one block, which makes the loss.  Few tokens
// take one launch.  The backward pass makes p again from the logits: what a kept p
// would cost to write and read is more.  100k tokens of 16 experts: 6.3 us and 7.6 for the
// loss, the gradient 5.0, where the bytes take 2: the launches' latency.
#include "numeric.hpp"

#include <algorithm>

namespace spira_hip {

namespace balance {

constexpr int kMostExperts = 512, kHeld = 8;

// A token's probabilities by G lanes, eight experts each; whether it has an expert.
template <class T, int G>
__device__ __forceinline__ bool softmax(const T *logits, int experts, int lane, float (&p)[kHeld]) {
#pragma unroll
  for (int i = 0; i < kHeld / kVec<T>; ++i) {
    const int at = lane * kHeld + i * kVec<T>;
    const Chunk<T> c = load_chunk(logits + at, experts - at);
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) p[i * kVec<T> + j] = at + j < experts ? c.v[j] : -__builtin_inff();
  }
  float top = p[0];
#pragma unroll
  for (int i = 1; i < kHeld; ++i) top = fmaxf(top, p[i]);
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  // (NaN stays, as its exponential and in the sum)
  const float base = top == -__builtin_inff() ? 0.f : top;
  float sum = 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    p[i] = expf(p[i] - base);
    sum += p[i];
  }
  sum = group_sum<G>(sum);
  const bool some = !(sum == 0.f);
  const float by = some ? 1.f / sum : 0.f;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) p[i] *= by;
  return some;
}

struct Args {
  const void *logits;
  int64_t tokens;
  int experts, blocks;
  const int32_t *offsets;  // [experts + 1] of the assignments
  float *partial;          // [blocks, experts + 1]: sums of p, tokens that have an expert
  float *loss, *mean, *kept;  // kept: f [experts], E / tokens
  int32_t *counts;
};

// sum over the block's 1024 (NT) threads, the same in each
template <int NT> __device__ __forceinline__ float block_sum(float v, float *shared) {
  v = group_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s += shared[i];
  return s;
}

// The loss from the experts' sums: thread e has expert e's.
template <int NT> __device__ __forceinline__ void finish(const Args &a, const float *sums, float *shared) {
  const int e = threadIdx.x;
  const bool there = e < a.experts;
  const int32_t n = there ? a.offsets[e + 1] - a.offsets[e] : 0;
  // (the assignments are consecutive: their number is exact)
  const float all = static_cast<float>(a.offsets[a.experts] - a.offsets[0]), tokens = sums[a.experts];
  const float share = all > 0.f ? static_cast<float>(n) / all : 0.f;
  const float mean = there && tokens > 0.f ? sums[e] / tokens : 0.f;
  const float loss = block_sum<NT>(share * mean, shared) * static_cast<float>(a.experts);
  if (there) {
    a.counts[e] = n;
    a.mean[e] = mean;
    a.kept[e] = share;
  }
  if (e == 0) {
    *a.loss = loss;
    a.kept[a.experts] = tokens > 0.f ? static_cast<float>(a.experts) / tokens : 0.f;
  }
}

// ONE: the only block, which makes the loss too
template <class T, int G, bool ONE> __global__ __launch_bounds__(512) void sums_kernel(const Args a) {
  constexpr int NT = 512, TOKENS = NT / G;
  __shared__ float part[8][G * kHeld + 1], total[kMostExperts + 1], shared[8];
  const int lane = threadIdx.x % G, wave = threadIdx.x >> 6;
  float sum[kHeld] = {}, n = 0;
  for (int64_t t = blockIdx.x * static_cast<int64_t>(TOKENS) + threadIdx.x / G; t < a.tokens;
       t += gridDim.x * static_cast<int64_t>(TOKENS)) {
    float p[kHeld];
    const bool some = softmax<T, G>(static_cast<const T *>(a.logits) + t * a.experts, a.experts, lane, p);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) sum[i] += p[i];
    n += some ? 1.f : 0.f;
  }
  // the groups of a wave, then the waves in order
#pragma unroll
  for (int o = G; o < 64; o *= 2) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) sum[i] += __shfl_xor(sum[i], o, 64);
    n += __shfl_xor(n, o, 64);
  }
  if ((threadIdx.x & 63) < G) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) part[wave][lane * kHeld + i] = sum[i];
    if (lane == 0) part[wave][G * kHeld] = n;
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= a.experts; e += NT) {
    float s = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += part[w][e < a.experts ? e : G * kHeld];
    if constexpr (ONE) total[e] = s;
    else a.partial[blockIdx.x * static_cast<int64_t>(a.experts + 1) + e] = s;
  }
  if constexpr (ONE) {
    __syncthreads();
    finish<NT>(a, total, shared);
  }
}

// the blocks' sums, `rows` threads to a column, joined in order
__global__ __launch_bounds__(1024) void loss_kernel(const Args a) {
  __shared__ float part[1024 + 512], total[kMostExperts + 1], shared[16];
  const int width = a.experts + 1, rows = 1024 / width;
  const int e = threadIdx.x % width, r = threadIdx.x / width;
  float s = 0;
  if (r < rows) {
#pragma unroll 8
    for (int b = r; b < a.blocks; b += rows) s += a.partial[b * static_cast<int64_t>(width) + e];
    part[r * width + e] = s;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < width; i += 1024) {
    float v = 0;
    for (int q = 0; q < rows; ++q) v += part[q * width + i];
    total[i] = v;
  }
  __syncthreads();
  finish<1024>(a, total, shared);
}

template <class T, int G>
__global__ __launch_bounds__(256) void backward_kernel(const T *logits, int64_t tokens, int experts, const float *kept,
                                                       const float *dloss, T *dlogits) {
  const int lane = threadIdx.x % G;
  float f[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) f[i] = lane * kHeld + i < experts ? kept[lane * kHeld + i] : 0.f;
  const float by = *dloss * kept[experts];
  for (int64_t t = blockIdx.x * static_cast<int64_t>(256 / G) + threadIdx.x / G; t < tokens;
       t += gridDim.x * static_cast<int64_t>(256 / G)) {
    float p[kHeld], along = 0;
    softmax<T, G>(logits + t * experts, experts, lane, p);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) along += p[i] * f[i];
    along = group_sum<G>(along);
#pragma unroll
    for (int i = 0; i < kHeld / kVec<T>; ++i) {
      Chunk<T> c;
#pragma unroll
      for (int j = 0; j < kVec<T>; ++j) c.v[j] = by * p[i * kVec<T> + j] * (f[i * kVec<T> + j] - along);
      const int at = lane * kHeld + i * kVec<T>;
      store_chunk(dlogits + t * experts + at, experts - at, c);
    }
  }
}

// f(lanes of a token)
template <class F> int with_lanes(int experts, F &&f) {
  using std::integral_constant;
  const int64_t lanes = div_up(experts, kHeld);
  if (lanes <= 1) return f(integral_constant<int, 1>{});
  if (lanes <= 2) return f(integral_constant<int, 2>{});
  if (lanes <= 4) return f(integral_constant<int, 4>{});
  if (lanes <= 8) return f(integral_constant<int, 8>{});
  if (lanes <= 16) return f(integral_constant<int, 16>{});
  if (lanes <= 32) return f(integral_constant<int, 32>{});
  return f(integral_constant<int, 64>{});
}

static int check(int64_t tokens, int experts) {
  SPIRA_HIP_REQUIRE(tokens >= 0 && tokens < (int64_t(1) << 31), "balance_loss: bad number of tokens");
  SPIRA_HIP_REQUIRE(experts > 0 && experts <= kMostExperts, "balance_loss: needs 1 to 512 experts");
  return kOk;
}

// Blocks of the sums: two to a CU, each four turns or more, and no more sums than one
// block adds up in a few loads a thread.
static int blocks_of(int64_t tokens, int experts, int lanes) {
  const int64_t turns = div_up(tokens, 4 * (512 / lanes));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({turns, 512, 65536 / (experts + 1)})));
}

}  // namespace balance

}  // namespace spira_hip

using namespace spira_hip;

extern "C" {

int spira_hip_balance_workspace(int64_t tokens, int experts, size_t *bytes) {
  SPIRA_HIP_REQUIRE(bytes, "balance_loss: null arguments");
  if (int rc = balance::check(tokens, experts)) return rc;
  return balance::with_lanes(experts, [&](auto G) -> int {
    const int blocks = balance::blocks_of(tokens, experts, decltype(G)::value);
    *bytes = blocks > 1 ? static_cast<size_t>(blocks) * (experts + 1) * sizeof(float) : 0;
    return kOk;
  });
}

int spira_hip_balance(const void *logits, int64_t tokens, int experts, int dtype, const int32_t *offsets, float *loss,
                      int32_t *counts, float *probabilities, float *kept, void *workspace, size_t workspace_bytes,
                      hipStream_t stream) {
  if (int rc = balance::check(tokens, experts)) return rc;
  SPIRA_HIP_REQUIRE((tokens == 0 || logits) && offsets && loss && counts && probabilities && kept,
                    "balance_loss: null arguments");
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return balance::with_lanes(experts, [&](auto G) -> int {
      constexpr int g = decltype(G)::value;
      const int blocks = balance::blocks_of(tokens, experts, g);
      balance::Args a{logits, tokens, experts, blocks, offsets, nullptr, loss, probabilities, kept, counts};
      if (blocks == 1) {
        hipLaunchKernelGGL((balance::sums_kernel<T, g, true>), dim3(1), dim3(512), 0, stream, a);
        SPIRA_HIP_LAUNCH_CHECK();
        return kOk;
      }
      SPIRA_HIP_REQUIRE(workspace && workspace_bytes >= static_cast<size_t>(blocks) * (experts + 1) * sizeof(float),
                        "balance_loss: workspace too small");
      a.partial = static_cast<float *>(workspace);
      hipLaunchKernelGGL((balance::sums_kernel<T, g, false>), dim3(blocks), dim3(512), 0, stream, a);
      SPIRA_HIP_LAUNCH_CHECK();
      hipLaunchKernelGGL(balance::loss_kernel, dim3(1), dim3(1024), 0, stream, a);
      SPIRA_HIP_LAUNCH_CHECK();
      return kOk;
    });
  });
}

int spira_hip_balance_backward(const void *logits, int64_t tokens, int experts, int dtype, const float *kept,
                               const float *dloss, void *dlogits, hipStream_t stream) {
  if (int rc = balance::check(tokens, experts)) return rc;
  if (tokens == 0) return kOk;
  SPIRA_HIP_REQUIRE(logits && kept && dloss && dlogits, "balance_loss: null arguments");
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return balance::with_lanes(experts, [&](auto G) -> int {
      constexpr int g = decltype(G)::value;
      const int64_t blocks = std::min<int64_t>(div_up(tokens, 256 / g), 4096);
      hipLaunchKernelGGL((balance::backward_kernel<T, g>), dim3(blocks), dim3(256), 0, stream,
                         static_cast<const T *>(logits), tokens, experts, kept, dloss, static_cast<T *>(dlogits));
      SPIRA_HIP_LAUNCH_CHECK();
      return kOk;
    });
  });
}

}  // extern "C"
