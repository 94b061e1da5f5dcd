// Dropout from a counter-based generator (gfx950): element i of the row-major
// features is kept where word i % 4 of philox4x32-7(counter (i / 4, offset),
// key seed) is at least floor(p 2^32), so that the gradient makes the same mask
// again and none is stored.
//
// Philox: Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3" (SC 2011).  Seven rounds are the fewest that pass their test
// batteries; the rounds' 32-bit multiplications, a quarter of the vector rate,
// are what a chunk costs next to its bytes.
#include "numeric.hpp"

namespace spira_hip {

namespace dropout {

struct Words {
  uint32_t v[4];
};

__device__ __forceinline__ Words philox(uint64_t counter, uint64_t offset, uint64_t seed) {
  uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32);
  uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int round = 0; round < 7; ++round) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// (threshold: 2^32 where nothing is kept.  A dropped value is not multiplied, so
// that what it holds, infinities and NaN too, does not come through.)
template <class T>
__global__ __launch_bounds__(256) void dropout_kernel(const T *x, const T *residual, int64_t first, int64_t n,
                                                      uint64_t threshold, float scale, uint64_t seed, uint64_t offset,
                                                      T *y) {
  const int64_t i = ((first + blockIdx.x) * 256 + threadIdx.x) * kVec<T>;
  if (i >= n) return;
  Chunk<T> c = load_chunk(x + i, n - i);
#pragma unroll
  for (int w = 0; w < kVec<T> / 4; ++w) {
    const Words r = philox(static_cast<uint64_t>(i / 4 + w), offset, seed);
#pragma unroll
    for (int j = 0; j < 4; ++j) c.v[4 * w + j] = r.v[j] >= threshold ? c.v[4 * w + j] * scale : 0.f;
  }
  if (residual) {
    const Chunk<T> add = load_chunk(residual + i, n - i);
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) c.v[j] += add.v[j];
  }
  store_chunk(y + i, n - i, c);
}

}  // namespace dropout

}  // namespace spira_hip

using namespace spira_hip;

extern "C" int spira_hip_dropout(const void *x, const void *residual, int64_t n, int dtype, double p, uint64_t seed,
                                 uint64_t offset, void *y, hipStream_t stream) {
  SPIRA_HIP_REQUIRE(p >= 0.0 && p <= 1.0, "dropout: p must be in [0, 1]");
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (n <= 0) return kOk;
    SPIRA_HIP_REQUIRE(n < (int64_t(1) << 38), "dropout: too many elements");
    SPIRA_HIP_REQUIRE(x && y, "dropout: null features");
    const auto threshold = static_cast<uint64_t>(p * 4294967296.0);
    const float scale = p < 1.0 ? static_cast<float>(1.0 / (1.0 - p)) : 0.f;
    return in_slices(div_up(n, 256 * kVec<T>), [&](int64_t first, dim3 blocks) {
      hipLaunchKernelGGL(dropout::dropout_kernel<T>, blocks, dim3(256), 0, stream, static_cast<const T *>(x),
                         static_cast<const T *>(residual), first, n, threshold, scale, seed, offset,
                         static_cast<T *>(y));
    });
  });
}
