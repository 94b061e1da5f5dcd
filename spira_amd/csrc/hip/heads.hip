// Norms of the queries and keys of each head and their rotation by positions
// (gfx950), in one pass over both:
//
//   n = x / sqrt(mean(x^2) + eps) * w        (or n = x, without w)
//   y = n, each pair (a, b) of it turned by an angle: (a cos t - b sin t, a sin t + b cos t)
//
// Pair p of d / 2 is (p, p + d / 2), or (2 p, 2 p + 1) interleaved.  With A axes,
// band a of the pairs, a (d / 2) / A to (a + 1) (d / 2) / A, turns by axis a: its pair
// j of n by position[a] base^(-j / n) radians.
//
// A turn's speed is held as a fraction of a whole turn in 64-bit fixed point (in
// the kernel's arguments), so that a position times it, modulo one turn, is an
// integer product and as good at position 2^31 as at 1.  Sines are made once for a
// row, in LDS, for all of its heads.
//
// A block takes a few rows at a time, G lanes a head's vector of a row, eight pairs
// each.  Everything in fp32, outputs rounded once; sums over rows (the gradients of
// w) go over the blocks in a fixed order.  Bound by memory: 200k rows of 6 heads of 32,
// fp16, 52 us where their bytes take 29 (rows lie 576 bytes apart, 384 of them read); 16384
// rows of 20 heads of 64, bf16, 26 us and 37 for the gradients.
#include "numeric.hpp"

#include <algorithm>
#include <cmath>

namespace spira_hip {

namespace heads {

constexpr int kMostDim = 128, kPairs = 8;  // values of a head, pairs a lane

struct Side {  // queries or keys
  const void *x, *w, *dy;
  int64_t row, head;  // strides in values
  int heads;
  void *y;  // [n, heads, d]: outputs or gradients
};
struct Args {
  Side side[2];
  int64_t n;
  int d, axes, rows;  // rows of a block at a time
  float eps;
  const int32_t *positions;  // [n, axes] or null
  float *partial;            // [blocks, 2, d]
  uint64_t speed[kMostDim / 2];  // 2^64 turns of a pair by a position
  uint8_t axis[kMostDim / 2];
};

// cos and sin of `turn` / 2^64 of a whole turn: of what the nearest quarter leaves, at
// most an eighth of a turn, by their series (to x^11: 2e-9 left), then turned by the
// quarter.  Off by 2^-22.7 at most, of which the angle's own three roundings are
// most.
__device__ __forceinline__ float2 turned(uint64_t turn) {
  const uint32_t t = static_cast<uint32_t>(turn >> 32), quarter = (t + 0x20000000u) >> 30;
  const float x = static_cast<float>(static_cast<int32_t>(t - (quarter << 30))) * 1.46291808e-9f;  // 2 pi / 2^32
  const float y = x * x;
  const float s = x + x * y * (-1.f / 6 + y * (1.f / 120 + y * (-1.f / 5040 + y * (1.f / 362880))));
  const float c = 1.f + y * (-0.5f + y * (1.f / 24 + y * (-1.f / 720 + y * (1.f / 40320 - y * (1.f / 3628800)))));
  const float u = quarter & 1 ? s : c, v = quarter & 1 ? c : s;
  return {(quarter + 1) & 2 ? -u : u, quarter & 2 ? -v : v};
}

// a lane's pairs: firsts, then seconds
struct Pairs {
  float a[kPairs], b[kPairs];
};

template <class T> __device__ __forceinline__ void store8(T *p, int at, int n, const float (&v)[kPairs]) {
#pragma unroll
  for (int i = 0; i < kPairs / kVec<T>; ++i) {
    Chunk<T> c;
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) c.v[j] = v[i * kVec<T> + j];
    store_chunk(p + at + i * kVec<T>, n - at - i * kVec<T>, c);
  }
}
template <class T>
__device__ __forceinline__ void store_pairs(T *p, int lane, int d, int half, bool interleaved, const Pairs &r) {
  if (interleaved) {
    float lo[kPairs], hi[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs / 2; ++i) {
      lo[2 * i] = r.a[i];
      lo[2 * i + 1] = r.b[i];
      hi[2 * i] = r.a[kPairs / 2 + i];
      hi[2 * i + 1] = r.b[kPairs / 2 + i];
    }
    store8(p, lane * 2 * kPairs, d, lo);
    store8(p, lane * 2 * kPairs + kPairs, d, hi);
  } else {
    store8(p, lane * kPairs, half, r.a);
    store8(p + half, lane * kPairs, d - half, r.b);
  }
}

// a lane's pairs as they lie in memory
template <class T> struct RawPairs {
  uintx4_t a[kPairs / kVec<T>], b[kPairs / kVec<T>];
};
template <class T>
__device__ __forceinline__ RawPairs<T> load_raw_pairs(const T *p, int lane, int d, int half, bool interleaved) {
  RawPairs<T> r;
  const int first = interleaved ? lane * 2 * kPairs : lane * kPairs, second = interleaved ? first + kPairs : half + first;
  const int upto = interleaved ? d : half;
#pragma unroll
  for (int i = 0; i < kPairs / kVec<T>; ++i) {
    r.a[i] = load_raw(p + first + i * kVec<T>, p ? upto - first - i * kVec<T> : 0);
    r.b[i] = load_raw(p + second + i * kVec<T>, p ? d - second - i * kVec<T> : 0);
  }
  return r;
}
template <class T> __device__ __forceinline__ Pairs unpack_pairs(const RawPairs<T> &raw, bool interleaved) {
  float lo[kPairs], hi[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs / kVec<T>; ++i) {
    const Chunk<T> x = unpack<T>(raw.a[i]), y = unpack<T>(raw.b[i]);
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) {
      lo[i * kVec<T> + j] = x.v[j];
      hi[i * kVec<T> + j] = y.v[j];
    }
  }
  Pairs r;
#pragma unroll
  for (int i = 0; i < kPairs / 2; ++i) {
    r.a[i] = interleaved ? lo[2 * i] : lo[i];
    r.b[i] = interleaved ? lo[2 * i + 1] : hi[i];
    r.a[kPairs / 2 + i] = interleaved ? hi[2 * i] : lo[kPairs / 2 + i];
    r.b[kPairs / 2 + i] = interleaved ? hi[2 * i + 1] : hi[kPairs / 2 + i];
  }
  return r;
}

constexpr int kMostTurns = 2048;  // of the rows that a block holds

// cos and sin of the rows' pairs
__device__ __forceinline__ void make_turns(const Args &a, int64_t first, int count, float2 *turns) {
  const int half = a.d / 2;
  for (int i = threadIdx.x; i < count * half; i += 256) {
    const int r = i / half, p = i - r * half;
    const int64_t at = a.positions[(first + r) * a.axes + a.axis[p]];
    turns[i] = turned(static_cast<uint64_t>(at) * a.speed[p]);
  }
}

// a vector of a block's rows, and the one `by` rows and `more` heads on
struct Item {
  int r, h;
  __device__ __forceinline__ void advance(int by, int more, int heads) {
    r += by;
    h += more;
    if (h >= heads) {
      h -= heads;
      ++r;
    }
  }
};

// A lane's vectors come one turn ahead: the next one's loads are under way while it
// works on this one, and the first's while the sines are made.
template <class T, int G, bool INTERLEAVED> __global__ __launch_bounds__(256) void forward_kernel(const Args a) {
  __shared__ float2 turns[kMostTurns];
  constexpr int GROUPS = 256 / G;
  const int lane = threadIdx.x % G, group = threadIdx.x / G, half = (a.d + 1) / 2;
  const float inv_d = 1.f / static_cast<float>(a.d);
  const int all = a.side[0].heads + a.side[1].heads;
  RawPairs<T> w[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) w[s] = load_raw_pairs(static_cast<const T *>(a.side[s].w), lane, a.d, half, INTERLEAVED);
  for (int64_t first = blockIdx.x * static_cast<int64_t>(a.rows); first < a.n; first += gridDim.x * static_cast<int64_t>(a.rows)) {
    const int rows = static_cast<int>(std::min<int64_t>(a.rows, a.n - first));
    Item at{group / all, group % all}, then = at;
    const auto fetch = [&](const Item &at) {
      const int k = at.h >= a.side[0].heads;
      const T *x = static_cast<const T *>(k ? a.side[1].x : a.side[0].x);
      const int64_t row = k ? a.side[1].row : a.side[0].row, head = k ? a.side[1].head : a.side[0].head;
      return load_raw_pairs(at.r < rows ? x + (first + at.r) * row + (k ? at.h - a.side[0].heads : at.h) * head : nullptr,
                            lane, a.d, half, INTERLEAVED);
    };
    RawPairs<T> next = fetch(at);
    if (a.positions) {
      __syncthreads();
      make_turns(a, first, rows, turns);
      __syncthreads();
    }
    for (; at.r < rows; at = then) {
      const int r = at.r, h = at.h, k = h >= a.side[0].heads;
      Pairs v = unpack_pairs<T>(next, INTERLEAVED);
      then.advance(GROUPS / all, GROUPS % all, all);
      next = fetch(then);
      if (k ? a.side[1].w : a.side[0].w) {
        float ss = 0;
#pragma unroll
        for (int j = 0; j < kPairs; ++j) ss += v.a[j] * v.a[j] + v.b[j] * v.b[j];
        const float inv = rsqrtf(group_sum<G>(ss) * inv_d + a.eps);
        RawPairs<T> raw;
#pragma unroll
        for (int j = 0; j < kPairs / kVec<T>; ++j) {
          raw.a[j] = k ? w[1].a[j] : w[0].a[j];
          raw.b[j] = k ? w[1].b[j] : w[0].b[j];
        }
        const Pairs by = unpack_pairs<T>(raw, INTERLEAVED);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          v.a[j] *= inv * by.a[j];
          v.b[j] *= inv * by.b[j];
        }
      }
      if (a.positions) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const int p = lane * kPairs + j;
          const float2 t = turns[r * half + (p < half ? p : 0)];
          const float x = v.a[j], y = v.b[j];
          v.a[j] = x * t.x - y * t.y;
          v.b[j] = x * t.y + y * t.x;
        }
      }
      const int64_t to = k ? (first + r) * a.side[1].heads + h - a.side[0].heads : (first + r) * a.side[0].heads + h;
      store_pairs(static_cast<T *>(k ? a.side[1].y : a.side[0].y) + to * a.d, lane, a.d, half, INTERLEAVED, v);
    }
  }
}

template <class T, int G, bool INTERLEAVED> __global__ __launch_bounds__(256) void backward_kernel(const Args a) {
  __shared__ float2 turns[kMostTurns];
  constexpr int GROUPS = 256 / G;
  const int lane = threadIdx.x % G, group = threadIdx.x / G, half = (a.d + 1) / 2;
  const float inv_d = 1.f / static_cast<float>(a.d);
  Pairs dw[2] = {};
  for (int64_t first = blockIdx.x * static_cast<int64_t>(a.rows); first < a.n; first += gridDim.x * static_cast<int64_t>(a.rows)) {
    const int count = static_cast<int>(std::min<int64_t>(a.rows, a.n - first));
    if (a.positions) {
      __syncthreads();
      make_turns(a, first, count, turns);
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const Side &side = a.side[k];
      if (!side.dy) continue;
      const RawPairs<T> w_raw = load_raw_pairs(static_cast<const T *>(side.w), lane, a.d, half, INTERLEAVED);
      RawPairs<T> next_g, next_x;
      Item item{group / side.heads, group % side.heads}, then = item;
      const auto fetch = [&](const Item &x) {
        const bool there = x.r < count;
        const int64_t at = ((first + x.r) * side.heads + x.h) * a.d;
        next_g = load_raw_pairs(there ? static_cast<const T *>(side.dy) + at : nullptr, lane, a.d, half, INTERLEAVED);
        next_x = load_raw_pairs(there && side.w ? static_cast<const T *>(side.x) + (first + x.r) * side.row + x.h * side.head : nullptr,
                                lane, a.d, half, INTERLEAVED);
      };
      fetch(item);
      for (; item.r < count; item = then) {
        const int r = item.r;
        const int64_t at = ((first + r) * side.heads + item.h) * a.d;
        Pairs g = unpack_pairs<T>(next_g, INTERLEAVED), v = unpack_pairs<T>(next_x, INTERLEAVED);
        then.advance(GROUPS / side.heads, GROUPS % side.heads, side.heads);
        fetch(then);
        if (a.positions) {
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            const int p = lane * kPairs + j;
            const float2 t = turns[r * half + (p < half ? p : 0)];
            const float x = g.a[j], y = g.b[j];
            g.a[j] = x * t.x + y * t.y;
            g.b[j] = y * t.x - x * t.y;
          }
        }
        if (side.w) {
          float ss = 0, along = 0;
#pragma unroll
          for (int j = 0; j < kPairs; ++j) ss += v.a[j] * v.a[j] + v.b[j] * v.b[j];
          const float inv = rsqrtf(group_sum<G>(ss) * inv_d + a.eps);
          const Pairs w = unpack_pairs<T>(w_raw, INTERLEAVED);
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            v.a[j] *= inv;
            v.b[j] *= inv;
            dw[k].a[j] += g.a[j] * v.a[j];
            dw[k].b[j] += g.b[j] * v.b[j];
            g.a[j] *= w.a[j];
            g.b[j] *= w.b[j];
            along += g.a[j] * v.a[j] + g.b[j] * v.b[j];
          }
          along = group_sum<G>(along) * inv_d;
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            g.a[j] = inv * (g.a[j] - v.a[j] * along);
            g.b[j] = inv * (g.b[j] - v.b[j] * along);
          }
        }
        if (side.y) store_pairs(static_cast<T *>(side.y) + at, lane, a.d, half, INTERLEAVED, g);
      }
    }
  }
  if (!a.partial) return;
  // the block's groups in order, by way of LDS, a side at a time
  float *sums = reinterpret_cast<float *>(turns);  // [4, 128]: the waves' sums
  static_assert(sizeof(turns) >= 4 * kMostDim * sizeof(float), "room for the waves' sums");
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int j = 0; j < kPairs; ++j)
#pragma unroll
      for (int o = G; o < 64; o *= 2) {
        dw[k].a[j] += __shfl_xor(dw[k].a[j], o, 64);
        dw[k].b[j] += __shfl_xor(dw[k].b[j], o, 64);
      }
    __syncthreads();
    if ((threadIdx.x & 63) < G) {
      float *to = sums + (threadIdx.x >> 6) * kMostDim;
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const int p = lane * kPairs + j, x = INTERLEAVED ? 2 * p : p, y = INTERLEAVED ? 2 * p + 1 : half + p;
        if (p < half) to[x] = dw[k].a[j];
        if (p < half && y < a.d) to[y] = dw[k].b[j];
      }
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < a.d) {
      float s = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) s += sums[q * kMostDim + threadIdx.x];
      a.partial[(blockIdx.x * static_cast<int64_t>(2) + k) * a.d + threadIdx.x] = s;
    }
  }
}

// columns of the blocks' sums: 16 columns a block, 64 threads to each, joined in a
// fixed tree
template <class T>
__global__ __launch_bounds__(1024) void columns_kernel(const float *partial, int blocks, int d, void *dwq, void *dwk) {
  __shared__ float s[64][17];
  T *to = static_cast<T *>(blockIdx.y == 0 ? dwq : dwk);
  if (!to) return;
  const int col = blockIdx.x * 16 + threadIdx.x % 16, q = threadIdx.x / 16;
  float v = 0;
  if (col < d)
    for (int b = q; b < blocks; b += 64) v += partial[(b * static_cast<int64_t>(2) + blockIdx.y) * d + col];
  s[q][threadIdx.x % 16] = v;
  __syncthreads();
  for (int half = 32; half > 0; half /= 2) {
    if (q < half) s[q][threadIdx.x % 16] += s[q + half][threadIdx.x % 16];
    __syncthreads();
  }
  if (q == 0 && col < d) to[col] = from_float<T>(s[0][threadIdx.x]);
}

// f(lanes of a head's vector)
template <class F> int with_lanes(int d, F &&f) {
  using std::integral_constant;
  const int64_t lanes = div_up((d + 1) / 2, kPairs);
  if (lanes <= 1) return f(integral_constant<int, 1>{});
  if (lanes <= 2) return f(integral_constant<int, 2>{});
  if (lanes <= 4) return f(integral_constant<int, 4>{});
  return f(integral_constant<int, 8>{});
}

static int check(const spira_hip_heads_t &x) {
  SPIRA_HIP_REQUIRE(x.rows >= 0 && x.rows < (int64_t(1) << 31), "norm_rotate_heads: bad number of rows");
  SPIRA_HIP_REQUIRE(x.heads > 0 && x.kv_heads > 0 && x.heads <= 65536 && x.kv_heads <= 65536,
                    "norm_rotate_heads: needs 1 to 65536 heads");
  SPIRA_HIP_REQUIRE(x.head_dim > 0 && x.head_dim <= kMostDim, "norm_rotate_heads: needs heads of 1 to 128 values");
  SPIRA_HIP_REQUIRE(x.rows == 0 || (x.queries && x.key), "norm_rotate_heads: null features");
  if (x.axes > 0) {
    SPIRA_HIP_REQUIRE(x.rows == 0 || x.positions, "norm_rotate_heads: null positions");
    SPIRA_HIP_REQUIRE(x.head_dim % 2 == 0 && x.axes <= x.head_dim / 2,
                      "norm_rotate_heads: a rotation needs an even number of values and a pair for each axis");
    SPIRA_HIP_REQUIRE(x.base > 0 && x.base < HUGE_VAL, "norm_rotate_heads: the base must be positive and finite");
  } else {
    SPIRA_HIP_REQUIRE(x.axes == 0, "norm_rotate_heads: bad number of axes");
  }
  return kOk;
}

// Rows that a block takes at a time: some 1024 lanes' vectors, as many sines as LDS
// holds, and no fewer blocks than the CUs have room for.
static int block_rows(const spira_hip_heads_t &x, int lanes) {
  const int64_t vectors = static_cast<int64_t>(x.heads + x.kv_heads) * lanes;
  int64_t rows = std::max<int64_t>(1, 1024 / vectors);
  rows = std::min<int64_t>(rows, kMostTurns / std::max(1, x.head_dim / 2));
  return static_cast<int>(std::max<int64_t>(1, std::min(rows, div_up(x.rows, 1024))));
}
static int64_t blocks_of(const spira_hip_heads_t &x, int lanes, int most) {
  return std::min<int64_t>(div_up(x.rows, block_rows(x, lanes)), most);
}
constexpr int kForwardBlocks = 1 << 23, kBackwardBlocks = 512;

// Turns of the pairs by a position, and their axes, in long double: 64 bits of the turn's
// fraction.  A band's speeds are a geometric row: one power, then products, whose roundings
// leave 2^-58 of a speed (2^-26 radians at position 2^31, below fp32's own).  A power each
// takes longer than a launch: 32 of them 14 us.
static void speeds(double base, int pairs, int axes, uint64_t *speed, uint8_t *axis) {
  for (int a = 0; a < axes; ++a) {
    const int lo = a * pairs / axes, hi = (a + 1) * pairs / axes;
    const long double by = hi - lo > 1 ? powl(static_cast<long double>(base), -1.0L / (hi - lo)) : 1.0L;
    long double turns = 1 / 6.283185307179586476925286766559L;
    for (int p = lo; p < hi; ++p, turns *= by) {
      // (a fraction of 64 bits is below 2^64 times it)
      speed[p] = static_cast<uint64_t>((turns < 1 ? turns : turns - floorl(turns)) * 18446744073709551616.0L);
      axis[p] = static_cast<uint8_t>(a);
    }
  }
}

static Args arguments(const spira_hip_heads_t &x, int lanes) {
  Args a{};
  a.side[0] = {x.queries, x.query_weight, nullptr, x.query_row, x.query_head, x.heads, nullptr};
  a.side[1] = {x.key, x.key_weight, nullptr, x.key_row, x.key_head, x.kv_heads, nullptr};
  a.n = x.rows;
  a.d = x.head_dim;
  a.axes = x.axes;
  a.rows = block_rows(x, lanes);
  a.eps = x.eps;
  if (x.axes > 0) {
    a.positions = x.positions;
    speeds(x.base, x.head_dim / 2, x.axes, a.speed, a.axis);
  }
  return a;
}

}  // namespace heads

}  // namespace spira_hip

using namespace spira_hip;

extern "C" {

int spira_hip_norm_rotate_heads(const spira_hip_heads_t *x, void *queries, void *key, hipStream_t stream) {
  SPIRA_HIP_REQUIRE(x, "norm_rotate_heads: null arguments");
  if (int rc = heads::check(*x)) return rc;
  if (x->rows == 0) return kOk;
  SPIRA_HIP_REQUIRE(queries && key, "norm_rotate_heads: null outputs");
  return with_type(x->dtype, [&](auto t) -> int {
    return heads::with_lanes(x->head_dim, [&](auto G) -> int {
      constexpr int g = decltype(G)::value;
      heads::Args a = heads::arguments(*x, g);
      a.side[0].y = queries;
      a.side[1].y = key;
      using T = decltype(t);
      const auto kernel = x->interleaved ? heads::forward_kernel<T, g, true> : heads::forward_kernel<T, g, false>;
      hipLaunchKernelGGL(kernel, dim3(heads::blocks_of(*x, g, heads::kForwardBlocks)), dim3(256), 0, stream, a);
      SPIRA_HIP_LAUNCH_CHECK();
      return kOk;
    });
  });
}

int spira_hip_norm_rotate_heads_backward_workspace(const spira_hip_heads_t *x, size_t *bytes) {
  SPIRA_HIP_REQUIRE(x && bytes, "norm_rotate_heads: null arguments");
  if (int rc = heads::check(*x)) return rc;
  return heads::with_lanes(x->head_dim, [&](auto G) -> int {
    *bytes = static_cast<size_t>(heads::blocks_of(*x, decltype(G)::value, heads::kBackwardBlocks)) * 2 * x->head_dim *
             sizeof(float);
    return kOk;
  });
}

int spira_hip_norm_rotate_heads_backward(const spira_hip_heads_t *x, const void *dout_queries, const void *dout_key,
                                         void *dqueries, void *dkey, void *dquery_weight, void *dkey_weight,
                                         void *workspace, size_t workspace_bytes, hipStream_t stream) {
  SPIRA_HIP_REQUIRE(x, "norm_rotate_heads: null arguments");
  if (int rc = heads::check(*x)) return rc;
  SPIRA_HIP_REQUIRE((x->query_weight || !dquery_weight) && (x->key_weight || !dkey_weight),
                    "norm_rotate_heads: a gradient of no weight");
  // (tensors without rows may have no address)
  SPIRA_HIP_REQUIRE(x->rows == 0 || ((dout_queries || !(dqueries || dquery_weight)) && (dout_key || !(dkey || dkey_weight))),
                    "norm_rotate_heads: null gradients");
  return with_type(x->dtype, [&](auto t) -> int {
    using T = decltype(t);
    return heads::with_lanes(x->head_dim, [&](auto G) -> int {
      constexpr int g = decltype(G)::value;
      const int64_t blocks = heads::blocks_of(*x, g, heads::kBackwardBlocks);
      heads::Args a = heads::arguments(*x, g);
      a.side[0].dy = dqueries || dquery_weight ? dout_queries : nullptr;
      a.side[1].dy = dkey || dkey_weight ? dout_key : nullptr;
      a.side[0].y = dqueries;
      a.side[1].y = dkey;
      if (dquery_weight || dkey_weight) {
        SPIRA_HIP_REQUIRE(workspace_bytes >= static_cast<size_t>(blocks) * 2 * x->head_dim * sizeof(float) &&
                              (workspace || blocks == 0),
                          "norm_rotate_heads: workspace too small");
        a.partial = static_cast<float *>(workspace);
      }
      if (blocks > 0) {
        const auto kernel = x->interleaved ? heads::backward_kernel<T, g, true> : heads::backward_kernel<T, g, false>;
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, a);
        SPIRA_HIP_LAUNCH_CHECK();
      }
      if (dquery_weight || dkey_weight) {
        hipLaunchKernelGGL(heads::columns_kernel<T>, dim3(div_up(x->head_dim, 16), 2), dim3(1024), 0, stream, a.partial,
                           static_cast<int>(blocks), x->head_dim, dquery_weight, dkey_weight);
        SPIRA_HIP_LAUNCH_CHECK();
      }
      return kOk;
    });
  });
}

}  // extern "C"
