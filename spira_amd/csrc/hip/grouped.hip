// Products grouped by expert (gfx950): group e holds rows offsets[e] to
// offsets[e + 1], any number of them, and has its own weights W[e]
// [c_in, c_out].
//
//   forward   y[r]  = act(x[source(r)] W[e] + b[e])
//   rows'     dx[r] = dz[r] W[e]^T
//   weights'  dW[e] = sum_r x[source(r)]^T dz[r],  db[e] = sum_r dz[r]
//
// One tile core serves all three.  An operand's tile lies in LDS either with
// the summed index along its rows of 128 bytes (KC: features; weights of the
// rows' gradient), or with it across (KO: weights of the forward pass; both
// operands of the weights' gradient), as it lies in memory: no operand is
// transposed beforehand, the 16-bit KO fragments are transposed by the LDS read
// itself (ds_read_b64_tr_b16).
//
// Which group a tile belongs to, each wave finds out by itself from the offsets,
// on the device: nothing is read back, and uneven groups cost whole tiles only
// at their ends.  Offsets that are no ascending row numbers cannot lead a tile
// out of the arrays (they are clamped), and rows outside all groups get zeros.
//
// A wave multiplies with the weights as the first operand, so that a lane holds
// four consecutive output channels of one row.
#include "numeric.hpp"

#include <algorithm>

namespace spira_hip {

namespace grouped {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) short4v lds_short4;
typedef __attribute__((address_space(3))) void lds_void;

// ---------------------------------------------------------------------------
// groups
// ---------------------------------------------------------------------------
struct Groups {
  const int32_t *offsets;  // [count + 1]
  int count;
  int64_t rows;
};

struct Part {
  int group;  // -1: the index lies past the last part, `begin` parts after it
  int64_t begin, end;
};

__device__ __forceinline__ int64_t bound(const Groups &g, int i) {
  const int64_t v = g.offsets[i];
  return v < 0 ? 0 : v > g.rows ? g.rows : v;
}

// Part `index` of the groups cut into parts of `size` rows, in group order; the
// same on every lane of the wave.  Lanes count the parts of 64 groups at a time.
__device__ __forceinline__ Part find_part(const Groups &g, int size, int64_t index) {
  const int lane = lane_id();
  int64_t before = 0;
  for (int first = 0; first < g.count; first += 64) {
    const int e = first + lane;
    const int64_t lo = e < g.count ? bound(g, e) : 0, hi = e < g.count ? bound(g, e + 1) : 0;
    const int parts = hi > lo ? static_cast<int>((hi - lo + size - 1) / size) : 0;
    int upto = parts;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int u = __shfl_up(upto, o, 64);
      if (lane >= o) upto += u;
    }
    const uint64_t past = ballot(before + upto > index);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int64_t nth = index - before - (__shfl(upto, at, 64) - __shfl(parts, at, 64));
      const int64_t begin = __shfl(lo, at, 64) + nth * size, end = __shfl(hi, at, 64);
      return {uniform(first + at), uniform(begin), uniform(begin + size < end ? begin + size : end)};
    }
    before += __shfl(upto, 63, 64);
  }
  return {-1, uniform(index - before), 0};
}

// the first part of group `group`, and how many it has
__device__ __forceinline__ void parts_of(const Groups &g, int size, int group, int64_t &first, int64_t &count) {
  const int lane = lane_id();
  int64_t sum = 0;
  for (int e = lane; e < group; e += 64) {
    const int64_t n = bound(g, e + 1) - bound(g, e);
    sum += n > 0 ? (n + size - 1) / size : 0;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  const int64_t n = bound(g, group + 1) - bound(g, group);
  first = sum;
  count = n > 0 ? (n + size - 1) / size : 0;
}

// parts of all groups
__device__ __forceinline__ int64_t count_parts(const Groups &g, int size) {
  int64_t first, count;
  parts_of(g, size, g.count - 1, first, count);
  return first + count;
}

// Block w's place among `count` pieces of work so that each of the 8 XCDs (w %
// 8) takes one range of them; w itself past them.
__device__ __forceinline__ uint32_t xcd_order(uint32_t w, uint32_t count) {
  if (w >= count) return w;
  const uint32_t q = count / 8, r = count % 8, x = w % 8;
  return x * q + (x < r ? x : r) + w / 8;
}

// Block w's part and column among parts x cols, in XCD order: the columns of a
// part together, so that an XCD's L2 holds a few parts' rows and a group's
// weights.  Past the last, part.begin counts the blocks and `idle` is their number.
struct Place {
  Part part;
  uint32_t col;
  int64_t idle;
};
__device__ __forceinline__ Place find_place(const Groups &g, int size, uint32_t w, uint32_t cols, uint32_t blocks) {
  if (g.count > 64) {
    const uint32_t work = static_cast<uint32_t>(count_parts(g, size)) * cols, at = xcd_order(w, work);
    if (at >= work) return {{-1, at - work, 0}, 0, blocks - work};
    return {find_part(g, size, at / cols), at % cols, 0};
  }
  // (the offsets read once)
  const int lane = lane_id();
  const int64_t lo = lane < g.count ? bound(g, lane) : 0, hi = lane < g.count ? bound(g, lane + 1) : 0;
  const uint32_t parts = hi > lo ? static_cast<uint32_t>(hi - lo + size - 1) / size : 0;
  uint32_t upto = parts;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const uint32_t u = __shfl_up(upto, o, 64);
    if (lane >= o) upto += u;
  }
  const uint32_t work = uniform(__shfl(upto, 63, 64)) * cols, at = xcd_order(w, work);
  if (at >= work) return {{-1, at - work, 0}, 0, blocks - work};
  const uint32_t index = at / cols;
  const int e = __builtin_ctzll(ballot(upto > index));
  const int64_t nth = index - (__shfl(upto, e, 64) - __shfl(parts, e, 64));
  const int64_t begin = __shfl(lo, e, 64) + nth * size, end = __shfl(hi, e, 64);
  return {{uniform(e), uniform(begin), uniform(begin + size < end ? begin + size : end)}, at % cols, 0};
}

// most parts that any offsets of `count` groups over `rows` rows can have
static int64_t most_parts(int64_t rows, int64_t count, int64_t size) {
  return (rows + std::min(rows, count) * (size - 1)) / size;
}

// zeros in the rows outside all groups, by worker `index` of those without a part
template <class T>
__device__ void clear_ungrouped(const Groups &g, T *y, int64_t n, int64_t index, int64_t workers, int threads) {
  const int64_t lo = bound(g, 0), hi = bound(g, g.count) > lo ? bound(g, g.count) : lo;
  const int64_t chunks = (n + kVec<T> - 1) / kVec<T>, open = lo + g.rows - hi;
  for (int64_t i = index * threads + threadIdx.x; i < open * chunks; i += workers * threads) {
    const int64_t k = i / chunks, r = k < lo ? k : hi + k - lo, at = (i - k * chunks) * kVec<T>;
    store_chunk(y + r * n + at, n - at, Chunk<T>{});
  }
}

// ---------------------------------------------------------------------------
// tiles
// ---------------------------------------------------------------------------
constexpr int kStep = 128;  // bytes of the summed index per step
template <class T> constexpr int kStepK = kStep / static_cast<int>(sizeof(T));

// Four 16-bit values of 16 lanes, transposed: lane i of the 16 gets value i % 4
// of lanes i / 4 + {0, 4, 8, 12}.
__device__ __forceinline__ short4v read_tr(const char *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(const_cast<char *>(p)));
}

// KC: row r's 16-byte chunk c at r * 128 + (c ^ (r / 2 % 8)) * 16, so that the
// 16 lanes that read one chunk of 16 rows meet all banks once.
__device__ __forceinline__ int kc_at(int r, int c) { return r * kStep + ((c ^ ((r >> 1) & 7)) << 4); }

// KO: row k of N values.  16 bits: a transposing read takes, at the same 32
// bytes of a row, rows k..k+3 and k+8..k+11 (and so on) at once: those pairs of
// chunks are spread over the banks.  32 bits: rows k, k+4, k+8, k+12.
template <class T, int N> __device__ __forceinline__ int ko_at(int k, int c) {
  constexpr int ROW = N * static_cast<int>(sizeof(T));
  if constexpr (sizeof(T) == 4) {
    c ^= ((k >> 2) & 3) << 2;
  } else if constexpr (ROW >= 256) {
    c ^= ((k & 3) | ((k >> 1) & 4)) << 1;
  } else {
    c ^= (((k >> 1) & 1) | ((k >> 2) & 2)) << 1;
  }
  return k * ROW + (c << 4);
}

// fragment kk (of 2) of 16 rows from r0: lane l holds row l % 16, chunk l / 16
__device__ __forceinline__ uintx4_t kc_frag(const char *tile, int r0, int kk) {
  const int lane = lane_id();
  return *reinterpret_cast<const uintx4_t *>(tile + kc_at(r0 + (lane & 15), kk * 4 + (lane >> 4)));
}
template <class T, int N> __device__ __forceinline__ uintx4_t ko_frag(const char *tile, int n0, int kk) {
  const int lane = lane_id(), i = lane & 15, q = lane >> 4;
  if constexpr (sizeof(T) == 2) {
    const int k = kk * 32 + q * 8 + (i >> 2), c = n0 / 8 + ((i & 3) >> 1), half = (i & 1) * 8;
    const auto lo = read_tr(tile + ko_at<T, N>(k, c) + half), hi = read_tr(tile + ko_at<T, N>(k + 4, c) + half);
    const uintx2_t a = __builtin_bit_cast(uintx2_t, lo), b = __builtin_bit_cast(uintx2_t, hi);
    return {a[0], a[1], b[0], b[1]};
  } else {
    uintx4_t r;
    const int c = n0 / 4 + (i >> 2);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      r[j] = *reinterpret_cast<const uint32_t *>(tile + ko_at<T, N>(kk * 16 + q * 4 + j, c) + (i & 3) * 4);
    return r;
  }
}

template <class T> __device__ __forceinline__ void mma(floatx4_t &d, uintx4_t a, uintx4_t b) {
  if constexpr (std::is_same_v<T, _Float16>) {
    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), d, 0, 0, 0);
  } else if constexpr (std::is_same_v<T, __bf16>) {
    d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), d, 0, 0, 0);
  } else {
    // (element i of every lane's four: the summed index in another order, the
    // same for both operands)
    const floatx4_t x = __builtin_bit_cast(floatx4_t, a), y = __builtin_bit_cast(floatx4_t, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], d, 0, 0, 0);
  }
}

// A thread's chunks of a tile on their way through registers.
template <int N> struct Staged {
  uintx4_t v[N];
};

// Tiles through registers, for what DMA cannot feed: rows or views off 16-byte
// boundaries, odd widths, and tensors of 2 GiB and more under one descriptor.
// 128 x 128 outputs by four waves, 64 x 64 each.
constexpr int kRows = 128, kCols = 128, kThreads = 256;

template <class T> struct Product {
  static constexpr int KC_CHUNKS = kRows * 8 / kThreads;                               // chunks a thread and tile
  static constexpr int CPR = kCols * static_cast<int>(sizeof(T)) / 16;                 // chunks a KO row
  static constexpr int KO_CHUNKS = kStepK<T> * CPR / kThreads;
  static constexpr int TILE = kRows * kStep;                                           // bytes of either form
  static_assert(KC_CHUNKS == 4 && KO_CHUNKS == 4 && TILE == kStepK<T> * kCols * int(sizeof(T)), "tile shape");
};

// KC tile of rows row(i) (null: none) from column k0 of `width`
template <class T, class RowPtr>
__device__ __forceinline__ Staged<4> stage_kc(RowPtr &&row, int64_t k0, int64_t width) {
  Staged<4> s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int id = threadIdx.x + i * kThreads;
    const T *p = row(i);
    const int64_t k = k0 + (id & 7) * kVec<T>;
    s.v[i] = load_raw(p + k, p ? width - k : 0);
  }
  return s;
}
__device__ __forceinline__ void place_kc(char *tile, const Staged<4> &s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int id = threadIdx.x + i * kThreads;
    *reinterpret_cast<uintx4_t *>(tile + kc_at(id >> 3, id & 7)) = s.v[i];
  }
}
// KO tile: rows row(k) (null: none) for k of the step, from column n0 of `width`
template <class T, class RowPtr>
__device__ __forceinline__ Staged<4> stage_ko(RowPtr &&row, int64_t n0, int64_t width) {
  Staged<4> s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int id = threadIdx.x + i * kThreads;
    const T *p = row(id / Product<T>::CPR);
    const int64_t n = n0 + (id % Product<T>::CPR) * kVec<T>;
    s.v[i] = load_raw(p + n, p ? width - n : 0);
  }
  return s;
}
template <class T> __device__ __forceinline__ void place_ko(char *tile, const Staged<4> &s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int id = threadIdx.x + i * kThreads;
    *reinterpret_cast<uintx4_t *>(tile + ko_at<T, kCols>(id / Product<T>::CPR, id % Product<T>::CPR)) = s.v[i];
  }
}

struct Sums {
  floatx4_t v[4][4];  // [row tile][channel tile]
};

// acc[m][n] += rows' fragments x channels' fragments of one step
template <class T, class MFrag, class NFrag> __device__ __forceinline__ void multiply(Sums &acc, MFrag &&mf, NFrag &&nf) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    uintx4_t m[4], n[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = mf(i, kk);
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = nf(i, kk);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) mma<T>(acc.v[i][j], n[j], m[i]);
  }
}

// four consecutive values of a row
template <class T> __device__ __forceinline__ void store4(T *p, int64_t n, floatx4_t v) {
  if constexpr (sizeof(T) == 2) {
    typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(2)));
    if (n >= 4) {
      const T r[4] = {from_float<T>(v[0]), from_float<T>(v[1]), from_float<T>(v[2]), from_float<T>(v[3])};
      u2 w;
      __builtin_memcpy(&w, r, 8);
      *reinterpret_cast<u2 *>(p) = w;
      return;
    }
  } else if (n >= 4) {
    *reinterpret_cast<uintx4_a4_t *>(p) = __builtin_bit_cast(uintx4_t, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) p[i] = from_float<T>(v[i]);
}

struct RowsArgs {
  Groups g;
  const int32_t *source;  // row of x behind each row (or null: itself)
  int64_t num_sources;
  const void *x, *w, *bias;
  int64_t k, n;  // summed width, output width
  int relu;
  void *y;
};

// Forward (KO weights [k, n]) and rows' gradient (KC weights [n, k]).  O: type of
// the outputs, the operands' own or, for shares that are yet to be added, fp32.
template <class T, bool KO, class O> __global__ __launch_bounds__(kThreads) void rows_kernel(const RowsArgs a) {
  using P = Product<T>;
  __shared__ __align__(1024) char lds[4 * P::TILE];  // two stages of both tiles
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const Part part = find_part(a.g, kRows, blockIdx.x);
  if (part.group < 0) {
    if (blockIdx.y == 0) {
      const int64_t used = blockIdx.x - part.begin;
      clear_ungrouped(a.g, static_cast<O *>(a.y), a.n, part.begin, gridDim.x - used, kThreads);
    }
    return;
  }
  const int64_t n0 = blockIdx.y * static_cast<int64_t>(kCols);
  const T *w = static_cast<const T *>(a.w) + part.group * a.k * a.n;
  const T *row[4], *wrow[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int id = threadIdx.x + i * kThreads;
    const int64_t r = part.begin + (id >> 3);
    int64_t s = r < part.end ? r : -1;
    if (s >= 0 && a.source) {
      s = a.source[r];
      if (s >= a.num_sources) s = -1;
    }
    row[i] = s >= 0 ? static_cast<const T *>(a.x) + s * a.k : nullptr;
    const int64_t n = n0 + (id >> 3);
    wrow[i] = n < a.n ? w + n * a.k : nullptr;
  }
  auto stage_w = [&](int64_t k0) {
    if constexpr (KO)
      return stage_ko<T>([&](int k) -> const T * { return k0 + k < a.k ? w + (k0 + k) * a.n : nullptr; }, n0, a.n);
    else
      return stage_kc<T>([&](int i) { return wrow[i]; }, k0, a.k);
  };
  auto place = [&](int s, const Staged<4> &x, const Staged<4> &ws) {
    place_kc(lds + 2 * s * P::TILE, x);
    if constexpr (KO) place_ko<T>(lds + (2 * s + 1) * P::TILE, ws);
    else place_kc(lds + (2 * s + 1) * P::TILE, ws);
  };
  const int m0 = (wave >> 1) * 64, c0 = (wave & 1) * 64;
  Sums acc{};
  Staged<4> xs = stage_kc<T>([&](int i) { return row[i]; }, 0, a.k), ws = stage_w(0);
  place(0, xs, ws);
  __syncthreads();
  int s = 0;
  for (int64_t k0 = 0; k0 < a.k; k0 += kStepK<T>, s ^= 1) {
    const bool more = k0 + kStepK<T> < a.k;
    if (more) {
      xs = stage_kc<T>([&](int i) { return row[i]; }, k0 + kStepK<T>, a.k);
      ws = stage_w(k0 + kStepK<T>);
    }
    const char *xt = lds + 2 * s * P::TILE, *wt = xt + P::TILE;
    multiply<T>(
        acc, [&](int i, int kk) { return kc_frag(xt, m0 + i * 16, kk); },
        [&](int i, int kk) {
          if constexpr (KO) return ko_frag<T, kCols>(wt, c0 + i * 16, kk);
          else return kc_frag(wt, c0 + i * 16, kk);
        });
    if (more) place(s ^ 1, xs, ws);
    __syncthreads();
  }
  const T *bias = static_cast<const T *>(a.bias);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t n = n0 + c0 + j * 16 + (lane >> 4) * 4;
    floatx4_t b = {0, 0, 0, 0};
    if (bias)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (n + v < a.n) b[v] = to_float(bias[part.group * a.n + n + v]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = part.begin + m0 + i * 16 + (lane & 15);
      if (r >= part.end || n >= a.n) continue;
      floatx4_t v = acc.v[i][j] + b;
      if (a.relu)
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = v[q] < 0.f ? 0.f : v[q];
      store4(static_cast<O *>(a.y) + r * a.n + n, a.n - n, v);
    }
  }
}

// ---------------------------------------------------------------------------
// Rows streamed past weights that stay in LDS.  Where a group's weights fit
// there, the operator is bound by its rows' bytes (200k rows 96 -> 384, gathered:
// 46 us where its bytes take 33; tiles of both operands 123): a block lays the weights out
// once, one 1 KB block per MFMA fragment in lane order, and its eight waves then
// walk the rows of its part on their own, without barriers, each holding a
// tile's rows in registers and fetching the next tile's meanwhile.
//
// The 64 channels of four fragments are dealt out so that a lane's sums are 16
// consecutive channels of its row: whole 128-byte lines are written straight
// from registers.
// ---------------------------------------------------------------------------
constexpr int kStreamWaves = 8, kStreamThreads = 64 * kStreamWaves;
constexpr int kMostStreamFragments = 144;  // 1 KB each; at most 9 KB of bias beside them

// the channel (of 64) of operand row i of fragment j
__device__ __forceinline__ int dealt(int j, int i) { return (i >> 2) * 16 + j * 4 + (i & 3); }

struct StreamArgs {
  RowsArgs a;
  int part_rows;
};

// KF: fragments (64 bytes) of a row.  A wave takes 16 rows at a time (32 halve the
// reads of the weights from LDS and measure the same).
template <class T, bool KO, int KF, class O>
__global__ __launch_bounds__(kStreamThreads) __attribute__((amdgpu_waves_per_eu(KF <= 8 ? 4 : 2))) void stream_kernel(const StreamArgs sa) {
  constexpr int FK = 64 / static_cast<int>(sizeof(T));  // values of the summed index per fragment
  constexpr int MOST = kMostStreamFragments / kStreamWaves;
  extern __shared__ __align__(1024) char wlds[];
  const RowsArgs &a = sa.a;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, lq = lane >> 4;
  const Part part = find_part(a.g, sa.part_rows, blockIdx.x);
  if (part.group < 0) {
    clear_ungrouped(a.g, static_cast<O *>(a.y), a.n, part.begin, gridDim.x - (blockIdx.x - part.begin), kStreamThreads);
    return;
  }
  const T *w = static_cast<const T *>(a.w) + part.group * a.k * a.n;
  const int quads = static_cast<int>((a.n + 63) / 64);  // of fragments
  const int fragments = quads * 4 * KF;
  // the first tile's rows are on their way while the weights are laid out
  // (and the sources of the rows after them)
  uintx4_t next[KF];
  int32_t source = -1;
  auto look = [&](int64_t r0) {
    if (a.source) source = r0 + l16 < part.end ? a.source[r0 + l16] : -1;
  };
  auto fetch = [&](int64_t r0) {
    const int64_t r = r0 + l16;
    int64_t s = r < part.end ? r : -1;
    if (a.source) s = source < a.num_sources ? source : -1;
    const T *row = s >= 0 ? static_cast<const T *>(a.x) + s * a.k : nullptr;
    look(r0 + kStreamWaves * 16);
#pragma unroll
    for (int f = 0; f < KF; ++f) {
      const int64_t k = f * FK + lq * kVec<T>;
      next[f] = load_raw(row + k, row ? a.k - k : 0);
    }
  };
  look(part.begin + wave * 16);
  fetch(part.begin + wave * 16);
  // the bias too lies in LDS: a load from memory in the loop below would wait for
  // the rows under way before it
  float *bias = reinterpret_cast<float *>(wlds + fragments * 1024);
  for (int n = threadIdx.x; n < quads * 64; n += kStreamThreads)
    bias[n] = a.bias && n < a.n ? to_float(static_cast<const T *>(a.bias)[part.group * a.n + n]) : 0.f;
  if constexpr (KO) {
    // as they lie in memory, [KF FK, quads 64], zeros past their ends; then, all
    // in registers between two barriers, to fragments
    // (nine loads of a thread at a time under way)
    const int cpr = quads * 64 / kVec<T>, chunks = KF * FK * cpr;
    for (int first = threadIdx.x; first < chunks; first += 9 * kStreamThreads) {
      uintx4_t v[9];
#pragma unroll
      for (int q = 0; q < 9; ++q) {
        const int id = first + q * kStreamThreads, k = id / cpr, c = id - k * cpr;
        v[q] = load_raw(w + k * a.n + c * kVec<T>, k < a.k ? a.n - c * kVec<T> : 0);
      }
#pragma unroll
      for (int q = 0; q < 9; ++q) {
        const int id = first + q * kStreamThreads;
        if (id < chunks) *reinterpret_cast<uintx4_t *>(wlds + id * 16) = v[q];
      }
    }
    __syncthreads();
    uintx4_t v[MOST];
#pragma unroll
    for (int q = 0; q < MOST; ++q) {
      const int id = q * kStreamWaves + wave;
      if (id >= fragments) break;
      const int j = id / KF % 4, f = id % KF, col = id / (4 * KF) * 64;
      const int pitch = quads * 64 * static_cast<int>(sizeof(T));
      if constexpr (sizeof(T) == 2) {
        const char *at = wlds + (f * 32 + lq * 8 + (l16 >> 2)) * pitch + (col + dealt(j, (l16 & 3) * 4)) * 2;
        const auto lo = read_tr(at), hi = read_tr(at + 4 * pitch);
        const uintx2_t x = __builtin_bit_cast(uintx2_t, lo), y = __builtin_bit_cast(uintx2_t, hi);
        v[q] = uintx4_t{x[0], x[1], y[0], y[1]};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[q][i] = *reinterpret_cast<const uint32_t *>(wlds + (f * 16 + lq * 4 + i) * pitch + (col + dealt(j, l16)) * 4);
      }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < MOST; ++q) {
      const int id = q * kStreamWaves + wave;
      if (id < fragments) *reinterpret_cast<uintx4_t *>(wlds + id * 1024 + lane * 16) = v[q];
    }
  } else {
    for (int id = wave; id < fragments; id += kStreamWaves) {
      const int j = id / KF % 4, f = id % KF;
      const int64_t n = id / (4 * KF) * 64 + dealt(j, l16), k = f * FK + lq * kVec<T>;
      *reinterpret_cast<uintx4_t *>(wlds + id * 1024 + lane * 16) = load_raw(w + n * a.k + k, n < a.n ? a.k - k : 0);
    }
  }
  __syncthreads();
  for (int64_t r0 = part.begin + wave * 16; r0 < part.end; r0 += kStreamWaves * 16) {
    uintx4_t x[KF];
#pragma unroll
    for (int f = 0; f < KF; ++f) x[f] = next[f];
    fetch(r0 + kStreamWaves * 16);
    const int64_t r = r0 + l16;
    for (int q = 0; q < quads; ++q) {
      floatx4_t acc[4] = {};
      const char *wq = wlds + q * 4 * KF * 1024 + lane * 16;
#pragma unroll
      for (int f = 0; f < KF; ++f)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          mma<T>(acc[j], *reinterpret_cast<const uintx4_t *>(wq + (j * KF + f) * 1024), x[f]);
      const int64_t n = q * 64 + lq * 16;
      if (n >= a.n || r >= part.end) continue;
#pragma unroll
      for (int h = 0; h < 16 / kVec<O>; ++h) {
        Chunk<O> c;
#pragma unroll
        for (int v = 0; v < kVec<O>; ++v) {
          const float s = acc[(h * kVec<O> + v) / 4][v % 4] + bias[n + h * kVec<O> + v];
          c.v[v] = a.relu && s < 0.f ? 0.f : s;
        }
        store_chunk(static_cast<O *>(a.y) + r * a.n + n + h * kVec<O>, a.n - n - h * kVec<O>, c);
      }
    }
  }
}

// Whether the weights fit (their fragments), and the shape that holds a row.
template <class T> static bool streams(int64_t k, int64_t n) {
  const int64_t f = div_up(k * static_cast<int64_t>(sizeof(T)), 64);
  const int64_t kf = f <= 4 ? f : f <= 6 ? 6 : f <= 8 ? 8 : f <= 12 ? 12 : 16;
  return f <= 16 && kf * 4 * div_up(n, 64) <= kMostStreamFragments;
}

template <class T, bool KO, class O> static int launch_stream(const RowsArgs &a, hipStream_t stream) {
  const auto go = [&](auto KF) -> int {
    constexpr int kf = decltype(KF)::value;
    const size_t lds = div_up(a.n, 64) * (static_cast<size_t>(kf) * 4 * 1024 + 64 * sizeof(float));
    // Parts for all blocks that the CUs hold at once (two each, or one where the
    // weights take more than half the LDS), in one round: 200k rows 96 -> 384 in
    // parts of 512 rows 44.7 us, of 256 51.5, of 128 57.8; 40k rows 128 19.4, 512 28.5.
    const int64_t held = lds > 80 * 1024 ? 256 : 512, wave_rows = kStreamWaves * 16;
    const int rows = static_cast<int>(round_up(std::max<int64_t>(div_up(a.g.rows, held), 1), wave_rows));
    const auto kernel = stream_kernel<T, KO, kf, O>;
    SPIRA_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    hipLaunchKernelGGL(kernel, dim3(most_parts(a.g.rows, a.g.count, rows) + 1), dim3(kStreamThreads), lds, stream,
                       StreamArgs{a, rows});
    SPIRA_HIP_LAUNCH_CHECK();
    return kOk;
  };
  using std::integral_constant;
  switch (div_up(a.k * static_cast<int64_t>(sizeof(T)), 64)) {
    case 1: return go(integral_constant<int, 1>{});
    case 2: return go(integral_constant<int, 2>{});
    case 3: return go(integral_constant<int, 3>{});
    case 4: return go(integral_constant<int, 4>{});
    case 5: case 6: return go(integral_constant<int, 6>{});
    case 7: case 8: return go(integral_constant<int, 8>{});
    case 9: case 10: case 11: case 12: return go(integral_constant<int, 12>{});
    default: return go(integral_constant<int, 16>{});
  }
}

// ---------------------------------------------------------------------------
// Tiles fed by DMA: rows and widths of whole 16-byte chunks.  The global loads
// write LDS themselves (no registers, no address arithmetic but one add a
// load), three steps ahead of the products, in a ring of four stages of 64 bytes
// of the summed index.  (Two stages of 128 bytes leave a load the time of one
// step to arrive, and the matrix cores busy for 28 % of it.)  The LDS swizzle is
// made by the order in which the lanes fetch a row's chunks.  Chunks past a
// row's end and rows that are not there are out of the buffer's range: they load
// zeros, and so do the steps past the last, so that the loads in flight are
// always as many.
//
// ---------------------------------------------------------------------------
constexpr uint32_t kOutOfRange = 0x80000000u;
constexpr int64_t kBufferLimit = int64_t(1) << 31;

// A buffer descriptor: base, bytes, raw.
__device__ __forceinline__ uintx4_t buffer(const void *base, int64_t bytes) {
  const int64_t n = bytes < 0 ? 0 : bytes < kBufferLimit ? bytes : kBufferLimit - 1;
  const auto at = reinterpret_cast<uint64_t>(base);
  return {uniform(static_cast<uint32_t>(at)), uniform(static_cast<uint32_t>(at >> 32) & 0xFFFFu),
          uniform(static_cast<uint32_t>(n)), 0x00020000u};
}
// 1 KB to LDS, 16 bytes from each lane's offset.  In assembly, and waited for by
// the ring alone: the compiler's own count of such loads is not kept over the
// ring's loop, it would wait for all of them once a turn.  (No register is
// written.  What loads the compiler itself waits for, it waits longer.)
__device__ __forceinline__ void load_lds(uintx4_t from, uint32_t offset, char *to) {
  const uint32_t at = uniform(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void *)to)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(at), "v"(offset), "s"(from) : "memory", "m0");
}
// 256 bytes, 4 from each lane's offset
__device__ __forceinline__ void load_lds_word(uintx4_t from, uint32_t offset, void *to) {
  const uint32_t at = uniform(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void *)to)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :: "s"(at), "v"(offset), "s"(from) : "memory", "m0");
}
// Until all but the last N loads have landed and this wave's LDS reads are done,
// then the block's barrier.
template <int N> __device__ __forceinline__ void wait_loads_and_meet() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }  // vmcnt(0)

constexpr int kRing = 64;  // bytes of the summed index per stage
template <class T> constexpr int kRingK = kRing / static_cast<int>(sizeof(T));

template <class T, int M, int N, int WM, int WN> struct Tile {
  static constexpr int NW = (M / WM) * (N / WN), NT = 64 * NW;
  static constexpr int MI = WM / 16, NI = WN / 16;
  static constexpr int XL = M / 16 / NW, WL = N / 16 / NW;  // loads (1 KB) a wave and stage
  static constexpr int XBYTES = M * kRing, WBYTES = N * kRing;
  static_assert(XL >= 1 && WL >= 1 && XL * NW * 16 == M && WL * NW * 16 == N, "tile shape");
};

// KC stage: row r's chunk c (of 4) at r * 64 + (c ^ turn(r)) * 16.  A 16-byte LDS
// read serves lanes 0-3, 12-15, 20-27 at once (then 4-11, 16-19, 28-31, and so in
// the upper half): rows 0-3 and 12-15 of one chunk with rows 4-11 of the next.
// turn() is 0, 2, 3, 1 for the four rows-of-four, which keeps those apart.
__device__ __forceinline__ int turn(int r) { return ((r >> 1) & 2) ^ (((r >> 3) & 1) * 3); }
__device__ __forceinline__ int ring_at(int r, int c) { return r * kRing + ((c ^ turn(r)) << 4); }
__device__ __forceinline__ uintx4_t ring_frag(const char *tile, int r0) {
  const int lane = lane_id();
  return *reinterpret_cast<const uintx4_t *>(tile + ring_at(r0 + (lane & 15), lane >> 4));
}

// where lane `lane` of a stage's load `i` (1 KB) reads: KC row and chunk; KO row k and chunk
__device__ __forceinline__ void kc_source(int i, int lane, int &r, int &c) {
  r = i * 16 + (lane >> 2);
  c = (lane & 3) ^ turn(r);
}
template <class T, int N> __device__ __forceinline__ void ko_source(int i, int lane, int &k, int &c) {
  constexpr int CPR = N * static_cast<int>(sizeof(T)) / 16;
  const int id = i * 64 + lane;
  k = id / CPR;
  c = (ko_at<T, N>(k, id % CPR) - k * CPR * 16) >> 4;
}

template <class T, int MI, int NI> struct TileSums {
  floatx4_t v[MI][NI];
};

// What a wave reads of a stage a step ahead: the channels' fragments, and the
// first rows'.
constexpr int kAhead = 2;
template <int NI> struct Head {
  uintx4_t n[NI], m[kAhead];
};

// acc += a stage's products.  The first rows' begin at once behind the barrier, on
// the head read during the step before (without it the matrix cores wait for
// 80 KB of LDS reads of eight waves); the others' fragments arrive meanwhile, and
// then the next step's head.  m(i): rows' fragment i of this stage; ahead(f): the
// next stage's head.
template <class T, int MI, int NI, class M, class Ahead>
__device__ __forceinline__ void multiply_tile(TileSums<T, MI, NI> &acc, const Head<NI> &f, Head<NI> &next, bool busy,
                                              M &&m, Ahead &&ahead) {
  if (!busy) {
    ahead(next);
    return;
  }
  constexpr int REST = MI - kAhead, FIRST = REST / 2;
  static_assert(REST >= 2, "rows of a wave");
  uintx4_t r[REST];
  const auto products = [&](int i, uintx4_t x) {
#pragma unroll
    for (int j = 0; j < NI; ++j) mma<T>(acc.v[i][j], f.n[j], x);
  };
#pragma unroll
  for (int i = 0; i < FIRST; ++i) r[i] = m(kAhead + i);
#pragma unroll
  for (int i = 0; i < kAhead; ++i) products(i, f.m[i]);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = FIRST; i < REST; ++i) r[i] = m(kAhead + i);
#pragma unroll
  for (int i = 0; i < FIRST; ++i) products(kAhead + i, r[i]);
  __builtin_amdgcn_sched_barrier(0);
  ahead(next);
#pragma unroll
  for (int i = FIRST; i < REST; ++i) products(kAhead + i, r[i]);
}

// issue(step, stage), head(stage, f) and multiply(stage, next stage, f, next f)
// over `steps` steps; L: loads a wave and step.
template <int L, class F, class Issue, class ReadHead, class Multiply>
__device__ __forceinline__ void ring_loop(int steps, Issue &&issue, ReadHead &&head, Multiply &&multiply) {
  using std::integral_constant;
  constexpr integral_constant<int, 0> s0;
  constexpr integral_constant<int, 1> s1;
  constexpr integral_constant<int, 2> s2;
  constexpr integral_constant<int, 3> s3;
  if (steps <= 0) return;
  issue(0, s0);
  issue(1, s1);
  issue(2, s2);
  F a, b;
  wait_loads_and_meet<2 * L>();
  head(s0, a);
  for (int step = 0;;) {
    wait_loads_and_meet<L>();
    issue(step + 3, s3);
    multiply(s0, s1, a, b);
    if (++step == steps) break;
    wait_loads_and_meet<L>();
    issue(step + 3, s0);
    multiply(s1, s2, b, a);
    if (++step == steps) break;
    wait_loads_and_meet<L>();
    issue(step + 3, s1);
    multiply(s2, s3, a, b);
    if (++step == steps) break;
    wait_loads_and_meet<L>();
    issue(step + 3, s2);
    multiply(s3, s0, b, a);
    if (++step == steps) break;
  }
  wait_loads();  // (none may land in the LDS of a block that follows)
}
// stage s of four arrays
template <int S> __device__ __forceinline__ char *stage_of(char *a, char *b, char *c, char *d) {
  if constexpr (S == 0) return a;
  else if constexpr (S == 1) return b;
  else if constexpr (S == 2) return c;
  else return d;
}

// A lane's sums are four channels of each of four 16-channel tiles: quarter q of
// the wave holds channels 4 q of every tile.  Exchanged between the quarters (a 4
// x 4 transpose in two rounds of swaps), quarter q holds all 16 of tile q, and the
// wave writes 16 rows of whole 128-byte lines.  Every lane takes part; `there`:
// its row is to be written.  n: first of the 64 channels, of `width`.
template <class T> __device__ __forceinline__ void store_row(T *row, int64_t n, int64_t width, bool there,
                                                             const floatx4_t (&v)[4]) {
  constexpr int W = static_cast<int>(sizeof(T));  // words of four values
  uint32_t u[4][W];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    T t[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) t[q] = from_float<T>(v[j][q]);
    __builtin_memcpy(u[j], t, sizeof(t));
  }
#pragma unroll
  for (int w = 0; w < W; ++w) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const auto s = __builtin_amdgcn_permlane32_swap(u[j][w], u[j + 2][w], false, false);
      u[j][w] = s[0];
      u[j + 2][w] = s[1];
    }
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const auto s = __builtin_amdgcn_permlane16_swap(u[j][w], u[j + 1][w], false, false);
      u[j][w] = s[0];
      u[j + 1][w] = s[1];
    }
  }
  const int64_t at = n + (lane_id() >> 4) * 16;
  if (!there) return;
  const uint32_t *f = &u[0][0];
#pragma unroll
  for (int c = 0; c < W; ++c)
    // (widths are whole chunks)
    if (at + c * kVec<T> < width)
      *reinterpret_cast<Unaligned<T> *>(row + at + c * kVec<T>) = uintx4_t{f[4 * c], f[4 * c + 1], f[4 * c + 2], f[4 * c + 3]};
}

// The bias of a lane's channels, read before the products begin.
template <class T, int NI> struct BiasOf {
  T v[NI][4];
  __device__ __forceinline__ void load(const T *bias, int64_t n, int64_t width, int lane) {
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int64_t at = n + j * 16 + (lane >> 4) * 4;
#pragma unroll
      for (int q = 0; q < 4; ++q) v[j][q] = bias && at < width ? bias[at + q] : static_cast<T>(0.f);
    }
  }
  __device__ __forceinline__ floatx4_t at(int j) const {
    return {to_float(v[j][0]), to_float(v[j][1]), to_float(v[j][2]), to_float(v[j][3])};
  }
};

template <class T, bool KO, class O, int M, int N, int WM, int WN>
__global__ __launch_bounds__((Tile<T, M, N, WM, WN>::NT)) void tile_kernel(const RowsArgs a) {
  using S = Tile<T, M, N, WM, WN>;
  __shared__ __align__(1024) char x0[S::XBYTES], x1[S::XBYTES], x2[S::XBYTES], x3[S::XBYTES];
  __shared__ __align__(1024) char w0[S::WBYTES], w1[S::WBYTES], w2[S::WBYTES], w3[S::WBYTES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const Place place = find_place(a.g, M, blockIdx.x, static_cast<uint32_t>((a.n + N - 1) / N), gridDim.x);
  const Part part = place.part;
  if (part.group < 0) {
    clear_ungrouped(a.g, static_cast<O *>(a.y), a.n, part.begin, place.idle, S::NT);
    return;
  }
  const int64_t n0 = place.col * static_cast<int64_t>(N);
  const uint32_t kbytes = static_cast<uint32_t>(a.k * static_cast<int64_t>(sizeof(T)));
  const uint32_t nbytes = static_cast<uint32_t>(a.n * static_cast<int64_t>(sizeof(T)));
  const uintx4_t xr =
      a.source ? buffer(a.x, a.num_sources * kbytes)
               : buffer(static_cast<const char *>(a.x) + part.begin * kbytes, (part.end - part.begin) * kbytes);
  const uintx4_t wr =
      buffer(static_cast<const char *>(a.w) + part.group * a.k * nbytes, a.k * static_cast<int64_t>(nbytes));
  uint32_t xo[S::XL], xc[S::XL], wo[S::WL], wc[S::WL];
#pragma unroll
  for (int i = 0; i < S::XL; ++i) {
    int r, c;
    kc_source(wave * S::XL + i, lane, r, c);
    xc[i] = c * 16;
    xo[i] = kOutOfRange;
    if (part.begin + r < part.end) {
      const int64_t s = a.source ? a.source[part.begin + r] : r;
      if (s >= 0 && (!a.source || s < a.num_sources)) xo[i] = static_cast<uint32_t>(s) * kbytes + xc[i];
    }
  }
#pragma unroll
  for (int i = 0; i < S::WL; ++i) {
    int r, c;
    if constexpr (KO) {
      ko_source<T, N>(wave * S::WL + i, lane, r, c);
      wc[i] = 0;
      wo[i] = r * nbytes + static_cast<uint32_t>(n0 * sizeof(T)) + c * 16;
    } else {
      kc_source(wave * S::WL + i, lane, r, c);
      wc[i] = c * 16;
      wo[i] = n0 + r < a.n ? static_cast<uint32_t>(n0 + r) * kbytes + wc[i] : kOutOfRange;
    }
  }
  const int steps = static_cast<int>((kbytes + kRing - 1) / kRing);
  auto issue = [&](int step, auto stage) {
    constexpr int st = decltype(stage)::value;
    char *xs = stage_of<st>(x0, x1, x2, x3), *ws = stage_of<st>(w0, w1, w2, w3);
    const uint32_t kb = step * kRing;
#pragma unroll
    for (int i = 0; i < S::XL; ++i)
      load_lds(xr, kb + xc[i] < kbytes ? xo[i] + kb : kOutOfRange, xs + (wave * S::XL + i) * 1024);
    // (KO weights past the group's last row: out of range)
    const uint32_t wb = KO ? step * static_cast<uint32_t>(kRingK<T>) * nbytes : kb;
#pragma unroll
    for (int i = 0; i < S::WL; ++i)
      load_lds(wr, KO || kb + wc[i] < kbytes ? wo[i] + wb : kOutOfRange, ws + (wave * S::WL + i) * 1024);
  };
  const int m0 = wave / (N / WN) * WM, c0 = wave % (N / WN) * WN;
  const bool busy = part.begin + m0 < part.end;  // (a last part's rows may end before this wave's)
  TileSums<T, S::MI, S::NI> acc{};
  BiasOf<T, S::NI> bias;
  bias.load(a.bias ? static_cast<const T *>(a.bias) + part.group * a.n : nullptr, n0 + c0, a.n, lane);
  using F = Head<S::NI>;
  const auto rows_frag = [&](auto stage, int i) {
    return ring_frag(stage_of<decltype(stage)::value>(x0, x1, x2, x3), m0 + i * 16);
  };
  const auto head = [&](auto stage, F &f) {
    const char *ws = stage_of<decltype(stage)::value>(w0, w1, w2, w3);
#pragma unroll
    for (int i = 0; i < S::NI; ++i) {
      if constexpr (KO) f.n[i] = ko_frag<T, N>(ws, c0 + i * 16, 0);
      else f.n[i] = ring_frag(ws, c0 + i * 16);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f.m[i] = rows_frag(stage, i);
  };
  ring_loop<S::XL + S::WL, F>(steps, issue, head, [&](auto stage, auto after, const F &f, F &next) {
    multiply_tile<T>(
        acc, f, next, busy, [&](int i) { return rows_frag(stage, i); }, [&](F &n) { head(after, n); });
  });
#pragma unroll
  for (int i = 0; i < S::MI; ++i) {
    const int64_t r = part.begin + m0 + i * 16 + (lane & 15);
    floatx4_t v[S::NI];
#pragma unroll
    for (int j = 0; j < S::NI; ++j) {
      v[j] = acc.v[i][j] + bias.at(j);
      if (a.relu)
#pragma unroll
        for (int q = 0; q < 4; ++q) v[j][q] = v[j][q] < 0.f ? 0.f : v[j][q];
    }
    store_row<O>(static_cast<O *>(a.y) + r * a.n, n0 + c0, a.n, r < part.end, v);
  }
}

// Few rows to a group (a serving step's): the weights' bytes are all there is, and
// what counts is how many of them are under way.  A block takes 16 rows and 64
// columns, each of its four waves every fourth step with a ring of its own, without
// barriers; their sums are added in order at the end.
constexpr int kFewDepth = 4, kFewWaves = 4;
template <class T, bool KO, class O> __global__ __launch_bounds__(64 * kFewWaves) void few_kernel(const RowsArgs a) {
  using S = Tile<T, 16, 64, 16, 64>;
  constexpr int STAGE = S::XBYTES + S::WBYTES, L = S::XL + S::WL;
  static_assert(S::NW == 1 && (kFewDepth - 1) * L < 64, "a wave's own loads, counted");
  __shared__ __align__(1024) char rings[kFewWaves][kFewDepth * STAGE];
  static_assert(sizeof(rings) >= kFewWaves * 4096, "the sums of the waves");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char *ring = rings[wave];
  const Place place = find_place(a.g, 16, blockIdx.x, static_cast<uint32_t>((a.n + 63) / 64), gridDim.x);
  const Part part = place.part;
  if (part.group < 0) {
    clear_ungrouped(a.g, static_cast<O *>(a.y), a.n, part.begin, place.idle, 64 * kFewWaves);
    return;
  }
  const int64_t n0 = place.col * static_cast<int64_t>(64);
  const uint32_t kbytes = static_cast<uint32_t>(a.k * static_cast<int64_t>(sizeof(T)));
  const uint32_t nbytes = static_cast<uint32_t>(a.n * static_cast<int64_t>(sizeof(T)));
  const uintx4_t xr =
      a.source ? buffer(a.x, a.num_sources * kbytes)
               : buffer(static_cast<const char *>(a.x) + part.begin * kbytes, (part.end - part.begin) * kbytes);
  const uintx4_t wr =
      buffer(static_cast<const char *>(a.w) + part.group * a.k * nbytes, a.k * static_cast<int64_t>(nbytes));
  uint32_t xo[S::XL], xc[S::XL], wo[S::WL], wc[S::WL];
#pragma unroll
  for (int i = 0; i < S::XL; ++i) {
    int r, c;
    kc_source(i, lane, r, c);
    xc[i] = c * 16;
    xo[i] = kOutOfRange;
    if (part.begin + r < part.end) {
      const int64_t s = a.source ? a.source[part.begin + r] : r;
      if (s >= 0 && (!a.source || s < a.num_sources)) xo[i] = static_cast<uint32_t>(s) * kbytes + xc[i];
    }
  }
#pragma unroll
  for (int i = 0; i < S::WL; ++i) {
    int r, c;
    if constexpr (KO) {
      ko_source<T, 64>(i, lane, r, c);
      wc[i] = 0;
      wo[i] = r * nbytes + static_cast<uint32_t>(n0 * sizeof(T)) + c * 16;
    } else {
      kc_source(i, lane, r, c);
      wc[i] = c * 16;
      wo[i] = n0 + r < a.n ? static_cast<uint32_t>(n0 + r) * kbytes + wc[i] : kOutOfRange;
    }
  }
  BiasOf<T, 4> bias;
  bias.load(a.bias ? static_cast<const T *>(a.bias) + part.group * a.n : nullptr, n0, a.n, lane);
  const int steps = static_cast<int>((kbytes + kRing - 1) / kRing);
  auto issue = [&](int turn) {
    const int step = turn * kFewWaves + wave;
    char *xs = ring + turn % kFewDepth * STAGE, *ws = xs + S::XBYTES;
    const uint32_t kb = step * kRing;
#pragma unroll
    for (int i = 0; i < S::XL; ++i) load_lds(xr, kb + xc[i] < kbytes ? xo[i] + kb : kOutOfRange, xs + i * 1024);
    const uint32_t wb = KO ? step * static_cast<uint32_t>(kRingK<T>) * nbytes : kb;
#pragma unroll
    for (int i = 0; i < S::WL; ++i)
      load_lds(wr, kb + wc[i] < kbytes ? wo[i] + wb : kOutOfRange, ws + i * 1024);
  };
  for (int turn = 0; turn < kFewDepth; ++turn) issue(turn);
  floatx4_t acc[4] = {};
  for (int turn = 0; turn * kFewWaves + wave < steps; ++turn) {
    __builtin_amdgcn_s_waitcnt((((kFewDepth - 1) * L) & 15) | (7 << 4) | (15 << 8) | ((((kFewDepth - 1) * L) >> 4) << 14));
    asm volatile("" ::: "memory");
    const char *xs = ring + turn % kFewDepth * STAGE, *ws = xs + S::XBYTES;
    uintx4_t n[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (KO) n[j] = ko_frag<T, 64>(ws, j * 16, 0);
      else n[j] = ring_frag(ws, j * 16);
    }
    const uintx4_t m = ring_frag(xs, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) mma<T>(acc[j], n[j], m);
    // (the stage is read before it is loaded again)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    issue(turn + kFewDepth);
  }
  wait_loads();  // (none may land in what follows)
  asm volatile("" ::: "memory");
  __syncthreads();
  auto *sums = reinterpret_cast<floatx4_t *>(&rings[0][0]);
#pragma unroll
  for (int j = 0; j < 4; ++j) sums[(wave * 4 + j) * 64 + lane] = acc[j];
  __syncthreads();
  if (wave != 0) return;
  floatx4_t v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = bias.at(j);
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) v[j] += sums[(w * 4 + j) * 64 + lane];
    if (a.relu)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[j][q] = v[j][q] < 0.f ? 0.f : v[j][q];
  }
  const int64_t r = part.begin + (lane & 15);
  store_row<O>(static_cast<O *>(a.y) + r * a.n, n0, a.n, r < part.end, v);
}

static bool aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether DMA can feed the tiles.
template <class T> static bool dma_fits(const RowsArgs &a) {
  const int64_t size = sizeof(T);
  return a.k % kVec<T> == 0 && a.n % kVec<T> == 0 && aligned(a.x) && aligned(a.w) && a.k * a.n * size < kBufferLimit &&
         a.k * size <= (1 << 22) && (!a.source || a.num_sources * a.k * size < kBufferLimit);
}

template <class T, bool KO, class O, int M, int N, int WM, int WN> static int launch_tile(const RowsArgs &a, hipStream_t stream) {
  const int64_t blocks = (most_parts(a.g.rows, a.g.count, M)) * div_up(a.n, N) + 1;
  SPIRA_HIP_REQUIRE(launchable(blocks, Tile<T, M, N, WM, WN>::NT), "grouped_linear: too many tiles");
  hipLaunchKernelGGL((tile_kernel<T, KO, O, M, N, WM, WN>), dim3(blocks), dim3(Tile<T, M, N, WM, WN>::NT), 0, stream, a);
  SPIRA_HIP_LAUNCH_CHECK();
  return kOk;
}

template <class T, bool KO, class O> static int launch_few(const RowsArgs &a, hipStream_t stream) {
  const int64_t blocks = most_parts(a.g.rows, a.g.count, 16) * div_up(a.n, 64) + 1;
  SPIRA_HIP_REQUIRE(launchable(blocks, 64 * kFewWaves), "grouped_linear: too many tiles");
  hipLaunchKernelGGL((few_kernel<T, KO, O>), dim3(blocks), dim3(64 * kFewWaves), 0, stream, a);
  SPIRA_HIP_LAUNCH_CHECK();
  return kOk;
}

template <class T, bool KO, class O = T> static int launch_rows(const RowsArgs &a, hipStream_t stream) {
  // Few rows to a group, on average: how the rows lie, only the device knows.  A
  // block of few_kernel reads its weights for 16 rows only, so the few form is
  // taken where most of its blocks, however uneven the groups, run at once (512 do):
  // then it costs its latency, which is the shortest.  us against the large forms
  // below, groups of even sizes / sizes falling by 0.8 each:
  //   bf16 16 a group, 32 groups, 2048 -> 512 (496 blocks) 14.6 / 18.2 and 22.3 / 23.7
  //   4 a group, 32 groups, 512 -> 2048 (1216) 15.6 / 13.2 and 13.9 / 11.3
  //   16 a group, 256 groups, 1024 -> 1024 (8k) 130 / 80 and 111 / 32
  //   streamed weights: 16 a group, 64 groups, 96 -> 384 (744) 5.5 / 6.3 and 10.1 / 10.6;
  //   64 a group 256 -> 256 (1264) 10.5 / 12.4 and 18.0 / 18.7, 96 -> 384 (1896) 13.5 / 15.5 and 10.5 / 10.9
  // Tiles of fp32 take the matrix cores four times the rows that are there: 16 a group,
  // 128 groups, 2048 -> 2048 390 / 352 and 1009 / 440, 32 a group 634 / 634 and 1009 /
  // 515, of any number of blocks.  (All rows in one group: 582 and 270.)
  const bool stream_fits = streams<T>(a.k, a.n);
  const int64_t few = stream_fits ? 64 : sizeof(T) == 4 ? 32 : 16;
  const int64_t most_blocks = stream_fits ? 1280 : sizeof(T) == 4 ? INT64_MAX : 1024;
  if (a.g.rows <= few * a.g.count && most_parts(a.g.rows, a.g.count, 16) * div_up(a.n, 64) <= most_blocks &&
      dma_fits<T>(a))
    return launch_few<T, KO, O>(a, stream);
  if (stream_fits) return launch_stream<T, KO, O>(a, stream);
  if (dma_fits<T>(a)) {
    // The large tile reads each operand half as often from L2 and LDS: 32k rows
    // 1024 -> 2048 in 16 even groups 141 us, with the small one 197.  It needs
    // groups that fill its rows, and blocks for every CU.
    if constexpr (sizeof(T) == 2)
      if (a.g.rows / a.g.count >= 256 && a.n > 128 && div_up(a.g.rows, 256) * div_up(a.n, 256) >= 256)
        return launch_tile<T, KO, O, 256, 256, 128, 64>(a, stream);
    return launch_tile<T, KO, O, 128, 128, 64, 64>(a, stream);
  }
  hipLaunchKernelGGL((rows_kernel<T, KO, O>), dim3(most_parts(a.g.rows, a.g.count, kRows) + 1, div_up(a.n, kCols)),
                     dim3(kThreads), 0, stream, a);
  SPIRA_HIP_LAUNCH_CHECK();
  return kOk;
}

struct WeightsArgs {
  Groups g;
  const int32_t *source;
  int64_t num_sources;
  const void *x, *dz;
  int64_t ci, co;
  int part_rows;   // rows per part; 0: whole groups
  float *partial;  // [parts, ci, co], or null: dw is written
  void *dw;
};

// dW[e] or a part's share of it: both operands KO, summed over rows.
template <class T> __global__ __launch_bounds__(kThreads) void weights_kernel(const WeightsArgs a) {
  using P = Product<T>;
  __shared__ __align__(1024) char lds[4 * P::TILE];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  Part part;
  if (a.partial) {
    part = find_part(a.g, a.part_rows, blockIdx.z);
    if (part.group < 0) return;
  } else {
    part = {static_cast<int>(blockIdx.z), bound(a.g, blockIdx.z), bound(a.g, blockIdx.z + 1)};
  }
  const int64_t n0 = blockIdx.x * static_cast<int64_t>(kCols), m0 = blockIdx.y * static_cast<int64_t>(kRows);
  auto stage_x = [&](int64_t r0) {
    return stage_ko<T>(
        [&](int k) -> const T * {
          int64_t s = r0 + k < part.end ? r0 + k : -1;
          if (s >= 0 && a.source) {
            s = a.source[s];
            if (s >= a.num_sources) s = -1;
          }
          return s >= 0 ? static_cast<const T *>(a.x) + s * a.ci : nullptr;
        },
        m0, a.ci);
  };
  auto stage_z = [&](int64_t r0) {
    return stage_ko<T>(
        [&](int k) -> const T * {
          return r0 + k < part.end ? static_cast<const T *>(a.dz) + (r0 + k) * a.co : nullptr;
        },
        n0, a.co);
  };
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  Sums acc{};
  Staged<4> xs = stage_x(part.begin), zs = stage_z(part.begin);
  place_ko<T>(lds, xs);
  place_ko<T>(lds + P::TILE, zs);
  __syncthreads();
  int s = 0;
  for (int64_t r0 = part.begin; r0 < part.end; r0 += kStepK<T>, s ^= 1) {
    const bool more = r0 + kStepK<T> < part.end;
    if (more) {
      xs = stage_x(r0 + kStepK<T>);
      zs = stage_z(r0 + kStepK<T>);
    }
    const char *xt = lds + 2 * s * P::TILE, *zt = xt + P::TILE;
    multiply<T>(
        acc, [&](int i, int kk) { return ko_frag<T, kRows>(xt, wm + i * 16, kk); },
        [&](int i, int kk) { return ko_frag<T, kCols>(zt, wn + i * 16, kk); });
    if (more) {
      place_ko<T>(lds + 2 * (s ^ 1) * P::TILE, xs);
      place_ko<T>(lds + (2 * (s ^ 1) + 1) * P::TILE, zs);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + wm + i * 16 + (lane & 15), n = n0 + wn + j * 16 + (lane >> 4) * 4;
      if (m >= a.ci || n >= a.co) continue;
      if (a.partial)
        store4(a.partial + (blockIdx.z * a.ci + m) * a.co + n, a.co - n, acc.v[i][j]);
      else
        store4(static_cast<T *>(a.dw) + (part.group * a.ci + m) * a.co + n, a.co - n, acc.v[i][j]);
    }
}

// The same fed by DMA, as tile_kernel.  The sources of gathered rows come the same
// way, three steps before the loads that need them, to a ring of each wave's own.
template <class T, bool GATHER, int M, int N, int WM, int WN>
__global__ __launch_bounds__((Tile<T, M, N, WM, WN>::NT)) __attribute__((amdgpu_waves_per_eu(2))) void weights_tile_kernel(const WeightsArgs a) {
  using S = Tile<T, M, N, WM, WN>;
  __shared__ __align__(1024) char x0[S::XBYTES], x1[S::XBYTES], x2[S::XBYTES], x3[S::XBYTES];
  __shared__ __align__(1024) char z0[S::WBYTES], z1[S::WBYTES], z2[S::WBYTES], z3[S::WBYTES];
  __shared__ int32_t sources[GATHER ? S::NW : 1][4][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t mt = (a.ci + M - 1) / M, nt = (a.co + N - 1) / N, tiles = mt * nt;
  const int64_t parts = a.partial ? count_parts(a.g, a.part_rows) : a.g.count;
  const int64_t place = blockIdx.x;
  if (place >= parts * tiles) return;
  const int64_t nth = place / tiles;
  Part part;
  if (a.partial) part = find_part(a.g, a.part_rows, nth);
  else part = {static_cast<int>(nth), uniform(bound(a.g, nth)), uniform(bound(a.g, nth + 1))};
  const int64_t m0 = place % tiles / nt * M, n0 = place % nt * N;
  const uint32_t xbytes = static_cast<uint32_t>(a.ci * static_cast<int64_t>(sizeof(T)));
  const uint32_t zbytes = static_cast<uint32_t>(a.co * static_cast<int64_t>(sizeof(T)));
  const uintx4_t gathered = buffer(a.x, a.num_sources * xbytes);
  int xk[S::XL], zk[S::WL];
  uint32_t xo[S::XL], zo[S::WL];
#pragma unroll
  for (int i = 0; i < S::XL; ++i) {
    int c;
    ko_source<T, M>(wave * S::XL + i, lane, xk[i], c);
    xo[i] = static_cast<uint32_t>(m0 * sizeof(T)) + c * 16;
    if (xo[i] >= xbytes) xo[i] = kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < S::WL; ++i) {
    int c;
    ko_source<T, N>(wave * S::WL + i, lane, zk[i], c);
    zo[i] = static_cast<uint32_t>(n0 * sizeof(T)) + c * 16;
    if (zo[i] >= zbytes) zo[i] = kOutOfRange;
  }
  const uintx4_t list = buffer(GATHER ? a.source + part.begin : nullptr, GATHER ? (part.end - part.begin) * 4 : 0);
  auto look = [&](int step, int slot) {
    load_lds_word(list, lane < kRingK<T> ? (step * kRingK<T> + lane) * 4u : kOutOfRange, sources[wave][slot]);
  };
  auto issue = [&](int step, auto stage) {
    constexpr int st = decltype(stage)::value;
    char *xs = stage_of<st>(x0, x1, x2, x3), *zs = stage_of<st>(z0, z1, z2, z3);
    const int64_t r0 = part.begin + static_cast<int64_t>(step) * kRingK<T>;
    if constexpr (GATHER) {
      int32_t src[S::XL];
#pragma unroll
      for (int i = 0; i < S::XL; ++i) src[i] = sources[wave][st][xk[i]];
#pragma unroll
      for (int i = 0; i < S::XL; ++i) {
        const bool in = r0 + xk[i] < part.end && src[i] >= 0 && src[i] < a.num_sources && xo[i] != kOutOfRange;
        load_lds(gathered, in ? static_cast<uint32_t>(src[i]) * xbytes + xo[i] : kOutOfRange,
                 xs + (wave * S::XL + i) * 1024);
      }
      look(step + 3, (st + 3) % 4);
    } else {
      const uintx4_t xr = buffer(static_cast<const char *>(a.x) + r0 * xbytes, (part.end - r0) * xbytes);
#pragma unroll
      for (int i = 0; i < S::XL; ++i) load_lds(xr, xo[i] + xk[i] * xbytes, xs + (wave * S::XL + i) * 1024);
    }
    const uintx4_t zr = buffer(static_cast<const char *>(a.dz) + r0 * zbytes, (part.end - r0) * zbytes);
#pragma unroll
    for (int i = 0; i < S::WL; ++i) load_lds(zr, zo[i] + zk[i] * zbytes, zs + (wave * S::WL + i) * 1024);
  };
  const int wm = wave / (N / WN) * WM, wn = wave % (N / WN) * WN;
  TileSums<T, S::MI, S::NI> acc{};
  const int steps = part.begin < part.end ? static_cast<int>((part.end - part.begin + kRingK<T> - 1) / kRingK<T>) : 0;
  if constexpr (GATHER) {
    look(0, 0);
    look(1, 1);
    look(2, 2);
    wait_loads();
    asm volatile("" ::: "memory");
  }
  using F = Head<S::NI>;
  const auto rows_frag = [&](auto stage, int i) {
    return ko_frag<T, M>(stage_of<decltype(stage)::value>(x0, x1, x2, x3), wm + i * 16, 0);
  };
  const auto head = [&](auto stage, F &f) {
#pragma unroll
    for (int i = 0; i < S::NI; ++i)
      f.n[i] = ko_frag<T, N>(stage_of<decltype(stage)::value>(z0, z1, z2, z3), wn + i * 16, 0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f.m[i] = rows_frag(stage, i);
  };
  ring_loop<S::XL + S::WL + (GATHER ? 1 : 0), F>(steps, issue, head,
                                                 [&](auto stage, auto after, const F &f, F &next) {
                                                   multiply_tile<T>(
                                                       acc, f, next, true, [&](int i) { return rows_frag(stage, i); },
                                                       [&](F &n) { head(after, n); });
                                                 });
#pragma unroll
  for (int i = 0; i < S::MI; ++i) {
    const int64_t m = m0 + wm + i * 16 + (lane & 15);
    if (a.partial) store_row<float>(a.partial + (nth * a.ci + m) * a.co, n0 + wn, a.co, m < a.ci, acc.v[i]);
    else store_row<T>(static_cast<T *>(a.dw) + (part.group * a.ci + m) * a.co, n0 + wn, a.co, m < a.ci, acc.v[i]);
  }
}

template <class T> static bool dma_fits(const WeightsArgs &a) {
  const int64_t size = sizeof(T);
  return a.ci % kVec<T> == 0 && a.co % kVec<T> == 0 && aligned(a.x) && aligned(a.dz) && a.ci * size <= (1 << 22) &&
         a.co * size <= (1 << 22) && (!a.source || a.num_sources * a.ci * size < kBufferLimit);
}

template <class T, int M, int N, int WM, int WN>
static int launch_weights_tile(const WeightsArgs &a, int64_t parts, hipStream_t stream) {
  const int64_t blocks = parts * div_up(a.co, N) * div_up(a.ci, M);
  const dim3 threads(Tile<T, M, N, WM, WN>::NT);
  SPIRA_HIP_REQUIRE(launchable(blocks, threads.x), "grouped_linear_weights_gradient: too many tiles");
  if (a.source)
    hipLaunchKernelGGL((weights_tile_kernel<T, true, M, N, WM, WN>), dim3(blocks), threads, 0, stream, a);
  else
    hipLaunchKernelGGL((weights_tile_kernel<T, false, M, N, WM, WN>), dim3(blocks), threads, 0, stream, a);
  SPIRA_HIP_LAUNCH_CHECK();
  return kOk;
}
// The large tile where there are blocks for every CU: 32k rows 1024 -> 2048 in 16
// groups 172 us, with the small one 185.
template <class T> static int launch_weights(const WeightsArgs &a, int64_t parts, hipStream_t stream) {
  if constexpr (sizeof(T) == 2)
    if (a.ci > 128 && a.co > 128 && parts * div_up(a.ci, 256) * div_up(a.co, 256) >= 256)
      return launch_weights_tile<T, 256, 256, 128, 64>(a, parts, stream);
  return launch_weights_tile<T, 128, 128, 64, 64>(a, parts, stream);
}

// out[e] = sum of the group's parts (`size` values each): 16 lanes of four values
// by 16 threads, each over every 16th part, joined in a fixed tree
template <class T>
__global__ __launch_bounds__(256) void join_kernel(const Groups g, int part_rows, int64_t parts, const float *partial,
                                                   int64_t size, T *out) {
  __shared__ floatx4_t sums[16][16];
  int64_t first, count;
  parts_of(g, part_rows, blockIdx.y, first, count);
  // (overlapping groups count more parts than there are)
  const int64_t last = std::min(first + count, parts);
  const int c = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int64_t i = (blockIdx.x * static_cast<int64_t>(16) + c) * 4;
  floatx4_t sum = {0, 0, 0, 0};
  for (int64_t p = first + q; p < last; p += 16) {
    const float *v = partial + p * size + i;
    if (size - i >= 4) {
      sum += __builtin_bit_cast(floatx4_t, *reinterpret_cast<const uintx4_a4_t *>(v));
    } else {
      for (int j = 0; j < size - i; ++j) sum[j] += v[j];
    }
  }
  sums[q][c] = sum;
  for (int half = 8; half > 0; half /= 2) {
    __syncthreads();
    if (q < half) sums[q][c] += sums[q + half][c];
  }
  if (q == 0 && i < size) store4(out + blockIdx.y * size + i, size - i, sums[0][c]);
}

// dz = dy where y > 0 (or dy), and the parts' column sums of it: 64 columns by
// 16 row lanes
template <class T>
__global__ __launch_bounds__(256) void activation_kernel(const Groups g, int part_rows, const T *dy, const T *y,
                                                         int64_t co, T *dz, float *partial) {
  constexpr int COLS = 16 * kVec<T>;
  __shared__ float sums[16][COLS + 1];
  const Part part = find_part(g, part_rows, blockIdx.y);
  if (part.group < 0) return;
  const int c = threadIdx.x & 15, rl = threadIdx.x >> 4;
  const int64_t at = blockIdx.x * static_cast<int64_t>(COLS) + c * kVec<T>;
  float s[kVec<T>] = {};
  if (at < co)
    for (int64_t r = part.begin + rl; r < part.end; r += 16) {
      Chunk<T> d = load_chunk(dy + r * co + at, co - at);
      if (y) {
        const Chunk<T> v = load_chunk(y + r * co + at, co - at);
#pragma unroll
        for (int j = 0; j < kVec<T>; ++j) d.v[j] = v.v[j] > 0.f ? d.v[j] : 0.f;
        store_chunk(dz + r * co + at, co - at, d);
      }
#pragma unroll
      for (int j = 0; j < kVec<T>; ++j) s[j] += d.v[j];
    }
  if (!partial) return;
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) sums[rl][c * kVec<T> + j] = s[j];
  __syncthreads();
  const int64_t n = blockIdx.x * static_cast<int64_t>(COLS) + threadIdx.x;
  if (threadIdx.x < COLS && n < co) {
    float v = 0;
#pragma unroll
    for (int q = 0; q < 16; ++q) v += sums[q][threadIdx.x];
    partial[blockIdx.y * co + n] = v;
  }
}

static int check_sizes(int64_t rows, int groups, int64_t ci, int64_t co) {
  // (2^23 short of 31 bits: rows_kernel has 256 threads to 128 rows, and a block more to each group)
  SPIRA_HIP_REQUIRE(rows >= 0 && rows <= (int64_t(1) << 31) - (1 << 23), "grouped_linear: bad number of rows");
  SPIRA_HIP_REQUIRE(groups > 0 && groups <= 32767, "grouped_linear: needs 1 to 32767 groups");
  SPIRA_HIP_REQUIRE(ci > 0 && co > 0 && ci <= (1 << 20) && co <= (1 << 20), "grouped_linear: bad widths");
  return kOk;
}
static int check(int64_t rows, int groups, const int32_t *offsets, int64_t ci, int64_t co) {
  if (int rc = check_sizes(rows, groups, ci, co)) return rc;
  SPIRA_HIP_REQUIRE(offsets, "grouped_linear: no offsets");
  return kOk;
}

// (grids have 65535 blocks in y and z: larger parts for more rows than that; the
// groups alone are at most half as many)
static int64_t launch_limit(int64_t rows, int64_t groups, int64_t size) {
  while (most_parts(rows, groups, size) > 65535 - 1) size *= 2;
  return size;
}

// Rows per part of the weights' gradient; 0: whole groups, no parts.  Parts are
// cut where the weights' tiles alone would leave the chip idle, at least 128 rows
// each: 20k fp32 rows 63 -> 130 in parts of 128 31 us, of 256 42.
static int weight_parts(int64_t rows, int64_t groups, int64_t ci, int64_t co) {
  const int64_t tiles = div_up(ci, kRows) * div_up(co, kCols) * groups;
  const int64_t want = 4 * 256;
  if (tiles >= want || rows == 0) return 0;
  const int64_t size = std::max<int64_t>(round_up(div_up(rows * div_up(ci, kRows) * div_up(co, kCols), want), 64), 128);
  return static_cast<int>(launch_limit(rows, groups, size));
}

// Rows per part of the column sums: blocks for every CU, at most 256 rows each.
template <class T> static int64_t sum_rows(int64_t rows, int64_t groups, int64_t co) {
  const int64_t size = round_up(div_up(rows * div_up(co, 16 * kVec<T>), 1024), 16);
  return launch_limit(rows, groups, std::min<int64_t>(std::max<int64_t>(size, 32), 256));
}

}  // namespace grouped

}  // namespace spira_hip

using namespace spira_hip;

extern "C" {

int spira_hip_grouped_linear(int64_t rows, int groups, const int32_t *offsets, const int32_t *sources,
                             int64_t num_sources, const void *x, int c_in, const void *weights, const void *bias,
                             int c_out, int dtype, int relu, void *y, hipStream_t stream) {
  if (int rc = grouped::check(rows, groups, offsets, c_in, c_out)) return rc;
  SPIRA_HIP_REQUIRE(weights && (rows == 0 || y) && (x || num_sources == 0) && num_sources >= 0 &&
                        (sources || num_sources >= rows),
                    "grouped_linear: null tensor or too few sources");
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (rows == 0) return kOk;
    grouped::RowsArgs a{{offsets, groups, rows}, sources, num_sources, x, weights, bias, c_in, c_out, relu, y};
    return grouped::launch_rows<T, true>(a, stream);
  });
}

int spira_hip_grouped_linear_rows_gradient(int64_t rows, int groups, const int32_t *offsets, const void *dz, int c_out,
                                           const void *weights, int c_in, int dtype, void *dx, hipStream_t stream) {
  if (int rc = grouped::check(rows, groups, offsets, c_in, c_out)) return rc;
  SPIRA_HIP_REQUIRE(weights && (rows == 0 || (dz && dx)), "grouped_linear_rows_gradient: null tensor");
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (rows == 0) return kOk;
    grouped::RowsArgs a{{offsets, groups, rows}, nullptr, rows, dz, weights, nullptr, c_out, c_in, 0, dx};
    return grouped::launch_rows<T, false>(a, stream);
  });
}

int spira_hip_grouped_linear_tokens_gradient_workspace(int64_t rows, int k, int c_in, size_t *bytes) {
  if (int rc = grouped::check_sizes(rows, 1, c_in, 1)) return rc;
  SPIRA_HIP_REQUIRE(k > 0, "grouped_linear_tokens_gradient: bad sizes");
  *bytes = static_cast<size_t>(rows) * c_in * sizeof(float);
  return kOk;
}

int spira_hip_grouped_linear_tokens_gradient(int64_t rows, int groups, const int32_t *offsets, const int32_t *slots,
                                             int64_t tokens, int k, const void *dz, int c_out, const void *weights,
                                             int c_in, int dtype, void *dx, void *workspace, size_t workspace_bytes,
                                             hipStream_t stream) {
  if (int rc = grouped::check(rows, groups, offsets, c_in, c_out)) return rc;
  SPIRA_HIP_REQUIRE(tokens >= 0 && k > 0, "grouped_linear_tokens_gradient: bad sizes");
  SPIRA_HIP_REQUIRE(weights && (rows == 0 || dz) && (tokens == 0 || (slots && dx)),
                    "grouped_linear_tokens_gradient: null tensor");
  size_t need = 0;
  if (int rc = spira_hip_grouped_linear_tokens_gradient_workspace(rows, k, c_in, &need)) return rc;
  SPIRA_HIP_REQUIRE(workspace_bytes >= need && (workspace || need == 0),
                    "grouped_linear_tokens_gradient: workspace too small");
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    grouped::RowsArgs a{{offsets, groups, rows}, nullptr, rows, dz, weights, nullptr, c_out, c_in, 0, workspace};
    // (one share a token is the sum: it is rounded at once, and takes half the bytes)
    if (k == 1) {
      if (rows > 0)
        if (int rc = grouped::launch_rows<T, false>(a, stream)) return rc;
      return spira_hip_combine(workspace, rows, slots, nullptr, tokens, k, c_in, dtype, dx, stream);
    }
    // (more stay fp32: 16 bits would round shares that cancel, and lose those past 65504.  It costs their bytes,
    // 585 -> 638 us for a step of 16k tokens, two choices, 1024 -> 2048)
    if (rows > 0)
      if (int rc = grouped::launch_rows<T, false, float>(a, stream)) return rc;
    return sum_slots(static_cast<const float *>(workspace), rows, slots, tokens, k, c_in, dtype, dx, stream);
  });
}

int spira_hip_grouped_linear_weights_gradient_workspace(int64_t rows, int groups, int c_in, int c_out, size_t *bytes) {
  if (int rc = grouped::check_sizes(rows, groups, c_in, c_out)) return rc;
  const int part = grouped::weight_parts(rows, groups, c_in, c_out);
  *bytes = part == 0 ? 0 : grouped::most_parts(rows, groups, part) * static_cast<size_t>(c_in) * c_out * sizeof(float);
  return kOk;
}

int spira_hip_grouped_linear_weights_gradient(int64_t rows, int groups, const int32_t *offsets, const int32_t *sources,
                                              int64_t num_sources, const void *x, int c_in, const void *dz, int c_out,
                                              int dtype, void *dw, void *workspace, size_t workspace_bytes,
                                              hipStream_t stream) {
  if (int rc = grouped::check(rows, groups, offsets, c_in, c_out)) return rc;
  SPIRA_HIP_REQUIRE(dw && (rows == 0 || dz) && (x || num_sources == 0) && num_sources >= 0 &&
                        (sources || num_sources >= rows),
                    "grouped_linear_weights_gradient: null tensor or too few sources");
  size_t need = 0;
  spira_hip_grouped_linear_weights_gradient_workspace(rows, groups, c_in, c_out, &need);
  SPIRA_HIP_REQUIRE(workspace_bytes >= need && (workspace || need == 0),
                    "grouped_linear_weights_gradient: workspace too small");
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const int part = grouped::weight_parts(rows, groups, c_in, c_out);
    grouped::WeightsArgs a{{offsets, groups, rows}, sources, num_sources, x, dz, c_in, c_out, part,
                           part ? static_cast<float *>(workspace) : nullptr, dw};
    const int64_t z = part ? grouped::most_parts(rows, groups, part) : groups;
    if (grouped::dma_fits<T>(a)) {
      if (int rc = grouped::launch_weights<T>(a, z, stream)) return rc;
    } else
      hipLaunchKernelGGL(grouped::weights_kernel<T>,
                       dim3(div_up(c_out, grouped::kCols), div_up(c_in, grouped::kRows), z), dim3(grouped::kThreads), 0,
                       stream, a);
    SPIRA_HIP_LAUNCH_CHECK();
    if (part) {
      const int64_t size = static_cast<int64_t>(c_in) * c_out;
      hipLaunchKernelGGL(grouped::join_kernel<T>, dim3(div_up(size, 64), groups), dim3(256), 0, stream, a.g, part, z,
                         a.partial, size, static_cast<T *>(dw));
      SPIRA_HIP_LAUNCH_CHECK();
    }
    return kOk;
  });
}

int spira_hip_grouped_linear_activation_gradient_workspace(int64_t rows, int groups, int c_out, int dtype,
                                                           size_t *bytes) {
  if (int rc = grouped::check_sizes(rows, groups, 1, c_out)) return rc;
  return with_type(dtype, [&](auto t) -> int {
    const int64_t part = grouped::sum_rows<decltype(t)>(rows, groups, c_out);
    *bytes = grouped::most_parts(rows, groups, part) * static_cast<size_t>(c_out) * sizeof(float);
    return kOk;
  });
}

int spira_hip_grouped_linear_activation_gradient(int64_t rows, int groups, const int32_t *offsets, const void *dy,
                                                 const void *y, int c_out, int dtype, void *dz, void *dbias,
                                                 void *workspace, size_t workspace_bytes, hipStream_t stream) {
  if (int rc = grouped::check(rows, groups, offsets, 1, c_out)) return rc;
  SPIRA_HIP_REQUIRE((rows == 0 || dy) && (y == nullptr || dz || rows == 0) && (y || dbias),
                    "grouped_linear_activation_gradient: null tensor");
  return with_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const int64_t part = grouped::sum_rows<T>(rows, groups, c_out);
    const int64_t parts = grouped::most_parts(rows, groups, part);
    SPIRA_HIP_REQUIRE(!dbias || workspace_bytes >= static_cast<size_t>(parts) * c_out * sizeof(float),
                      "grouped_linear_activation_gradient: workspace too small");
    const grouped::Groups g{offsets, groups, rows};
    auto *partial = dbias ? static_cast<float *>(workspace) : nullptr;
    if (rows > 0) {
      hipLaunchKernelGGL(grouped::activation_kernel<T>, dim3(div_up(c_out, 16 * kVec<T>), parts), dim3(256), 0, stream,
                         g, static_cast<int>(part), static_cast<const T *>(dy), static_cast<const T *>(y), c_out,
                         static_cast<T *>(dz), partial);
      SPIRA_HIP_LAUNCH_CHECK();
    }
    if (dbias) {
      hipLaunchKernelGGL(grouped::join_kernel<T>, dim3(div_up(c_out, 64), groups), dim3(256), 0, stream, g,
                         static_cast<int>(part), parts, partial, static_cast<int64_t>(c_out), static_cast<T *>(dbias));
      SPIRA_HIP_LAUNCH_CHECK();
    }
    return kOk;
  });
}

}  // extern "C"
