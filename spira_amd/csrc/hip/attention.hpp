// What the attention kernels share: packed sequences and their tiles, tiles of
// rows in LDS, fragments of the 32 x 32 matrix instructions.
//
// All products put the rows that a tile holds (keys; in the keys' gradient,
// queries) first and the columns that a wave owns (queries; keys) second, so that
// a lane's sums belong to one column, that of lane % 32:
//
//   scores  S^T = K Q^T        (a lane: 16 of 32 keys, the lane 32 on the others)
//   output  O^T += V^T P^T     (P^T: the scores' registers as they are)
//
// Statistics of a column need no broadcast, and P goes from the first product's
// sums to the second's operand without a move: in the sums, register r of half h =
// lane / 32 is row 8 (r / 4) + 4 h + r % 4, so a step of 16 rows takes registers 8
// s to 8 s + 7, and the other operand's fragment takes rows 4 h + {0..3} and 8 + 4
// h + {0..3}, which two transposing LDS reads give (ds_read_b64_tr_b16).
#pragma once

#include "tiles.hpp"

namespace spira_hip {

namespace attention {

using namespace tiles;

typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kMostHeadDim = 128;

// ---------------------------------------------------------------------------
// sequences
// ---------------------------------------------------------------------------
// Sequence b has the queries offsets[b] to offsets[b + 1] and the first
// key_counts[b] (or all) of the keys key_offsets[b] to key_offsets[b + 1].
struct Sequences {
  const int32_t *offsets, *key_offsets, *key_counts;
  int count;
  int64_t rows, keys;
};
struct Sequence {
  int64_t q0, k0;  // first query and key
  int nq, nk;
  int room;  // keys and the room behind them
};

// (whatever the numbers are, no row outside the tensors)
__device__ __forceinline__ int64_t clamp_row(int64_t v, int64_t most) { return v < 0 ? 0 : v > most ? most : v; }
__device__ __forceinline__ Sequence sequence_at(const Sequences &s, int b) {
  const int64_t q0 = clamp_row(s.offsets[b], s.rows), q1 = clamp_row(s.offsets[b + 1], s.rows);
  const int64_t k0 = clamp_row(s.key_offsets[b], s.keys), k1 = clamp_row(s.key_offsets[b + 1], s.keys);
  const int counted = s.key_counts ? s.key_counts[b] : INT32_MAX;
  Sequence r{q0, k0, q1 > q0 ? static_cast<int>(q1 - q0) : 0, 0, k1 > k0 ? static_cast<int>(k1 - k0) : 0};
  r.nk = counted < 0 ? 0 : counted < r.room ? counted : r.room;
  return r;
}

// Which sequence, and which piece of it.  A lane holds a sequence's numbers while the
// wave looks; the one found goes to all from there.
struct Found : Sequence {
  bool there;
  int nth, of;  // the piece within its sequence, and their number
};
__device__ __forceinline__ Found found_at(const Sequence &held, int lane, int nth, int of) {
  Found f;
  f.q0 = uniform(static_cast<int64_t>(__shfl(held.q0, lane, 64)));
  f.k0 = uniform(static_cast<int64_t>(__shfl(held.k0, lane, 64)));
  f.nq = uniform(__shfl(held.nq, lane, 64));
  f.nk = uniform(__shfl(held.nk, lane, 64));
  f.room = uniform(__shfl(held.room, lane, 64));
  f.there = true;
  f.nth = uniform(nth);
  f.of = uniform(of);
  return f;
}
// Sequences cut into pieces: of `size` keys (their room), or of `size` columns, `scale` to a
// query.
struct Cut {
  bool keys;
  int scale, size;  // (columns and keys are less than 2^31)
  __device__ __forceinline__ int pieces(const Sequence &x) const {
    const uint32_t all = static_cast<uint32_t>(keys ? x.room : x.nq) * scale;
    return static_cast<int>((all + size - 1) / static_cast<uint32_t>(size));
  }
  // Where sequence b's pieces begin among the launch's blocks: what the rows before it fill,
  // and a block for each sequence.  No less than its pieces lie between it and the next
  // one's, and all end at what the rows fill and a block for each.
  __device__ __forceinline__ int64_t start(const Sequences &s, int b) const {
    return clamp_row((keys ? s.key_offsets : s.offsets)[b], keys ? s.keys : s.rows) * scale / size + b;
  }
};

// Block `index`'s piece, the same on every lane: the sequence by bisection, 64 places at
// once.  (Counting the pieces before it took 25000 windows of 8 voxels 4.1 ms.)
__device__ __forceinline__ Found find_piece(const Sequences &s, int64_t index, const Cut &cut) {
  const int lane = lane_id();
  int lo = 0;
  for (int hi = s.count; hi - lo > 1;) {
    const int step = (hi - lo + 63) / 64, b = lo + lane * step;
    const uint64_t before = ballot(b < hi && cut.start(s, b) <= index);
    const int at = before ? 63 - __builtin_clzll(before) : 0;
    lo += at * step;
    hi = std::min(hi, lo + step);
  }
  lo = uniform(lo);
  const Sequence held = sequence_at(s, lo);
  const int64_t nth = index - cut.start(s, lo);
  const int of = cut.pieces(held);
  if (nth < 0 || nth >= of) return Found{};
  return found_at(held, 0, static_cast<int>(nth), of);
}

// Piece `index` in the order of what is left of its sequence from it on, the most
// first: with a causal mask that is a piece's work, and the longest begin first.  nth
// is what is left behind it (0: the sequence's last).  Lanes hold the sequences; of more
// than 64, sequence by sequence.
__device__ __forceinline__ Found find_longest(const Sequences &s, int64_t index, const Cut &cut) {
  if (s.count > 64) {
    Found f = find_piece(s, index, cut);
    f.nth = f.of - 1 - f.nth;
    return f;
  }
  const int lane = lane_id();
  const Sequence held = sequence_at(s, lane < s.count ? lane : s.count - 1);
  const int n = lane < s.count ? cut.pieces(held) : 0;
  // pieces with more than r left, themselves among it: the sum of max(0, n - r)
  const auto longer = [&](int r) {
    int64_t sum = n > r ? n - r : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    return uniform(sum);
  };
  int most = n;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) most = std::max(most, __shfl_xor(most, o, 64));
  int lo = 0, hi = uniform(most);  // longer(lo) > index >= longer(hi)
  if (longer(0) <= index) return Found{};
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (longer(mid) > index) lo = mid;
    else hi = mid;
  }
  const int64_t rank = index - longer(hi);
  const uint64_t level = ballot(n >= hi);
  const int b = __builtin_ctzll(ballot((level >> lane & 1) && lane_prefix(level) == rank));
  return found_at(held, b, hi - 1, __shfl(n, b, 64));
}

// zeros in the rows (of `width` values) that no sequence covers, by the launch's
// blocks together
template <class T>
__device__ void clear_uncovered(const int32_t *offsets, int count, int64_t rows, T *y, int64_t width, int64_t block,
                                int64_t blocks) {
  const int64_t lo = clamp_row(offsets[0], rows), last = clamp_row(offsets[count], rows), hi = last > lo ? last : lo;
  const int64_t chunks = (width + kVec<T> - 1) / kVec<T>, open = lo + rows - hi;
  for (int64_t i = block * blockDim.x + threadIdx.x; i < open * chunks; i += blocks * blockDim.x) {
    const int64_t k = i / chunks, r = k < lo ? k : hi + k - lo, at = (i - k * chunks) * kVec<T>;
    store_chunk(y + r * width + at, width - at, Chunk<T>{});
  }
}

// ---------------------------------------------------------------------------
// tiles of rows in LDS
// ---------------------------------------------------------------------------
// Rows of DP values (the head's, rounded up to 32) at a pitch of a power of two.
// The 16-byte chunk c of row r lies at slot c ^ swizzle(r): 16 consecutive rows'
// chunk c, and four consecutive rows' 64 bytes, each meet all banks once.
template <class T, int DP> struct Rows {
  static constexpr int SIZE = static_cast<int>(sizeof(T));
  static constexpr int PITCH = (DP == 96 ? 128 : DP) * SIZE;  // bytes
  static constexpr int CPR = PITCH / 16;                      // chunks a row
  static constexpr int STEPS = DP / 16, TILES = DP / 32;
  __device__ static __forceinline__ int swizzle(int r) {
    if constexpr (PITCH == 64) return (r >> 2) & 3;
    else if constexpr (PITCH == 128) return ((r & 2) << 1) | ((r >> 2) & 3);
    else return ((r & 3) << 2) | ((r >> 2) & 3);
  }
  __device__ static __forceinline__ int at(int r, int c) { return r * PITCH + ((c ^ swizzle(r)) << 4); }
};

// eight values of the summed index
template <class T> struct Frag {
  uintx4_t v[sizeof(T) / 2];
};

template <class T> __device__ __forceinline__ void mma(floatx16 &d, const Frag<T> &a, const Frag<T> &b) {
  if constexpr (std::is_same_v<T, _Float16>) {
    d = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a.v[0]), __builtin_bit_cast(half8, b.v[0]), d,
                                               0, 0, 0);
  } else if constexpr (std::is_same_v<T, __bf16>) {
    d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a.v[0]), __builtin_bit_cast(bf8, b.v[0]), d, 0,
                                                0, 0);
  } else {
    // (element i of both halves' eight: the summed index in another order, the same
    // for both operands)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const floatx4_t x = __builtin_bit_cast(floatx4_t, a.v[i]), y = __builtin_bit_cast(floatx4_t, b.v[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) d = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], d, 0, 0, 0);
    }
  }
}

// Registers 8 s to 8 s + 7 of sums as an operand.  For 16 bits each is rounded to
// the inputs' type, as the matrix instructions take it: half a step of a term of
// the sum that follows, which itself is rounded to that type once.
template <class T> __device__ __forceinline__ Frag<T> as_operand(const floatx16 &p, int s) {
  Frag<T> f;
  if constexpr (sizeof(T) == 2) {
    typedef float float2v __attribute__((ext_vector_type(2)));
    typedef T pair __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (two at a time: one instruction)
      const pair t = __builtin_convertvector((float2v{p[8 * s + 2 * i], p[8 * s + 2 * i + 1]}), pair);
      f.v[0][i] = __builtin_bit_cast(uint32_t, t);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      f.v[i] = __builtin_bit_cast(uintx4_t, floatx4_t{p[8 * s + 4 * i], p[8 * s + 4 * i + 1], p[8 * s + 4 * i + 2],
                                                      p[8 * s + 4 * i + 3]});
  }
  return f;
}

// The same of 16 bits and of numbers that are not negative, rounded to below them by 2^-12 of
// themselves or more: what is left is positive wherever they are, and an infinity that
// both parts are multiplied with stays one.
template <class T> __device__ __forceinline__ Frag<T> below_operand(const floatx16 &p, int s) {
  Frag<T> f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = p[8 * s + 2 * i] * (1 - 0x1p-12f), b = p[8 * s + 2 * i + 1] * (1 - 0x1p-12f);
    if constexpr (std::is_same_v<T, _Float16>) f.v[0][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    else f.v[0][i] = __builtin_bit_cast(uint32_t, a) >> 16 | (__builtin_bit_cast(uint32_t, b) & 0xFFFF0000u);
  }
  return f;
}

// What as_operand's rounding left of them, as another operand: with both, the sums that
// follow are as good as in fp32.
template <class T> __device__ __forceinline__ Frag<T> rest_operand(const floatx16 &p, int s, const Frag<T> &rounded) {
  T t[8];
  __builtin_memcpy(t, &rounded, sizeof(t));
  floatx16 rest{};
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = p[8 * s + i] - to_float(t[i]);
  return as_operand<T>(rest, 0);
}

// Where a lane reads of a tile.  What a fragment's number changes of an address is
// bits that the swizzle has not moved together: an exclusive or of a constant, and
// a constant offset.
template <class T, int DP> struct Reader {
  using R = Rows<T, DP>;
  uint32_t row, col;  // LDS addresses in the tile
  __device__ __forceinline__ explicit Reader() {
    const int lane = lane_id(), h = lane >> 5;
    row = R::at(lane & 31, h * (R::SIZE / 2));
    if constexpr (sizeof(T) == 2) {
      const int i = lane & 15;
      col = R::at(4 * h + (i >> 2), ((lane >> 4) & 1) * 2 + ((i & 3) >> 1)) + (i & 1) * 8;
    } else {
      col = R::at(4 * h, (lane & 31) >> 2) + (lane & 3) * 4;
    }
  }
  // rows r0 to r0 + 31 as the first operand of step st of 16 values
  __device__ __forceinline__ Frag<T> rows(lds_char *tile, int r0, int st) const {
    Frag<T> f;
#pragma unroll
    for (int i = 0; i < R::SIZE / 2; ++i) f.v[i] = *(lds_chunk *)(tile + r0 * R::PITCH + (row ^ (st * 16 * R::SIZE + i * 16)));
    return f;
  }
  // values 32 n to 32 n + 31 as the first operand, summed over rows r0 to r0 + 15
  __device__ __forceinline__ Frag<T> cols(lds_char *tile, int r0, int n) const {
    Frag<T> f;
    lds_char *at = tile + r0 * R::PITCH;
    if constexpr (sizeof(T) == 2) {
      const auto lo = read_tr(at + (col ^ (n * 64))), hi = read_tr(at + 8 * R::PITCH + (col ^ (n * 64 + 32)));
      const uintx2_t a = __builtin_bit_cast(uintx2_t, lo), b = __builtin_bit_cast(uintx2_t, hi);
      f.v[0] = {a[0], a[1], b[0], b[1]};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // (row i % 4 and the rows 8 behind change the swizzle as R::at says)
        const int r = (i / 4) * 8 + i % 4;
        f.v[i / 4][i % 4] = *(lds_word *)(at + r * R::PITCH + (col ^ (n * 128) ^ (R::swizzle(r) << 4)));
      }
    }
    return f;
  }
};
// a column's row of memory as the second operand of step st, zeros past d and
// without a row
template <class T> __device__ __forceinline__ Frag<T> load_frag(const T *row, int d, int st) {
  Frag<T> f;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
    const int at = st * 16 + (lane_id() >> 5) * 8 + i * kVec<T>;
    f.v[i] = load_raw(row + at, row ? d - at : 0);
  }
  return f;
}

// Tiles of R rows from memory to LDS by NT threads (of which this is `thread`): n rows
// of `stride` bytes, zeros behind them and behind a row's d values.
// DMA (rows, strides and addresses of whole 16-byte chunks): under way on return, a
// load of 1 KB per wave and instruction; chunks outside are out of the buffer's
// range.  Else through registers, written on return.
template <class T, int DP, int R, int NT, bool DMA> struct Fetch {
  using S = Rows<T, DP>;
  static constexpr int LOADS = R * S::CPR / NT;
  // rows from one load to the next, whose chunks a thread takes in the same order where
  // these are whole swizzles
  static constexpr int TURN = NT / S::CPR;
  static constexpr bool SAME = TURN % 16 == 0;
  static_assert(LOADS >= 1 && LOADS * NT == R * S::CPR, "tile shape");
  int64_t stride;
  int thread, d;
  uint32_t first[SAME ? 1 : LOADS];
  __device__ __forceinline__ Fetch(int64_t stride, int d, int thread) : stride(stride), thread(thread), d(d) {
    if constexpr (DMA) {
#pragma unroll
      for (int i = 0; i < (SAME ? 1 : LOADS); ++i) {
        const int id = i * NT + thread, r = id / S::CPR, c = (id % S::CPR) ^ S::swizzle(r);
        first[i] = c * 16 < d * S::SIZE ? static_cast<uint32_t>(r) * static_cast<uint32_t>(stride) + c * 16 : kOutOfRange;
      }
    }
  }
  __device__ __forceinline__ void operator()(const char *rows, int64_t n, lds_char *tile) const {
    if constexpr (DMA) {
      lds_char *to = tile + (thread & ~63) * 16;
      const auto bytes = [&](int64_t m, int64_t most) {
        m = m < most ? m : most;
        return m > 0 ? (m - 1) * stride + d * S::SIZE : int64_t(0);
      };
      if constexpr (SAME) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
          load_lds(buffer(rows + i * TURN * stride, bytes(n - i * TURN, TURN)), first[0], (lds_void *)(to + i * NT * 16));
      } else {
        const uintx4_t from = buffer(rows, bytes(n, R));
#pragma unroll
        for (int i = 0; i < LOADS; ++i) load_lds(from, first[i], (lds_void *)(to + i * NT * 16));
      }
    } else {
      uintx4_t v[LOADS];
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int id = i * NT + thread, r = id / S::CPR, c = (id % S::CPR) ^ S::swizzle(r);
        v[i] = load_raw(reinterpret_cast<const T *>(rows + r * stride) + c * kVec<T>, r < n ? d - c * kVec<T> : 0);
      }
#pragma unroll
      for (int i = 0; i < LOADS; ++i) *(lds_chunk *)(tile + (i * NT + thread) * 16) = v[i];
    }
  }
};

// step(t, stage) for t in [0, n), the two stages in turn from `first` on
template <class Step> __device__ __forceinline__ void ring(int n, int first, Step &&step) {
  using std::integral_constant;
  int t = 0;
  if (first == 1 && n > 0) {
    step(0, integral_constant<int, 1>{});
    t = 1;
  }
  while (t < n) {
    step(t, integral_constant<int, 0>{});
    if (++t == n) break;
    step(t, integral_constant<int, 1>{});
    ++t;
  }
}

// the larger (or the sum) of the two halves' values of a column
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

// ---------------------------------------------------------------------------
// infinities and NaN where the mask hides them
// ---------------------------------------------------------------------------
// A hidden row's weight is 0, and 0 times an infinity or NaN is NaN: where some
// columns see a row and others do not, such values are taken out of the tile before
// its product and added to the columns that see them, from memory.

// Zeros for what is not finite in a tile's R rows, by NT threads; whether this one
// found any.
template <class T, int DP, int R, int NT> __device__ __forceinline__ bool clear_not_finite(lds_char *tile, int thread) {
  constexpr uint32_t E = sizeof(T) == 4 ? 0x7F800000u : std::is_same_v<T, _Float16> ? 0x7C00u : 0x7F80u;
  // (heads of up to 32 values in 16 bits: 32 rows have fewer chunks than a block has threads)
  constexpr int CHUNKS = R * Rows<T, DP>::CPR;
  bool found = false;
#pragma unroll
  for (int i = 0; i < (CHUNKS + NT - 1) / NT; ++i) {
    if (CHUNKS % NT != 0 && i * NT + thread >= CHUNKS) break;
    lds_chunk *at = (lds_chunk *)(tile + (i * NT + thread) * 16);
    uintx4_t v = *at;
    bool here = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if ((v[j] & E) == E) {
        v[j] &= sizeof(T) == 4 ? 0u : 0xFFFF0000u;
        here = true;
      }
      if (sizeof(T) == 2 && ((v[j] >> 16) & E) == E) {
        v[j] &= 0xFFFFu;
        here = true;
      }
    }
    if (here) *at = v;
    found |= here;
  }
  return found;
}

// acc += what is not finite in n rows of memory, for the columns that see the row
// (sees(i): whether this lane's does)
template <class T, int DP, class Sees>
__device__ __forceinline__ void add_not_finite(floatx16 (&acc)[DP / 32], const char *rows, int64_t stride, int n, int d,
                                               Sees &&sees) {
  const int h = lane_id() >> 5;
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    const T *row = reinterpret_cast<const T *>(rows + i * stride) + 4 * h;
    const bool seen = sees(i);
#pragma unroll
    for (int m = 0; m < DP / 32; ++m)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int at = 32 * m + 8 * (r / 4) + r % 4;
        const float v = at + 4 * h < d ? to_float(row[at]) : 0.f;
        if (seen && !(__builtin_fabsf(v) < __builtin_inff())) acc[m][r] += v;
        if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (few registers: it is a rare path)
      }
  }
}

// ---------------------------------------------------------------------------
// columns to memory
// ---------------------------------------------------------------------------
// A column's sums times `by` to its row of d values, and what their rounding left of them
// to another (or null).  The halves exchange groups of four values, so that each lane
// writes eight consecutive ones.  Every lane takes part; `there`: its column is to be
// written.
template <class T, int DP>
__device__ __forceinline__ void store_column(T *row, int d, bool there, const floatx16 (&acc)[DP / 32], float by,
                                             T *rest = nullptr) {
  const int h = lane_id() >> 5;
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, acc[n][8 * m + i] * by),
                                                        __builtin_bit_cast(uint32_t, acc[n][8 * m + 4 + i] * by), false,
                                                        false);
        v[i] = __builtin_bit_cast(float, static_cast<uint32_t>(s[0]));
        v[4 + i] = __builtin_bit_cast(float, static_cast<uint32_t>(s[1]));
      }
      const int at = 32 * n + 8 * (2 * m + h);
#pragma unroll
      for (int c = 0; c < 8 / kVec<T>; ++c) {
        Chunk<T> k;
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) k.v[i] = v[c * kVec<T> + i];
        if (there) store_chunk(row + at + c * kVec<T>, d - at - c * kVec<T>, k);
        if (there && rest) {
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i) k.v[i] -= to_float(from_float<T>(k.v[i]));
          store_chunk(rest + at + c * kVec<T>, d - at - c * kVec<T>, k);
        }
      }
    }
}

// whether tiles (of at most 64 rows) can be fetched by DMA: their rows' zeros behind the last
// one come from the buffer's end, so no row may begin before the end of the one before it
inline bool dma_rows(const void *p, int64_t row, int64_t head, int d, int size) {
  const auto whole = [&](int64_t values) { return values * size % 16 == 0; };
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row >= d && whole(row) && whole(head) && whole(d) &&
         row * size * 64 < kBufferLimit / 2;
}

// f of the head's padded width
template <class F> int with_width(int d, F &&f) {
  using std::integral_constant;
  if (d <= 32) return f(integral_constant<int, 32>{});
  if (d <= 64) return f(integral_constant<int, 64>{});
  if (d <= 96) return f(integral_constant<int, 96>{});
  return f(integral_constant<int, 128>{});
}

// The sums of a wave's 32 columns to LDS, [32][DP + 4], where the waves of a block share
// the columns.
template <int DP> constexpr int kSumPitch = DP + 4;
template <int DP> __device__ __forceinline__ void put_sums(float *to, const floatx16 (&acc)[DP / 32]) {
  float *at = to + (lane_id() & 31) * kSumPitch<DP> + 4 * (lane_id() >> 5);
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<floatx4_t *>(at + 32 * n + 8 * g) =
          floatx4_t{acc[n][4 * g], acc[n][4 * g + 1], acc[n][4 * g + 2], acc[n][4 * g + 3]};
}

constexpr int kKeysByDma = 1, kQueriesByDma = 2;

// Strides in values.
struct Args {
  Sequences s;
  int heads, kv_heads, group, d, causal, dma;
  float scale;   // of the scores
  float scale2;  // scale log2 e
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  void *o;       // [rows, heads, d]
  float *stats;  // [heads, rows] log2 of the sum of exp2 of a row's scaled scores, less kLift; fp32: [2, heads,
                 // rows], their largest and the inverse of the sum beside it
  void *rest;    // [rows, heads, d], 16 bits: what the outputs' rounding left of them, for delta
  // few tokens
  float *partial, *partial_stats;
  int part_keys;  // keys a part
  // backward
  const void *dout, *out;
  float *delta;  // [heads, rows]
  void *dq, *dk, *dv;
};

// ---------------------------------------------------------------------------
// columns of queries
// ---------------------------------------------------------------------------
constexpr int kColumns = 128;  // of a block: a key head's query heads and their queries, heads fastest
// Whether blocks of 128 columns are too few to fill the CUs: then a block owns 32, and its
// waves share out the keys.  Forward, four sequences, heads of 64 (causal, 8 on 2): bf16 136
// blocks of 128 columns 16.1 us, of 32 15.3; 264 blocks 25.1 and 32.5.  fp32 72 blocks 28.1
// and 15.9, 258 (one sequence) 334 and 230, its dq, dk and dv 801 and 617.
inline bool few_columns(const spira_hip_attention_t &x) {
  const int64_t blocks = (x.rows * (x.heads / x.kv_heads) / kColumns + x.sequences) * x.kv_heads;
  return blocks < (x.dtype == SPIRA_F32 ? 512 : 192);
}
// keys of a tile
template <class T> constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;

// keys that query i of a sequence sees
__device__ __forceinline__ int visible(const Args &a, const Sequence &s, int i) {
  if (!a.causal) return s.nk;
  const int n = s.nk - (s.nq - 1 - i);
  return n < 0 ? 0 : n < s.nk ? n : s.nk;
}

// fp16: weights take part in sums lifted by 2^14, and their statistics are kept so:
// those of long sequences, some 1 / n each, would be below 2^-14, where the type has
// fewer bits.
template <class T> constexpr int kLift = std::is_same_v<T, _Float16> ? 14 : 0;
template <class T> constexpr float kLower = 1.f / static_cast<float>(1 << kLift<T>);

// ds is lifted with the weight that it is made of: n of them are some sqrt(n) below the sum
// that they make, and would lose their bits long before it does.  Where a column's largest
// passes 2^15 so, its lift is lowered by a power of two that takes it to 2^10, and the sums
// follow (until it passes 2^15 again): what is held is good to 2^-39, or 2^-35 of the
// column's largest.  Gradients of 100k voxels, 3 heads of 32, windows of 1024: 231
// us without, 245 with, 256 where every column is lowered; 16k tokens, 16 heads of 64 on 4, 291,
// 292 and 299.
template <class T> struct Lift {
  float by = 1;
  uint64_t lowered = 0;  // (lanes that have been, of the wave)
  template <int N> __device__ __forceinline__ void fit(floatx16 &ds, floatx16 (&acc)[N]) {
    if constexpr (kLift<T> > 0) {
      constexpr float most = 0x1p15f;
      float top = 0;
#pragma unroll
      for (int r = 0; r < 16; ++r) top = __builtin_fmaxf(top, __builtin_fabsf(ds[r]));
      const uint64_t over = ballot(top * by > most);
      if (over | lowered) {
        if (over) {
          // (both halves of a column as one)
          top = __builtin_fmaxf(top, other_half(top));
          const float next = top * by > most ? __builtin_ldexpf(1.f, 11 - __builtin_amdgcn_frexp_expf(top)) : by;
          const float ratio = next * (1.f / by);
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[n][r] *= ratio;
          by = next;
          lowered |= over;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] *= by;
      }
    }
  }
  __device__ __forceinline__ float lower() const { return kLift<T> > 0 ? kLower<T> / by : 1.f; }
};

// a row's statistics, and p from a raw score
template <class T> struct Stat {
  float base, by;
};
template <class T> __device__ __forceinline__ float weight(float s, float scale2, const Stat<T> &r) {
  const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s, scale2, -r.base));
  // (in fp32 the logarithm of the sum would be rounded to as much as 1e-6 of p)
  return sizeof(T) == 2 ? e : e * r.by;
}

int arguments(const spira_hip_attention_t &x, Args &a, int size);  // (attention.hip)
// (attention_keys.hip)
int key_splits(const spira_hip_attention_t &x);
size_t key_sums_bytes(const spira_hip_attention_t &x);
int key_gradients(const spira_hip_attention_t &x, const Args &a, hipStream_t stream);

// bytes of the gradients' workspace before the keys' sums: delta
inline size_t delta_bytes(const spira_hip_attention_t &x) {
  return round_up(static_cast<int64_t>(x.rows) * x.heads * static_cast<int64_t>(sizeof(float)), 256);
}

}  // namespace attention

}  // namespace spira_hip
