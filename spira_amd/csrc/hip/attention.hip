// Attention over packed sequences (gfx950), forward:
//
//   s_ij = scale q_i . k_j,  p_ij = exp(s_ij) / sum over the visible j of exp(s_ij),  o_i = sum_j p_ij v_j
//
// with `group` query heads to a key head; causal: query i of n sees key j of m if
// j <= i + m - n.  A row that sees no key gets zeros.
//
// Two forms.  Prompts: a block owns 128 columns (a key head's query heads and
// their queries, heads fastest), four waves of 32, and walks the keys in tiles
// that it holds in LDS, the next one under way while it multiplies.  Few tokens:
// the keys of a sequence are cut into parts, a block's one to four waves (by a row's
// bytes) walk a part's tiles each on their own (without barriers) for the same 32
// columns, and the parts are joined by a second launch.
//
// Prompts are bound by the matrix and the vector units in turn, and by power: 16 heads of
// 128 on 4 over 16384 tokens, causal, bf16: 1180 us = 931 TFLOP/s (8192^3 product of the
// library 1126), matrix cores busy 38 % at 2.05 GHz; heads of 32 over windows of 1024 voxels
// 85 us, vector instructions issuing for 56 % of it and the matrix cores busy for 19 %.  Few
// tokens are bound by memory: 32 caches of 4096 keys on average, 8 heads of 128: 121 us, 4.5
// TB/s in the kernel.
//
// In 16 bits weights are rounded to the features' type before their product, half a step of
// each term.  For few tokens and on the mask's edge a second operand holds what that leaves (one
// token against 700 keys 11.6 us without, 12.3 with; 32 caches 116 and 118; 100 queries against
// 100k keys 115 and 117), and outputs are as good as fp32 arithmetic's, rounded once.  Whole tiles
// of prompts go without: outputs are off by 1.2 to 1.4 times as much, and with it that prompt took
// 1623 us and the voxels 109.
//
// The softmax is taken in one pass with a running maximum and sum in fp32.  The
// maximum moves only when a score passes it by 2^8 (in exp2; fp16 2^4): the sums are
// exact under any reference, and columns are seldom scaled anew.
#include "attention.hpp"

#include <algorithm>

namespace spira_hip {

namespace attention {

// fp16: weights are lifted by 2^11 over that reference (2^15 at most, the type ends at 2^16): the
// many of some e^-17 beside one that takes nearly all would be a step or none of the type's 2^-24.
template <class T> constexpr float kRaise = std::is_same_v<T, _Float16> ? 11.f : 0.f;
template <class T> constexpr float kSlack = std::is_same_v<T, _Float16> ? 4.f : 8.f;

// The reference in exp2: rounded once, and so wherever sums of another reference are joined (as
// part of a longer expression it would not be).
__device__ __forceinline__ float reference(float m, float scale2) {
#pragma clang fp contract(off)
  return m * scale2;
}

// a wave's 32 columns on their way: output, reference maximum of the raw scores
// (-inf: nothing seen) and this half's share of the sum
template <int DP> struct Columns {
  floatx16 o[DP / 32];
  float m, l;
};

// One tile of KT keys.  MASKED: this lane's column sees the first `limit` of them (any
// number); else every column of the wave sees all.  FINE (16 bits): the weights with what
// their rounding leaves.
template <bool MASKED, bool FINE, class T, int DP, int KT>
__device__ __forceinline__ void attend_tile(Columns<DP> &c, const Frag<T> (&q)[DP / 16], const Reader<T, DP> &read,
                                            lds_char *kt, lds_char *vt, float scale2, int limit) {
  floatx16 s[KT / 32];
#pragma unroll
  for (int u = 0; u < KT / 32; ++u) {
    s[u] = floatx16{};
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) mma(s[u], read.rows(kt, 32 * u, st), q[st]);
  }
  if constexpr (MASKED) {
    const int mine = limit - 4 * (lane_id() >> 5);
#pragma unroll
    for (int u = 0; u < KT / 32; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 32 * u + 8 * (r / 4) + r % 4 < mine ? s[u][r] : -__builtin_inff();
  }
  float top = s[0][0];
#pragma unroll
  for (int u = 0; u < KT / 32; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) top = __builtin_fmaxf(top, s[u][r]);
  top = __builtin_fmaxf(top, other_half(top));
  // (each column by its own scores: a result does not depend on the wave's others)
  const bool moves = (top - c.m) * scale2 > kSlack<T>;
  if (ballot(moves)) {
    const float m = moves ? top : c.m, by = moves ? __builtin_amdgcn_exp2f(reference(c.m, scale2) - reference(m, scale2)) : 1.f;
    c.l *= by;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) c.o[n][r] *= by;
    c.m = m;
  }
  float base = c.m == -__builtin_inff() ? 0.f : -reference(c.m, scale2);
  if constexpr (kRaise<T> > 0) base += kRaise<T>;
#pragma unroll
  for (int u = 0; u < KT / 32; ++u) {
    float sum = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], scale2, base));
      sum += s[u][r];
    }
    c.l += sum;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      Frag<T> p, rest;
      if constexpr (FINE && sizeof(T) == 2) {
        p = below_operand<T>(s[u], st);
        rest = rest_operand<T>(s[u], st, p);
      } else {
        p = as_operand<T>(s[u], st);
      }
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) {
        const Frag<T> v = read.cols(vt, 32 * u + 16 * st, n);
        mma(c.o[n], v, p);
        if constexpr (FINE && sizeof(T) == 2) mma(c.o[n], v, rest);
      }
    }
  }
}

// a row's statistics for the gradients, from its reference (in exp2) and sum
template <class T>
__device__ __forceinline__ void put_statistics(const Args &a, int head, int64_t row, float m, float l) {
  float *to = a.stats + head * a.s.rows + row;
  const float base = m == -__builtin_inff() ? 0.f : m;
  if constexpr (sizeof(T) == 2) {
    *to = l == 0.f ? __builtin_inff() : base + __builtin_amdgcn_logf(l) - (kRaise<T> + kLift<T>);
  } else {
    to[0] = base;
    to[a.heads * a.s.rows] = l == 0.f ? 0.f : 1.f / l;
  }
}

// ---------------------------------------------------------------------------
// prompts
// ---------------------------------------------------------------------------
template <class T, int DP, bool DMA>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void prompt_kernel(const Args a) {
  using R = Rows<T, DP>;
  constexpr int KT = kKeys<T>, TILE = KT * R::PITCH;
  __shared__ __align__(1024) char lds[4 * TILE];
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6)), lane = lane_id();
  T *o = static_cast<T *>(a.o);
  clear_uncovered(a.s.offsets, a.s.count, a.s.rows, o, static_cast<int64_t>(a.heads) * a.d, blockIdx.x, gridDim.x);
  // (key heads fastest: where their number divides 8 or 8 it, an XCD's blocks share
  // few heads' keys)
  const int kv = blockIdx.x % a.kv_heads;
  const Found s = find_longest(a.s, blockIdx.x / a.kv_heads, Cut{false, a.group, kColumns});
  if (!s.there) return;
  const int total = s.nq * a.group, c0 = s.nth * kColumns, w0 = c0 + wave * 32;
  const int column = w0 + (lane & 31), j = column < total ? column : total - 1;
  const int i = j / a.group, head = kv * a.group + (j - i * a.group), limit = visible(a, s, i);
  const int most = w0 < total ? visible(a, s, std::min(w0 + 31, total - 1) / a.group) : 0;
  const int fewest = visible(a, s, c0 / a.group), end = visible(a, s, std::min(c0 + kColumns - 1, total - 1) / a.group);
  const int steps = (end + KT - 1) / KT, own = (most + KT - 1) / KT;
  const int64_t kstride = a.k_row * R::SIZE, vstride = a.v_row * R::SIZE;
  const char *keys = reinterpret_cast<const char *>(static_cast<const T *>(a.k) + s.k0 * a.k_row + kv * a.k_head);
  const char *values = reinterpret_cast<const char *>(static_cast<const T *>(a.v) + s.k0 * a.v_row + kv * a.v_head);
  const Fetch<T, DP, KT, 256, DMA> fetch_keys(kstride, a.d, threadIdx.x), fetch_values(vstride, a.d, threadIdx.x);
  const auto issue = [&](int t, int stage) {
    lds_char *to = (lds_char *)lds + stage * 2 * TILE;
    fetch_keys(keys + t * (KT * kstride), s.nk - t * KT, to);
    fetch_values(values + t * (KT * vstride), s.nk - t * KT, to + TILE);
  };
  if (steps > 0) issue(0, 0);
  Frag<T> q[DP / 16];
  {
    const T *row = static_cast<const T *>(a.q) + (s.q0 + i) * a.q_row + head * a.q_head;
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) q[st] = load_frag(row, a.d, st);
  }
  Columns<DP> c{};
  c.m = -__builtin_inff();
  const Reader<T, DP> read;
  // tiles that every column sees whole
  const int whole = std::min(fewest / KT, steps);
  ring(whole, 0, [&](int t, auto STAGE) {
    constexpr int stage = decltype(STAGE)::value;
    wait_loads_and_meet<0>();
    if (t + 1 < steps) issue(t + 1, stage ^ 1);
    lds_char *kt = (lds_char *)lds + stage * 2 * TILE;
    attend_tile<false, false, T, DP, KT>(c, q, read, kt, kt + TILE, a.scale2, 0);
  });
  // the others
  for (int t = whole; t < steps; ++t) {
    wait_loads_and_meet<0>();
    if (t + 1 < steps) issue(t + 1, (t + 1) & 1);
    lds_char *kt = (lds_char *)lds + (t & 1) * 2 * TILE;
    // (the same for the whole block)
    const bool found = a.causal && __syncthreads_or(clear_not_finite<T, DP, KT, 256>(kt + TILE, threadIdx.x));
    if (t < own) {
      const int mine = limit - t * KT;
      attend_tile<true, true, T, DP, KT>(c, q, read, kt, kt + TILE, a.scale2, mine);
      if (found)
        add_not_finite<T, DP>(c.o, values + t * (KT * vstride), vstride, std::min(s.nk - t * KT, KT), a.d,
                              [&](int x) { return x < mine; });
    }
  }
  const float l = c.l + other_half(c.l);
  const bool there = column < total;
  const int64_t at = ((s.q0 + i) * a.heads + head) * a.d;
  store_column<T, DP>(o + at, a.d, there, c.o, l == 0.f ? 0.f : 1.f / l, a.rest ? static_cast<T *>(a.rest) + at : nullptr);
  if (a.stats && there && lane < 32) put_statistics<T>(a, head, s.q0 + i, reference(c.m, a.scale2), l);
}

// ---------------------------------------------------------------------------
// few tokens
// ---------------------------------------------------------------------------
// Waves of a block, with two stages of two tiles of 32 keys each.  Parts of a long
// cache: blocks of 64 KB, two to a CU, so that one streams while the other begins.
// (32 caches of 4096 keys on average, 8 heads of 128: 125 us.  One wave a block with four
// stages, as many loads under way, 156; two with three stages, one block to a CU, 176:
// four waves a CU are what it takes to work off what arrives.)
template <class T, int DP, bool DIRECT> struct TokenShape {
  static constexpr int PITCH = Rows<T, DP>::PITCH;
  static constexpr int NW = DIRECT ? (PITCH >= 512 ? 2 : 4) : (PITCH >= 512 ? 1 : PITCH >= 256 ? 2 : 4);
};

// DIRECT: no sequence has more than one part; the outputs themselves
template <class T, int DP, bool DIRECT, bool DMA>
__global__ __launch_bounds__((64 * TokenShape<T, DP, DIRECT>::NW), 1) void token_kernel(const Args a) {
  using R = Rows<T, DP>;
  constexpr int KT = 32, TILE = KT * R::PITCH, NT = 64 * TokenShape<T, DP, DIRECT>::NW;
  constexpr int NW = TokenShape<T, DP, DIRECT>::NW;
  constexpr int LOADS = 2 * KT * R::CPR / 64, OPITCH = kSumPitch<DP>;
  static_assert(32 * OPITCH * 4 <= 4 * TILE, "a wave's sums take its stages' place");
  __shared__ __align__(1024) char lds[NW][4 * TILE];
  __shared__ float wm[NW][32], wl[NW][32], top[32], total_l[32];
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6)), lane = lane_id();
  lds_char *mine = (lds_char *)lds[wave];
  T *o = static_cast<T *>(a.o);
  if constexpr (DIRECT)
    clear_uncovered(a.s.offsets, a.s.count, a.s.rows, o, static_cast<int64_t>(a.heads) * a.d,
                    blockIdx.y * static_cast<int64_t>(gridDim.x) + blockIdx.x,
                    static_cast<int64_t>(gridDim.x) * gridDim.y);
  const int kv = blockIdx.x % a.kv_heads;
  // DIRECT: a piece is 32 columns (whose outputs are written without keys too); else a
  // part of the keys, for columns from blockIdx.y on
  const Found s = DIRECT ? find_longest(a.s, blockIdx.x / a.kv_heads, Cut{false, a.group, 32})
                         : find_piece(a.s, blockIdx.x / a.kv_heads, Cut{true, 1, a.part_keys});
  if (!s.there) return;
  const int first = DIRECT ? 0 : s.nth * a.part_keys, total = s.nq * a.group;
  if (!DIRECT && first >= s.nk) return;  // (room)
  const int64_t kstride = a.k_row * R::SIZE, vstride = a.v_row * R::SIZE;
  const char *keys = reinterpret_cast<const char *>(static_cast<const T *>(a.k) + (s.k0 + first) * a.k_row + kv * a.k_head);
  const char *values =
      reinterpret_cast<const char *>(static_cast<const T *>(a.v) + (s.k0 + first) * a.v_row + kv * a.v_head);
  const int part = DIRECT ? s.nk : std::min(s.nk - first, a.part_keys);
  const Fetch<T, DP, KT, 64, DMA> fetch_keys(kstride, a.d, lane), fetch_values(vstride, a.d, lane);
  const Reader<T, DP> read;
  for (int w0 = (DIRECT ? s.nth : blockIdx.y) * 32; w0 < total; w0 += gridDim.y * 32) {
    const int column = w0 + (lane & 31), j = column < total ? column : total - 1;
    const int i = j / a.group, head = kv * a.group + (j - i * a.group), limit = visible(a, s, i) - first;
    const int least = visible(a, s, w0 / a.group) - first;
    const int most = visible(a, s, std::min(w0 + 31, total - 1) / a.group) - first;
    const int end = std::min(part, most), steps = end > 0 ? (end + KT - 1) / KT : 0;
    const auto issue = [&](int t, int stage) {
      lds_char *to = mine + stage * 2 * TILE;
      const int64_t n = t < steps ? part - t * KT : 0;
      fetch_keys(keys + t * (KT * kstride), n, to);
      fetch_values(values + t * (KT * vstride), n, to + TILE);
    };
    issue(wave, 0);
    Frag<T> q[DP / 16];
    const T *row = static_cast<const T *>(a.q) + (s.q0 + i) * a.q_row + head * a.q_head;
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) q[st] = load_frag(row, a.d, st);
    // (waited for here, with the first tile: a later wait would be for the next one too)
#pragma unroll
    for (int st = 0; st < DP / 16; ++st)
#pragma unroll
      for (auto &v : q[st].v) asm volatile("" : "+v"(v));
    Columns<DP> c{};
    c.m = -__builtin_inff();
    for (int t = wave, stage = 0; t < steps; t += NW, stage ^= 1) {
      issue(t + NW, stage ^ 1);
      // until this tile's loads have landed (the next one's are on their way)
      static_assert(LOADS < 64, "vmcnt range");
      __builtin_amdgcn_s_waitcnt((LOADS & 15) | (7 << 4) | ((LOADS >> 4) << 14));
      asm volatile("" ::: "memory");
      lds_char *kt = mine + stage * 2 * TILE;
      if (std::min(least, part) >= (t + 1) * KT) {
        attend_tile<false, true, T, DP, KT>(c, q, read, kt, kt + TILE, a.scale2, 0);
        continue;
      }
      const bool found = a.causal && ballot(clear_not_finite<T, DP, KT, 64>(kt + TILE, lane)) != 0;
      const int seen = std::min(limit, part) - t * KT;
      attend_tile<true, true, T, DP, KT>(c, q, read, kt, kt + TILE, a.scale2, seen);
      if (found)
        add_not_finite<T, DP>(c.o, values + t * (KT * vstride), vstride, std::min(part - t * KT, KT), a.d,
                              [&](int x) { return x < seen; });
    }
    wait_loads();
    asm volatile("" ::: "memory");
    // the waves' columns to LDS, and their sum from there
    put_sums<DP>(reinterpret_cast<float *>(lds[wave]), c.o);
    const float l = c.l + other_half(c.l);
    if (lane < 32) {
      wm[wave][lane] = reference(c.m, a.scale2);
      wl[wave][lane] = l;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      float m = wm[0][lane], sum = 0;
#pragma unroll
      for (int w = 1; w < NW; ++w) m = __builtin_fmaxf(m, wm[w][lane]);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float by = wm[w][lane] == m ? 1.f : __builtin_amdgcn_exp2f(wm[w][lane] - m);
        sum += wl[w][lane] * by;
        wm[w][lane] = by;
      }
      top[lane] = m;
      total_l[lane] = sum;
    }
    __syncthreads();
    const int columns = std::min(32, total - w0);
    for (int k = threadIdx.x; k < columns * a.d; k += NT) {
      const int col = k / a.d, d = k - col * a.d;
      float v = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) v += wm[w][col] * reinterpret_cast<const float *>(lds[w])[col * OPITCH + d];
      const int q_at = (w0 + col) / a.group, h_at = kv * a.group + (w0 + col - q_at * a.group);
      const int64_t at = (s.q0 + q_at) * a.heads + h_at;
      const float sum = total_l[col];
      if constexpr (DIRECT) {
        const float value = sum == 0.f ? 0.f : v / sum;
        const T rounded = from_float<T>(value);
        o[at * a.d + d] = rounded;
        if (a.rest) static_cast<T *>(a.rest)[at * a.d + d] = from_float<T>(value - to_float(rounded));
      } else a.partial[(s.nth * a.s.rows * a.heads + at) * a.d + d] = v;
    }
    if constexpr (DIRECT) {
      if (a.stats && static_cast<int>(threadIdx.x) < columns)
        put_statistics<T>(a, head, s.q0 + i, top[lane], total_l[lane]);
      return;
    } else if (static_cast<int>(threadIdx.x) < columns) {
      float *to = a.partial_stats + (s.nth * a.s.rows * a.heads + (s.q0 + i) * a.heads + head) * 2;
      to[0] = top[lane];
      to[1] = total_l[lane];
    }
    __syncthreads();  // (the next columns' tiles take the sums' place)
  }
}

// The parts of a row of one head joined, by a block: its four waves take the parts in
// turn, half a wave each, four values a lane, so that many parts' sums are under way
// at once (and before their weights are known).
constexpr int kJoinParts = 8;  // at a time
template <class T> __global__ __launch_bounds__(256) void join_kernel(const Args a) {
  __shared__ float sums[kJoinParts][kMostHeadDim], stats[2];
  const int lane = lane_id(), slot = threadIdx.x / 32, d = (threadIdx.x & 31) * 4;
  const int64_t at = blockIdx.x, all = a.s.rows * a.heads, row = at / a.heads;
  // the row's sequence: of at most 64 by looking at all at once, of more the last that
  // begins at or before the row
  int parts = 0, lo = 0;
  if (a.s.count > 64)
    for (int hi = a.s.count; hi - lo > 1;) {
      const int mid = (lo + hi) / 2;
      if (a.s.offsets[mid] <= row) lo = mid;
      else hi = mid;
    }
  {
    const int b = a.s.count > 64 ? lo : lane;
    const Sequence s = sequence_at(a.s, b < a.s.count ? b : a.s.count - 1);
    const uint64_t found = ballot(b < a.s.count && row >= s.q0 && row < s.q0 + s.nq);
    if (found) {
      const int n = __shfl(s.nk, __builtin_ctzll(found), 64);
      parts = n > 0 ? (n - 1) / a.part_keys + 1 : 0;
    }
  }
  parts = uniform(parts);
  const auto stat = [&](int p, int i) { return a.partial_stats[(p * all + at) * 2 + i]; };
  constexpr int BATCH = 4;
  float v[4] = {}, m = -__builtin_inff();
  for (int p0 = 0; p0 < parts; p0 += kJoinParts * BATCH) {
    Chunk<float> part[BATCH];
    float pm[BATCH];
#pragma unroll
    for (int n = 0; n < BATCH; ++n) {
      const int p = p0 + n * kJoinParts + slot;
      const bool there = p < parts;
      part[n] = load_chunk(a.partial + ((there ? p : 0) * all + at) * a.d + d, there ? a.d - d : 0);
      pm[n] = there ? stat(p, 0) : -__builtin_inff();
    }
    float higher = m;
#pragma unroll
    for (int n = 0; n < BATCH; ++n) higher = __builtin_fmaxf(higher, pm[n]);
    const float by = m == higher ? 1.f : __builtin_amdgcn_exp2f(m - higher);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= by;
#pragma unroll
    for (int n = 0; n < BATCH; ++n) {
      const float w = pm[n] == higher ? 1.f : __builtin_amdgcn_exp2f(pm[n] - higher);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += w * part[n].v[i];
    }
    m = higher;
  }
  // the row's reference and sum, by the first wave
  if (threadIdx.x < 64) {
    float top = -__builtin_inff(), l = 0;
    for (int p = lane; p < parts; p += 64) {
      const float x = stat(p, 0), higher = __builtin_fmaxf(top, x);
      l = (top == higher ? l : l * __builtin_amdgcn_exp2f(top - higher)) +
          (x == higher ? stat(p, 1) : stat(p, 1) * __builtin_amdgcn_exp2f(x - higher));
      top = higher;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float om = __shfl_xor(top, o, 64), ol = __shfl_xor(l, o, 64), higher = __builtin_fmaxf(top, om);
      l = (top == higher ? l : l * __builtin_amdgcn_exp2f(top - higher)) +
          (om == higher ? ol : ol * __builtin_amdgcn_exp2f(om - higher));
      top = higher;
    }
    if (threadIdx.x == 0) {
      stats[0] = top;
      stats[1] = l;
    }
  }
  __syncthreads();
  const float top = stats[0], l = stats[1];
  const float w = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
  for (int i = 0; i < 4; ++i) sums[slot][d + i] = w * v[i];
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < a.d) {
    float o = 0;
#pragma unroll
    for (int n = 0; n < kJoinParts; ++n) o += sums[n][threadIdx.x];
    static_cast<T *>(a.o)[at * a.d + threadIdx.x] = from_float<T>(l == 0.f ? 0.f : o / l);
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
static int check(const spira_hip_attention_t &x) {
  constexpr int64_t most = (int64_t(1) << 31) - 256;  // (whole tiles are counted in 32 bits)
  SPIRA_HIP_REQUIRE(x.rows >= 0 && x.rows <= most && x.keys >= 0 && x.keys <= most, "attention: bad number of rows");
  SPIRA_HIP_REQUIRE(x.sequences > 0 && x.sequences <= 65536, "attention: needs 1 to 65536 sequences");
  SPIRA_HIP_REQUIRE(x.heads > 0 && x.kv_heads > 0 && x.heads <= 65536 && x.heads % x.kv_heads == 0,
                    "attention: the number of query heads must be a multiple of the key heads'");
  SPIRA_HIP_REQUIRE(x.head_dim > 0 && x.head_dim <= kMostHeadDim, "attention: needs heads of 1 to 128 values");
  SPIRA_HIP_REQUIRE(x.rows * (x.heads / x.kv_heads) <= most, "attention: too many queries");
  SPIRA_HIP_REQUIRE(x.scale > 0 && x.scale <= 1e38f, "attention: the scale must be positive and finite");
  SPIRA_HIP_REQUIRE(x.offsets && x.key_offsets, "attention: null offsets");
  SPIRA_HIP_REQUIRE((x.rows == 0 || x.queries) && (x.keys == 0 || (x.key && x.value)), "attention: null features");
  return kOk;
}

int arguments(const spira_hip_attention_t &x, Args &a, int size) {
  if (int rc = check(x)) return rc;
  a = Args{};
  a.s = {x.offsets, x.key_offsets, x.key_counts, x.sequences, x.rows, x.keys};
  a.heads = x.heads;
  a.kv_heads = x.kv_heads;
  a.group = x.heads / x.kv_heads;
  a.d = x.head_dim;
  a.causal = x.causal;
  a.scale = x.scale;
  a.scale2 = static_cast<float>(static_cast<double>(x.scale) * 1.4426950408889634);
  a.q = x.queries; a.q_row = x.query_row; a.q_head = x.query_head;
  a.k = x.key; a.k_row = x.key_row; a.k_head = x.key_head;
  a.v = x.value; a.v_row = x.value_row; a.v_head = x.value_head;
  const auto whole = [&](const void *p, int64_t row, int64_t head) { return dma_rows(p, row, head, x.head_dim, size); };
  a.dma = (whole(x.key, x.key_row, x.key_head) && whole(x.value, x.value_row, x.value_head) ? kKeysByDma : 0) |
          (whole(x.queries, x.query_row, x.query_head) ? kQueriesByDma : 0);
  return kOk;
}

// The form and, for few tokens, its parts.
struct Plan {
  bool tokens;
  int part_keys;
  int64_t parts;  // most of a sequence
};
static Plan plan(const spira_hip_attention_t &x, bool stats) {
  const int64_t group = x.heads / x.kv_heads, columns = div_up(x.rows * group, x.sequences);
  const Plan prompts{false, 0, 0}, direct{true, 1, 1};
  // Parts of the keys: where a sequence has few columns against many keys (or few rows in all,
  // whose join costs little however uneven the keys), and where whole columns' blocks leave
  // CUs idle and walk long caches.  100 queries of 8 heads on 2 against 100k keys 844 us by
  // whole columns, 121 in parts, 2048 keys 25.5 and 15.0; where there are blocks enough the
  // parts' sums cost more (2 sequences of 1024, themselves: 19.2 and 71.9; 65k voxels of 3
  // heads of 32 in windows of 64: 23 and 449, of 8: 127 and 601).  (A gradient's statistics
  // come from one block per column.)
  const bool few = few_columns(x), many_keys = x.keys / x.sequences >= 1024;
  const bool idle = (x.rows * group / 32 + x.sequences) * x.kv_heads < 256;
  const bool parted = columns <= 64 ? many_keys || x.rows * x.heads <= 8192 : many_keys && idle;
  if (stats || !parted) return few ? direct : prompts;
  const int64_t tiles = div_up(columns, 32);
  const int64_t size = round_up(std::max<int64_t>(div_up(x.keys * x.kv_heads * tiles, 2048), 256), 64);
  // (partial sums of at most 256 MB)
  int64_t part = size;
  while (x.rows * x.heads * div_up(x.keys, part) * (x.head_dim + 2) * 4 > (int64_t(1) << 28) && part < x.keys)
    part *= 2;
  // (no sequence has keys for more than four parts: a join would cost more)
  if (x.keys <= 4 * part) return few ? direct : prompts;
  return {true, static_cast<int>(part), div_up(x.keys, part)};
}

static size_t partial_bytes(const spira_hip_attention_t &x, const Plan &p) {
  return p.tokens && p.parts > 1 ? static_cast<size_t>(p.parts) * x.rows * x.heads * (x.head_dim + 2) * sizeof(float) : 0;
}

template <class T, int DP, bool DMA> static int launch_form(const Args &base, const Plan &p, hipStream_t stream) {
  Args a = base;
  if (!p.tokens) {
    const int64_t blocks = (a.s.rows * a.group / kColumns + a.s.count) * a.kv_heads;
    SPIRA_HIP_REQUIRE(launchable(blocks, 256), "attention: too many tiles for a launch");
    hipLaunchKernelGGL((prompt_kernel<T, DP, DMA>), dim3(blocks), dim3(256), 0, stream, a);
    SPIRA_HIP_LAUNCH_CHECK();
    return kOk;
  }
  a.part_keys = p.part_keys;
  const bool direct = p.parts <= 1;
  const int threads = 64 * (direct ? TokenShape<T, DP, true>::NW : TokenShape<T, DP, false>::NW);
  const int64_t blocks = ((direct ? a.s.rows * a.group / 32 : a.s.keys / p.part_keys) + a.s.count) * a.kv_heads;
  const uint32_t y = direct ? 1 : static_cast<uint32_t>(div_up(div_up(a.s.rows * a.group, a.s.count), 32));
  SPIRA_HIP_REQUIRE(launchable(blocks * y, threads), "attention: too many tiles for a launch");
  if (direct)
    hipLaunchKernelGGL((token_kernel<T, DP, true, DMA>), dim3(blocks, y), dim3(threads), 0, stream, a);
  else
    hipLaunchKernelGGL((token_kernel<T, DP, false, DMA>), dim3(blocks, y), dim3(threads), 0, stream, a);
  SPIRA_HIP_LAUNCH_CHECK();
  if (direct) return kOk;
  const int64_t joins = a.s.rows * a.heads;
  SPIRA_HIP_REQUIRE(launchable(joins, 256), "attention: too many rows for a launch");
  hipLaunchKernelGGL(join_kernel<T>, dim3(joins), dim3(256), 0, stream, a);
  SPIRA_HIP_LAUNCH_CHECK();
  return kOk;
}

template <class T, int DP> static int launch(const Args &a, const Plan &p, hipStream_t stream) {
  return a.dma & kKeysByDma ? launch_form<T, DP, true>(a, p, stream) : launch_form<T, DP, false>(a, p, stream);
}

}  // namespace attention

}  // namespace spira_hip

using namespace spira_hip;

extern "C" {

int spira_hip_attention_workspace(const spira_hip_attention_t *x, int gradient, size_t *bytes) {
  SPIRA_HIP_REQUIRE(x && bytes, "attention: null arguments");
  if (int rc = attention::check(*x)) return rc;
  *bytes = gradient ? attention::delta_bytes(*x) + attention::key_sums_bytes(*x) : attention::partial_bytes(*x, attention::plan(*x, false));
  return kOk;
}

int spira_hip_attention(const spira_hip_attention_t *x, void *out, float *stats, void *rest, void *workspace,
                        size_t workspace_bytes, hipStream_t stream) {
  SPIRA_HIP_REQUIRE(x, "attention: null arguments");
  attention::Args a;
  if (int rc = attention::arguments(*x, a, x->dtype == SPIRA_F32 ? 4 : 2)) return rc;
  if (x->rows == 0) return kOk;
  SPIRA_HIP_REQUIRE(out, "attention: null output");
  const attention::Plan p = attention::plan(*x, stats != nullptr);
  const size_t need = attention::partial_bytes(*x, p);
  SPIRA_HIP_REQUIRE(workspace_bytes >= need && (workspace || need == 0), "attention: workspace too small");
  a.o = out;
  a.stats = stats;
  // (in fp32 nothing that counts is left)
  a.rest = x->dtype == SPIRA_F32 ? nullptr : rest;
  a.partial = static_cast<float *>(workspace);
  a.partial_stats = a.partial ? a.partial + p.parts * x->rows * x->heads * x->head_dim : nullptr;
  return with_type(x->dtype, [&](auto t) -> int {
    return attention::with_width(x->head_dim, [&](auto W) -> int {
      return attention::launch<decltype(t), decltype(W)::value>(a, p, stream);
    });
  });
}

}  // extern "C"
