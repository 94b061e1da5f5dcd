// Attention over packed sequences (gfx950), gradients:
//
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i . v_j - delta_i),  delta_i = do_i . o_i,
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
//
// p comes again from the scores and a row's statistics.  Two kernels, one that owns
// queries and one that owns keys, each sum in registers and in one order: nothing
// is added by atomics, at the price of two products that both make (14 D
// operations a visible pair instead of 10).  A key head's sums go over its group's
// query heads within the block that owns the keys.
#include "attention.hpp"

#include <algorithm>

namespace spira_hip {

namespace attention {

// a row's statistics, and p from a raw score
template <class T> struct Stat {
  float base, by;
};
template <class T> __device__ __forceinline__ float weight(float s, float scale2, const Stat<T> &r) {
  const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s, scale2, -r.base));
  // (in fp32 the logarithm of the sum would be rounded to as much as 1e-6 of p)
  return sizeof(T) == 2 ? e : e * r.by;
}

// ---------------------------------------------------------------------------
// queries: delta and dq; columns as in the forward pass
// ---------------------------------------------------------------------------
constexpr int kColumns = 128;
template <class T> constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;

__device__ __forceinline__ int visible(const Args &a, const Sequence &s, int i) {
  if (!a.causal) return s.nk;
  const int n = i + 1 + s.nk - s.nq;
  return n < 0 ? 0 : n < s.nk ? n : s.nk;
}

template <class T, int DP, bool DMA>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void queries_kernel(const Args a) {
  using R = Rows<T, DP>;
  constexpr int KT = kKeys<T>, TILE = KT * R::PITCH;
  __shared__ __align__(1024) char lds[4 * TILE];
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6)), lane = lane_id(), h = lane >> 5;
  T *dq = static_cast<T *>(a.dq);
  if (dq)
    clear_uncovered(a.s.offsets, a.s.count, a.s.rows, dq, static_cast<int64_t>(a.heads) * a.d, blockIdx.x, gridDim.x);
  const int kv = blockIdx.x % a.kv_heads;
  const Found f = find_piece(a.s.count, blockIdx.x / a.kv_heads,
                             [&](int b) { return (queries_of(a.s, b) * a.group + kColumns - 1) / kColumns; });
  if (f.sequence < 0) return;
  const Sequence s = sequence_at(a.s, f.sequence);
  const int total = s.nq * a.group, c0 = (f.of - 1 - f.nth) * kColumns, w0 = c0 + wave * 32;
  const int column = w0 + (lane & 31), j = column < total ? column : total - 1;
  const int i = j / a.group, head = kv * a.group + (j - i * a.group), limit = visible(a, s, i);
  const int fewest = visible(a, s, c0 / a.group), end = dq ? visible(a, s, std::min(c0 + kColumns - 1, total - 1) / a.group) : 0;
  const int steps = (end + KT - 1) / KT;
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
  const int64_t at = (s.q0 + i) * a.heads + head;
  Frag<T> q[DP / 16], g[DP / 16];
  const T *row = static_cast<const T *>(a.q) + (s.q0 + i) * a.q_row + head * a.q_head;
  const T *grow = static_cast<const T *>(a.dout) + at * a.d, *orow = static_cast<const T *>(a.out) + at * a.d;
  float delta = 0;
#pragma unroll
  for (int st = 0; st < DP / 16; ++st) {
    q[st] = load_frag(row, a.d, st);
    g[st] = load_frag(grow, a.d, st);
    const Frag<T> of = load_frag(orow, a.d, st);
    T x[8], y[8];
    __builtin_memcpy(x, &g[st], sizeof(x));
    __builtin_memcpy(y, &of, sizeof(y));
#pragma unroll
    for (int e = 0; e < 8; ++e) delta += to_float(x[e]) * to_float(y[e]);
  }
  delta += other_half(delta);
  const bool there = column < total;
  const int64_t stat = head * a.s.rows + s.q0 + i;
  if (there && lane < 32) a.delta[stat] = delta;
  Stat<T> r{a.stats[stat], 1.f};
  if constexpr (sizeof(T) == 4) r.by = a.stats[a.heads * a.s.rows + stat];
  floatx16 acc[DP / 32] = {};
  const Reader<T, DP> read;
  // ds of 32 keys (MASKED: of which this lane's column sees the first `seen`), in place of their scores
  const auto gradients = [&](auto MASKED, lds_char *kt, lds_char *vt, int seen, floatx16 &ds) {
    floatx16 p{}, dp{};
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) {
      mma(p, read.rows(kt, 0, st), q[st]);
      mma(dp, read.rows(vt, 0, st), g[st]);
    }
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const float w = weight(p[x], a.scale2, r) * (dp[x] - delta);
      ds[x] = !decltype(MASKED)::value || 8 * (x / 4) + x % 4 < seen - 4 * h ? w : 0.f;
    }
  };
  const auto accumulate = [&](lds_char *kt, const floatx16 &ds) {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const Frag<T> f = as_operand<T>(ds, st);
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) mma(acc[n], read.cols(kt, 16 * st, n), f);
    }
  };
  const int whole = std::min(fewest / KT, steps);  // tiles that every column sees whole
  int t = 0;
  const auto step = [&](auto STAGE) {
    constexpr int stage = decltype(STAGE)::value;
    wait_loads_and_meet<0>();
    if (t + 1 < steps) issue(t + 1, stage ^ 1);
    lds_char *kt = (lds_char *)lds + stage * 2 * TILE;
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) {
      floatx16 ds;
      gradients(std::false_type{}, kt + 32 * u * R::PITCH, kt + TILE + 32 * u * R::PITCH, 0, ds);
      accumulate(kt + 32 * u * R::PITCH, ds);
    }
  };
  while (t < whole) {
    step(std::integral_constant<int, 0>{});
    if (++t == whole) break;
    step(std::integral_constant<int, 1>{});
    ++t;
  }
  // the others; the block stays together
  for (; t < steps; ++t) {
    wait_loads_and_meet<0>();
    if (t + 1 < steps) issue(t + 1, (t + 1) & 1);
#pragma unroll 1
    for (int u = 0; u < KT / 32; ++u) {
      lds_char *kt = (lds_char *)lds + (t & 1) * 2 * TILE + 32 * u * R::PITCH;
      const int first = t * KT + 32 * u, seen = limit - first;
      floatx16 ds;
      gradients(std::true_type{}, kt, kt + TILE, seen, ds);
      bool found = false;
      if (a.causal) {
        __syncthreads();  // (every wave has the scores)
        found = __syncthreads_or(clear_not_finite<T, DP, 32, 256>(kt, threadIdx.x));
      }
      accumulate(kt, ds);
      if (found)
        add_not_finite<T, DP>(acc, keys + first * kstride, kstride, std::min(s.nk - first, 32), a.d,
                              [&](int x) { return x < seen; });
    }
  }
  if (dq) store_column<T, DP>(dq + at * a.d, a.d, there, acc, a.scale);
}

// ---------------------------------------------------------------------------
// keys: dk and dv; a wave's columns are 32 keys, the tiles hold queries
// ---------------------------------------------------------------------------
constexpr int kOwnKeys = 128;
template <class T> constexpr int kQueries = sizeof(T) == 2 ? 64 : 32;

// SPLIT: a block takes every `splits`th step of its keys', from blockIdx.y on, and writes its
// sums in fp32 to be joined.
template <class T, int DP, bool DMA, bool SPLIT>
__global__ __launch_bounds__(256, sizeof(T) == 2 && DP <= 64 ? 2 : 1) void keys_kernel(const Args a) {
  using R = Rows<T, DP>;
  constexpr int QT = kQueries<T>, TILE = QT * R::PITCH;
  __shared__ __align__(1024) char lds[4 * TILE];
  __shared__ __align__(256) float rows[2][3][64];  // statistics and delta of a tile's rows
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6)), lane = lane_id(), h = lane >> 5;
  T *dk = static_cast<T *>(a.dk), *dv = static_cast<T *>(a.dv);
  const int64_t width = static_cast<int64_t>(a.kv_heads) * a.d;
  if (!SPLIT && dk) clear_uncovered(a.s.key_offsets, a.s.count, a.s.keys, dk, width, blockIdx.x, gridDim.x);
  if (!SPLIT && dv) clear_uncovered(a.s.key_offsets, a.s.count, a.s.keys, dv, width, blockIdx.x, gridDim.x);
  const int kv = blockIdx.x % a.kv_heads;
  const Found f = find_piece(a.s.count, blockIdx.x / a.kv_heads,
                             [&](int b) { return static_cast<int>((room_of(a.s, b) + int64_t(kOwnKeys) - 1) / kOwnKeys); });
  if (f.sequence < 0) return;
  const Sequence s = sequence_at(a.s, f.sequence);
  // (the first tile first: the most queries see it)
  const int c0 = f.nth * kOwnKeys, w0 = c0 + wave * 32, key = w0 + (lane & 31);
  const bool there = key < s.nk;
  // the first query that sees a key
  const auto first_of = [&](int k) { return a.causal ? std::max(0, k - (s.nk - s.nq)) : 0; };
  const int first = first_of(key), begin = first_of(c0) / QT;
  const int latest = first_of(std::min(c0 + kOwnKeys, s.nk) - 1);  // (from here on all of the block's keys are seen)
  const int end = (s.nq + QT - 1) / QT, span = c0 < s.nk ? std::max(0, end - begin) : 0;
  const int splits = SPLIT ? static_cast<int>(gridDim.y) : 1, part = SPLIT ? static_cast<int>(blockIdx.y) : 0;
  const int64_t all = static_cast<int64_t>(span) * a.group;
  const int steps = static_cast<int>(all > part ? (all - part + splits - 1) / splits : 0);
  const int64_t qstride = a.q_row * R::SIZE, gstride = static_cast<int64_t>(a.heads) * a.d * R::SIZE;
  const auto queries_of_head = [&](int head) {
    return reinterpret_cast<const char *>(static_cast<const T *>(a.q) + head * a.q_head);
  };
  const auto gradients_of = [&](int head) {
    return reinterpret_cast<const char *>(static_cast<const T *>(a.dout) + static_cast<int64_t>(head) * a.d);
  };
  const Fetch<T, DP, QT, 256, DMA> fetch_queries(qstride, a.d, threadIdx.x), fetch_gradients(gstride, a.d, threadIdx.x);
  const auto issue = [&](int stage, int g, int t) {
    lds_char *to = (lds_char *)lds + stage * 2 * TILE;
    const int head = kv * a.group + g;
    const int64_t q0 = s.q0 + t * QT;
    const int n = s.nq - t * QT;
    fetch_queries(queries_of_head(head) + q0 * qstride, n, to);
    fetch_gradients(gradients_of(head) + q0 * gstride, n, to + TILE);
    // (rows past the last: zeros, of which every product is zero)
    const int64_t bytes = std::min(n, QT) * 4;
    const uint32_t at = lane < QT ? lane * 4 : kOutOfRange;
    const int64_t row = head * a.s.rows + q0;
    if (wave == 0) load_lds_word(buffer(a.stats + row, bytes), at, rows[stage][0]);
    if (wave == 1) load_lds_word(buffer(a.delta + row, bytes), at, rows[stage][1]);
    if (sizeof(T) == 4 && wave == 2)
      load_lds_word(buffer(a.stats + a.heads * a.s.rows + row, bytes), at, rows[stage][2]);
  };
  // the head and tile of a step, and of the one that follows
  struct Where {
    int g, t;
  };
  const auto advance = [&](Where &w) {
    w.t += splits;
    while (w.t >= end) {
      w.t -= span;
      ++w.g;
    }
  };
  Where next{0, begin + part};
  if (steps > 0) {
    while (next.t >= end) {
      next.t -= span;
      ++next.g;
    }
    issue(0, next.g, next.t);
  }
  Where now = next;  // of the step at hand
  if (steps > 1) advance(next);
  Frag<T> k[DP / 16], v[DP / 16];
  {
    const T *krow = there ? static_cast<const T *>(a.k) + (s.k0 + key) * a.k_row + kv * a.k_head : nullptr;
    const T *vrow = there ? static_cast<const T *>(a.v) + (s.k0 + key) * a.v_row + kv * a.v_head : nullptr;
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) {
      k[st] = load_frag(krow, a.d, st);
      v[st] = load_frag(vrow, a.d, st);
    }
  }
  floatx16 ak[DP / 32] = {}, av[DP / 32] = {};
  const Reader<T, DP> read;
  // p and ds of 32 queries from row `row` of the tile on; MASKED: this lane's key is seen from the `mine`th on
  const auto weights = [&](auto MASKED, int stage, int row, int mine, floatx16 &p, floatx16 &ds) {
    lds_char *qt = (lds_char *)lds + stage * 2 * TILE + row * R::PITCH, *gt = qt + TILE;
    p = floatx16{};
    ds = floatx16{};
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) {
      mma(p, read.rows(qt, 0, st), k[st]);
      mma(ds, read.rows(gt, 0, st), v[st]);
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float *at = &rows[stage][0][row + 8 * x + 4 * h];
      const floatx4_t base = *reinterpret_cast<const floatx4_t *>(at);
      const floatx4_t delta = *reinterpret_cast<const floatx4_t *>(at + 64);
      floatx4_t by{};
      if constexpr (sizeof(T) == 4) by = *reinterpret_cast<const floatx4_t *>(at + 128);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float w = weight(p[4 * x + y], a.scale2, Stat<T>{base[y], by[y]});
        const bool seen = !decltype(MASKED)::value || 8 * x + y >= mine - 4 * h;
        ds[4 * x + y] = seen ? w * (ds[4 * x + y] - delta[y]) : 0.f;
        p[4 * x + y] = seen ? w : 0.f;
      }
    }
  };
  const auto accumulate = [&](floatx16 (&acc)[DP / 32], lds_char *tile, const floatx16 &p) {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const Frag<T> f = as_operand<T>(p, st);
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) mma(acc[n], read.cols(tile, 16 * st, n), f);
    }
  };
  const auto step = [&](int index, auto STAGE) {
    constexpr int stage = decltype(STAGE)::value;
    wait_loads_and_meet<0>();
    if (index + 1 < steps) {
      issue(stage ^ 1, next.g, next.t);
    }
    const int q0 = now.t * QT, head = kv * a.group + now.g;
    now = next;
    if (index + 2 < steps) advance(next);
    lds_char *qt = (lds_char *)lds + stage * 2 * TILE, *gt = qt + TILE;
    if (q0 >= latest) {
      if (w0 < s.nk)
#pragma unroll
        for (int u = 0; u < QT / 32; ++u) {
          floatx16 p, ds;
          weights(std::false_type{}, stage, 32 * u, 0, p, ds);
          accumulate(av, gt + 32 * u * R::PITCH, p);
          accumulate(ak, qt + 32 * u * R::PITCH, ds);
        }
      return;
    }
    // (the block stays together)
#pragma unroll 1
    for (int u = 0; u < QT / 32; ++u) {
      const int mine = first - q0 - 32 * u;
      floatx16 p, ds;
      weights(std::true_type{}, stage, 32 * u, mine, p, ds);
      lds_char *qu = qt + 32 * u * R::PITCH, *gu = gt + 32 * u * R::PITCH;
      __syncthreads();  // (every wave has the scores)
      const bool x = clear_not_finite<T, DP, 32, 256>(qu, threadIdx.x), y = clear_not_finite<T, DP, 32, 256>(gu, threadIdx.x);
      const bool found = __syncthreads_or(x || y);
      accumulate(av, gu, p);
      accumulate(ak, qu, ds);
      if (found) {
        const int64_t r0 = s.q0 + q0 + 32 * u;
        const int n = std::min(s.nq - q0 - 32 * u, 32);
        const auto sees = [&](int r) { return r >= mine; };
        add_not_finite<T, DP>(av, gradients_of(head) + r0 * gstride, gstride, n, a.d, sees);
        add_not_finite<T, DP>(ak, queries_of_head(head) + r0 * qstride, qstride, n, a.d, sees);
      }
    }
  };
  for (int index = 0; index < steps;) {
    step(index, std::integral_constant<int, 0>{});
    if (++index == steps) break;
    step(index, std::integral_constant<int, 1>{});
    ++index;
  }
  // (keys that are none, in the room behind the others, get zeros)
  if (!there) {
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) ak[n] = av[n] = floatx16{};
  }
  const int64_t to = ((s.k0 + key) * a.kv_heads + kv) * a.d;
  if constexpr (SPLIT) {
    float *sums = a.partial + part * 2 * a.s.keys * width + to;
    store_column<float, DP>(sums, a.d, there, ak, a.scale);
    store_column<float, DP>(sums + a.s.keys * width, a.d, there, av, 1.f);
    return;
  }
  if (dk) store_column<T, DP>(dk + to, a.d, key < s.room, ak, a.scale);
  if (dv) store_column<T, DP>(dv + to, a.d, key < s.room, av, 1.f);
}

// dk (blockIdx.y 0) and dv from the splits' sums, in their order; zeros in rows that are no keys
template <class T> __global__ __launch_bounds__(256) void sums_kernel(const Args a, int splits) {
  const int64_t width = static_cast<int64_t>(a.kv_heads) * a.d, chunks = (width + kVec<T> - 1) / kVec<T>;
  const int64_t id = blockIdx.x * static_cast<int64_t>(256) + threadIdx.x, row = id / chunks, at = (id - row * chunks) * kVec<T>;
  T *to = static_cast<T *>(blockIdx.y == 0 ? a.dk : a.dv);
  if (!to || row >= a.s.keys) return;
  bool there = false;
  // (sequences are ascending: the last that begins at or before the row)
  int lo = 0, hi = a.s.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.s.key_offsets[mid] <= row) lo = mid;
    else hi = mid;
  }
  const int64_t first = clamp_row(a.s.key_offsets[lo], a.s.keys);
  there = row >= first && row < first + keys_of(a.s, lo);
  Chunk<T> sum{};
  if (there) {
    const float *from = a.partial + blockIdx.y * a.s.keys * width + row * width + at;
    for (int p = 0; p < splits; ++p, from += 2 * a.s.keys * width)
#pragma unroll
      for (int c = 0; c < kVec<T> / 4; ++c) {
        const Chunk<float> x = load_chunk(from + 4 * c, width - at - 4 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum.v[4 * c + i] += x.v[i];
      }
  }
  store_chunk(to + row * width + at, width - at, sum);
}

int arguments(const spira_hip_attention_t &x, Args &a, int size);

// Parts of the keys' steps.  A block of 128 keys has as many steps as its sequence has
// queries (times the group's heads, over 64): a long sequence's blocks run on alone when
// the others are done.  With parts for 8 blocks a CU, however long the sequences, at
// most 8 of them (their sums in fp32 are written and read again).
static int key_splits(const spira_hip_attention_t &x) {
  const int64_t blocks = (x.keys / kOwnKeys + x.sequences) * x.kv_heads;
  const int64_t steps = div_up(x.rows, 64) * (x.heads / x.kv_heads);
  const int64_t bytes = 2 * x.keys * x.kv_heads * x.head_dim * 4;
  int64_t splits = std::min<int64_t>({2048 / std::max<int64_t>(blocks, 1), steps, 8});
  if (bytes > 0) splits = std::min<int64_t>(splits, (int64_t(1) << 30) / bytes);
  return static_cast<int>(std::max<int64_t>(splits, 1));
}
static size_t delta_bytes(const spira_hip_attention_t &x) {
  return round_up(static_cast<int64_t>(x.rows) * x.heads * static_cast<int64_t>(sizeof(float)), 256);
}
static size_t sums_bytes(const spira_hip_attention_t &x) {
  const int splits = key_splits(x);
  return splits > 1 ? static_cast<size_t>(splits) * 2 * x.keys * x.kv_heads * x.head_dim * sizeof(float) : 0;
}
size_t gradient_bytes(const spira_hip_attention_t &x) { return delta_bytes(x) + sums_bytes(x); }

template <class T, int DP, bool DMA> static int launch_keys(const Args &a, int splits, hipStream_t stream) {
  const int64_t blocks = (a.s.keys / kOwnKeys + a.s.count) * a.kv_heads;
  SPIRA_HIP_REQUIRE(launchable(blocks * splits, 256), "attention: too many tiles for a launch");
  if (splits == 1) {
    hipLaunchKernelGGL((keys_kernel<T, DP, DMA, false>), dim3(blocks), dim3(256), 0, stream, a);
    SPIRA_HIP_LAUNCH_CHECK();
    return kOk;
  }
  hipLaunchKernelGGL((keys_kernel<T, DP, DMA, true>), dim3(blocks, splits), dim3(256), 0, stream, a);
  SPIRA_HIP_LAUNCH_CHECK();
  const int64_t sums = div_up(a.s.keys * div_up(static_cast<int64_t>(a.kv_heads) * a.d, kVec<T>), 256);
  SPIRA_HIP_REQUIRE(launchable(sums * 2, 256), "attention: too many rows for a launch");
  hipLaunchKernelGGL(sums_kernel<T>, dim3(sums, 2), dim3(256), 0, stream, a, splits);
  SPIRA_HIP_LAUNCH_CHECK();
  return kOk;
}

template <class T, int DP> static int launch(const Args &a, int splits, hipStream_t stream) {
  if (a.s.rows > 0) {
    const int64_t blocks = (a.s.rows * a.group / kColumns + a.s.count) * a.kv_heads;
    SPIRA_HIP_REQUIRE(launchable(blocks, 256), "attention: too many tiles for a launch");
    if (a.dma & kKeysByDma)
      hipLaunchKernelGGL((queries_kernel<T, DP, true>), dim3(blocks), dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((queries_kernel<T, DP, false>), dim3(blocks), dim3(256), 0, stream, a);
    SPIRA_HIP_LAUNCH_CHECK();
  }
  if (a.s.keys > 0 && (a.dk || a.dv))
    return a.dma & kQueriesByDma ? launch_keys<T, DP, true>(a, splits, stream) : launch_keys<T, DP, false>(a, splits, stream);
  return kOk;
}

}  // namespace attention

}  // namespace spira_hip

using namespace spira_hip;

extern "C" {

int spira_hip_attention_backward(const spira_hip_attention_t *x, const void *out, const float *stats, const void *dout,
                                 void *dqueries, void *dkey, void *dvalue, void *workspace, size_t workspace_bytes,
                                 hipStream_t stream) {
  SPIRA_HIP_REQUIRE(x, "attention: null arguments");
  const int size = x->dtype == SPIRA_F32 ? 4 : 2;
  attention::Args a;
  if (int rc = attention::arguments(*x, a, size)) return rc;
  SPIRA_HIP_REQUIRE(x->rows == 0 || (out && stats && dout), "attention: null outputs of the forward pass");
  const size_t need = attention::gradient_bytes(*x);
  const int splits = attention::key_splits(*x);
  SPIRA_HIP_REQUIRE(workspace_bytes >= need && (workspace || need == 0), "attention: workspace too small");
  a.out = out;
  a.dout = dout;
  a.stats = const_cast<float *>(stats);
  a.delta = static_cast<float *>(workspace);
  a.partial = splits > 1 ? a.delta + attention::delta_bytes(*x) / sizeof(float) : nullptr;
  a.dq = dqueries;
  a.dk = dkey;
  a.dv = dvalue;
  if (!attention::dma_rows(dout, static_cast<int64_t>(x->heads) * x->head_dim, x->head_dim, x->head_dim, size))
    a.dma &= ~attention::kQueriesByDma;
  return with_type(x->dtype, [&](auto t) -> int {
    return attention::with_width(x->head_dim, [&](auto W) -> int {
      return attention::launch<decltype(t), decltype(W)::value>(a, splits, stream);
    });
  });
}

}  // extern "C"
