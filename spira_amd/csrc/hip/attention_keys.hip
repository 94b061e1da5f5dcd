// Attention over packed sequences (gfx950), gradients of the keys and values:
//
//   dv_j = sum_i p_ij do_i,   dk_j = scale sum_i ds_ij q_i
//
// (attention_backward.hip has the formulas of ds).  A block owns 128 keys, a wave 32 of
// them as its columns, and walks its group's query heads and their queries in tiles;
// p and ds go from the scores' registers to the products as they are.
//
// 16384 uneven packed tokens, 16 heads of 64 on 4, causal, bf16: 303 us (four products a
// pair, 700 TFLOP/s) and 15 to join two parts.  A block's steps in one part 797; three parts,
// each in a launch order of its own behind the one before, 382.
#include "attention.hpp"

#include <algorithm>

namespace spira_hip {

namespace attention {

// ---------------------------------------------------------------------------
// keys: dk and dv; a wave's columns are 32 keys, the tiles hold queries
// ---------------------------------------------------------------------------
constexpr int kOwnKeys = 128;
template <class T> constexpr int kQueries = sizeof(T) == 2 ? 64 : 32;

// SPLIT: a block takes every `splits`th step of its keys', the parts of a tile's keys behind
// each other in the launch, and writes its sums in fp32 to be joined.
template <class T, int DP, bool DMA, bool SPLIT>
__global__ __launch_bounds__(256, sizeof(T) == 2 && DP <= 64 ? 2 : 1) void keys_kernel(const Args a, int parts) {
  using R = Rows<T, DP>;
  constexpr int QT = kQueries<T>, TILE = QT * R::PITCH;
  __shared__ __align__(1024) char lds[4 * TILE];
  __shared__ __align__(256) float rows[2][4][64];  // statistics, delta and the sum's inverse of a tile's rows
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6)), lane = lane_id(), h = lane >> 5;
  T *dk = static_cast<T *>(a.dk), *dv = static_cast<T *>(a.dv);
  const int64_t width = static_cast<int64_t>(a.kv_heads) * a.d;
  if (!SPLIT && dk) clear_uncovered(a.s.key_offsets, a.s.count, a.s.keys, dk, width, blockIdx.x, gridDim.x);
  if (!SPLIT && dv) clear_uncovered(a.s.key_offsets, a.s.count, a.s.keys, dv, width, blockIdx.x, gridDim.x);
  const int kv = blockIdx.x % a.kv_heads;
  const int splits = SPLIT ? parts : 1;
  const int64_t piece = blockIdx.x / a.kv_heads;
  const int part = SPLIT ? static_cast<int>(piece % splits) : 0;
  const Found s = find_longest(a.s, piece / splits, Cut{true, 1, kOwnKeys});
  if (!s.there) return;
  const int c0 = (s.of - 1 - s.nth) * kOwnKeys, w0 = c0 + wave * 32, key = w0 + (lane & 31);
  const bool there = key < s.nk;
  // the first query that sees a key
  const auto first_of = [&](int k) { return a.causal ? std::max(0, k - (s.nk - s.nq)) : 0; };
  const int first = first_of(key), begin = first_of(c0) / QT;
  const int latest = first_of(std::min(c0 + kOwnKeys, s.nk) - 1);  // (from here on all of the block's keys are seen)
  const int end = c0 < s.nk ? (s.nq + QT - 1) / QT : 0, middle = std::max(begin, std::min((latest + QT - 1) / QT, end));
  // The tiles of all heads that some key hides from (or the block's last), then those of
  // all heads that see every key: `splits`th by splits`th of them.
  const auto mine_of = [&](int64_t n) { return static_cast<int>(n > part ? (n - part + splits - 1) / splits : 0); };
  const int64_t masked = static_cast<int64_t>(middle - begin) * a.group;
  const int hidden = mine_of(masked), steps = mine_of(masked + static_cast<int64_t>(std::max(0, end - middle)) * a.group);
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
    // a row of them for each wave (rows past the last: zeros, of which every product is zero)
    const int64_t bytes = n > 0 ? std::min(n, QT) * 4 : 0;
    const uint32_t at = lane < QT ? lane * 4 : kOutOfRange;
    const float *from = (wave == 1 ? a.delta : a.stats + (sizeof(T) == 4 && wave == 2 ? a.heads * a.s.rows : 0)) + head * a.s.rows + q0;
    load_lds_word(buffer(from, wave < (sizeof(T) == 4 ? 3 : 2) ? bytes : 0), at, rows[stage][wave]);
  };
  // a step's head and tile, and the step behind it
  struct Where {
    int g, t, whole;
  };
  const auto advance = [&](Where &w, int by) {
    w.t += by;
    while (w.g < a.group || !w.whole) {
      const int lo = w.whole ? middle : begin, hi = w.whole ? end : middle;
      if (w.t < hi) return;
      w.t += lo - hi;
      if (++w.g == a.group && !w.whole) {
        w.t += middle - lo;
        w.g = 0;
        w.whole = 1;
      }
    }
  };
  Where next{0, begin, 0};  // to be fetched
  if (steps > 0) advance(next, part);
  Where now = next;  // at hand
  if (steps > 0) {
    issue(0, next.g, next.t);
    advance(next, splits);
  }
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
  Lift<T> lift;  // of ds, and so of ak
  const Reader<T, DP> read;
  // p and ds of 32 queries from row `row` of the tile on; MASKED: this lane's key is seen from the `mine`th on
  const auto weights = [&](auto MASKED, int stage, int row, int mine, floatx16 &p, floatx16 &ds) {
    lds_char *qt = (lds_char *)lds + stage * 2 * TILE + row * R::PITCH, *gt = qt + TILE;
    p = floatx16{};
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) mma(p, read.rows(qt, 0, st), k[st]);
    ds = floatx16{};
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) mma(ds, read.rows(gt, 0, st), v[st]);
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
        // (w is lifted, and ds with it)
        ds[4 * x + y] = seen ? w * (ds[4 * x + y] - delta[y]) : 0.f;
        p[4 * x + y] = seen ? w : 0.f;
      }
    }
  };
  // FINE (16 bits): with what the rounding leaves, as for dq
  const auto accumulate = [&](auto FINE, floatx16 (&acc)[DP / 32], lds_char *tile, const floatx16 &p) {
    constexpr bool fine = decltype(FINE)::value && sizeof(T) == 2;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const Frag<T> f = as_operand<T>(p, st);
      Frag<T> g;
      if constexpr (fine) g = rest_operand<T>(p, st, f);
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) {
        const Frag<T> x = read.cols(tile, 16 * st, n);
        mma(acc[n], x, f);
        if constexpr (fine) mma(acc[n], x, g);
      }
    }
  };
  for (int index = 0; index < hidden; ++index) {
    wait_loads_and_meet<0>();
    if (index + 1 < steps) {
      issue((index + 1) & 1, next.g, next.t);
      advance(next, splits);
    }
    const int stage = index & 1, q0 = now.t * QT, head = kv * a.group + now.g;
    advance(now, splits);
#pragma unroll 1
    for (int u = 0; u < QT / 32; ++u) {
      const int mine = first - q0 - 32 * u;
      floatx16 p, ds;
      weights(std::true_type{}, stage, 32 * u, mine, p, ds);
      lds_char *qu = (lds_char *)lds + stage * 2 * TILE + 32 * u * R::PITCH, *gu = qu + TILE;
      __syncthreads();  // (every wave has the scores)
      const bool x = clear_not_finite<T, DP, 32, 256>(qu, threadIdx.x), y = clear_not_finite<T, DP, 32, 256>(gu, threadIdx.x);
      const bool found = __syncthreads_or(x || y);
      lift.fit(ds, ak);
      accumulate(std::true_type{}, av, gu, p);
      accumulate(std::true_type{}, ak, qu, ds);
      if (found) {
        const int64_t r0 = s.q0 + q0 + 32 * u;
        const int n = std::min(s.nq - q0 - 32 * u, 32);
        const auto sees = [&](int r) { return r >= mine; };
        add_not_finite<T, DP>(av, gradients_of(head) + r0 * gstride, gstride, n, a.d, sees);
        add_not_finite<T, DP>(ak, queries_of_head(head) + r0 * qstride, qstride, n, a.d, sees);
      }
    }
  }
  ring(steps - hidden, hidden & 1, [&](int index, auto STAGE) {
    constexpr int stage = decltype(STAGE)::value;
    wait_loads_and_meet<0>();
    if (hidden + index + 1 < steps) {
      issue(stage ^ 1, next.g, next.t);
      advance(next, splits);
    }
    if (w0 >= s.nk) return;
    lds_char *qt = (lds_char *)lds + stage * 2 * TILE, *gt = qt + TILE;
#pragma unroll
    for (int u = 0; u < QT / 32; ++u) {
      floatx16 p, ds;
      weights(std::false_type{}, stage, 32 * u, 0, p, ds);
      lift.fit(ds, ak);
      accumulate(std::false_type{}, av, gt + 32 * u * R::PITCH, p);
      accumulate(std::false_type{}, ak, qt + 32 * u * R::PITCH, ds);
    }
  });
  // (keys that are none, in the room behind the others, get zeros)
  if (!there) {
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) ak[n] = av[n] = floatx16{};
  }
  const float scale = a.scale * lift.lower();
  const int64_t to = ((s.k0 + key) * a.kv_heads + kv) * a.d;
  if constexpr (SPLIT) {
    float *sums = a.partial + part * 2 * a.s.keys * width + to;
    store_column<float, DP>(sums, a.d, there, ak, scale);
    store_column<float, DP>(sums + a.s.keys * width, a.d, there, av, kLower<T>);
    return;
  }
  if (dk) store_column<T, DP>(dk + to, a.d, key < s.room, ak, scale);
  if (dv) store_column<T, DP>(dv + to, a.d, key < s.room, av, kLower<T>);
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
  there = row >= first && row < first + sequence_at(a.s, lo).nk;
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

// Parts of the keys' steps.  A block of 128 keys has as many steps as its sequence has
// queries (times the group's heads, over 64): a long sequence's blocks run on alone when
// the others are done.  With parts for 5 blocks a CU, however long the sequences, at
// most 8 of them (their sums in fp32 are written and read again).
int key_splits(const spira_hip_attention_t &x) {
  const int64_t blocks = (x.keys / kOwnKeys + x.sequences) * x.kv_heads;
  const int64_t steps = div_up(x.rows, 64) * (x.heads / x.kv_heads);
  const int64_t bytes = 2 * x.keys * x.kv_heads * x.head_dim * 4;
  int64_t splits = std::min<int64_t>({1280 / std::max<int64_t>(blocks, 1), steps, 8});
  if (bytes > 0) splits = std::min<int64_t>(splits, (int64_t(1) << 30) / bytes);
  return static_cast<int>(std::max<int64_t>(splits, 1));
}
size_t key_sums_bytes(const spira_hip_attention_t &x) {
  const int splits = key_splits(x);
  return splits > 1 ? static_cast<size_t>(splits) * 2 * x.keys * x.kv_heads * x.head_dim * sizeof(float) : 0;
}
template <class T, int DP, bool DMA> static int launch_keys(const Args &a, int splits, hipStream_t stream) {
  const int64_t blocks = (a.s.keys / kOwnKeys + a.s.count) * a.kv_heads;
  SPIRA_HIP_REQUIRE(launchable(blocks * splits, 256), "attention: too many tiles for a launch");
  if (splits == 1) {
    hipLaunchKernelGGL((keys_kernel<T, DP, DMA, false>), dim3(blocks), dim3(256), 0, stream, a, 1);
    SPIRA_HIP_LAUNCH_CHECK();
    return kOk;
  }
  hipLaunchKernelGGL((keys_kernel<T, DP, DMA, true>), dim3(blocks * splits), dim3(256), 0, stream, a, splits);
  SPIRA_HIP_LAUNCH_CHECK();
  const int64_t sums = div_up(a.s.keys * div_up(static_cast<int64_t>(a.kv_heads) * a.d, kVec<T>), 256);
  SPIRA_HIP_REQUIRE(launchable(sums * 2, 256), "attention: too many rows for a launch");
  hipLaunchKernelGGL(sums_kernel<T>, dim3(sums, 2), dim3(256), 0, stream, a, splits);
  SPIRA_HIP_LAUNCH_CHECK();
  return kOk;
}

int key_gradients(const spira_hip_attention_t &x, const Args &a, hipStream_t stream) {
  if (a.s.keys == 0 || (!a.dk && !a.dv)) return kOk;
  const int splits = key_splits(x);
  return with_type(x.dtype, [&](auto t) -> int {
    using T = decltype(t);
    return with_width(x.head_dim, [&](auto W) -> int {
      constexpr int w = decltype(W)::value;
      return a.dma & kQueriesByDma ? launch_keys<T, w, true>(a, splits, stream) : launch_keys<T, w, false>(a, splits, stream);
    });
  });
}

}  // namespace attention

}  // namespace spira_hip
