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

template <class T, int DP>
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
  const int least = visible(a, s, std::min(w0, total - 1) / a.group);
  const int most = w0 < total ? visible(a, s, std::min(w0 + 31, total - 1) / a.group) : 0;
  const int fewest = visible(a, s, c0 / a.group), end = dq ? visible(a, s, std::min(c0 + kColumns - 1, total - 1) / a.group) : 0;
  const int steps = (end + KT - 1) / KT, own = (most + KT - 1) / KT;
  const int64_t kstride = a.k_row * R::SIZE, vstride = a.v_row * R::SIZE;
  const char *keys = reinterpret_cast<const char *>(static_cast<const T *>(a.k) + s.k0 * a.k_row + kv * a.k_head);
  const char *values = reinterpret_cast<const char *>(static_cast<const T *>(a.v) + s.k0 * a.v_row + kv * a.v_head);
  const auto issue = [&](int t) {
    lds_char *to = (lds_char *)lds + (t & 1) * 2 * TILE;
    fetch_tile<T, DP, KT, 256>(keys + t * (KT * kstride), kstride, s.nk - t * KT, a.d, a.dma & 1, to, threadIdx.x);
    fetch_tile<T, DP, KT, 256>(values + t * (KT * vstride), vstride, s.nk - t * KT, a.d, a.dma & 1, to + TILE,
                               threadIdx.x);
  };
  if (steps > 0) issue(0);
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
  for (int t = 0; t < steps; ++t) {
    wait_loads_and_meet<0>();
    if (t + 1 < steps) issue(t + 1);
    // (the same for the whole block, which then stays together)
    const bool hides = a.causal && fewest < (t + 1) * KT;
    if (t >= own && !hides) continue;
    lds_char *kt = (lds_char *)lds + (t & 1) * 2 * TILE, *vt = kt + TILE;
    const bool whole = least >= (t + 1) * KT;
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) {
      floatx16 p{}, dp{};
#pragma unroll
      for (int st = 0; st < DP / 16; ++st) {
        mma(p, row_frag<T, DP>(kt, 32 * u, st), q[st]);
        mma(dp, row_frag<T, DP>(vt, 32 * u, st), g[st]);
      }
      const int mine = limit - t * KT - 32 * u;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float ds = weight(p[x], a.scale2, r) * (dp[x] - delta);
        p[x] = whole || 8 * (x / 4) + x % 4 < mine - 4 * h ? ds : 0.f;
      }
      Frag<T> ds[2] = {as_operand<T>(p, 0), as_operand<T>(p, 1)};
      lds_char *tile = kt + 32 * u * R::PITCH;
      bool found = false;
      if (hides) {
        __syncthreads();  // (every wave has the scores)
        found = __syncthreads_or(clear_not_finite<T, DP, 32, 256>(tile, threadIdx.x));
      }
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) mma(acc[n], col_frag<T, DP>(tile, 16 * st, n), ds[st]);
      if (found)
        add_not_finite<T, DP>(acc, keys + (t * KT + 32 * u) * kstride, kstride, std::min(s.nk - t * KT - 32 * u, 32), a.d,
                              [&](int x) { return x < mine; });
    }
  }
  if (dq) store_column<T, DP>(dq + at * a.d, a.d, there, acc, a.scale);
}

// ---------------------------------------------------------------------------
// keys: dk and dv; a wave's columns are 32 keys, the tiles hold queries
// ---------------------------------------------------------------------------
constexpr int kOwnKeys = 128;
template <class T> constexpr int kQueries = sizeof(T) == 2 ? 64 : 32;

template <class T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 2 && DP <= 64 ? 2 : 1) void keys_kernel(const Args a) {
  using R = Rows<T, DP>;
  constexpr int QT = kQueries<T>, TILE = QT * R::PITCH;
  __shared__ __align__(1024) char lds[4 * TILE];
  __shared__ __align__(256) float rows[2][3][64];  // statistics and delta of a tile's rows
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6)), lane = lane_id(), h = lane >> 5;
  T *dk = static_cast<T *>(a.dk), *dv = static_cast<T *>(a.dv);
  const int64_t width = static_cast<int64_t>(a.kv_heads) * a.d;
  if (dk) clear_uncovered(a.s.key_offsets, a.s.count, a.s.keys, dk, width, blockIdx.x, gridDim.x);
  if (dv) clear_uncovered(a.s.key_offsets, a.s.count, a.s.keys, dv, width, blockIdx.x, gridDim.x);
  const int kv = blockIdx.x % a.kv_heads;
  const Found f = find_piece(a.s.count, blockIdx.x / a.kv_heads,
                             [&](int b) { return static_cast<int>((room_of(a.s, b) + int64_t(kOwnKeys) - 1) / kOwnKeys); });
  if (f.sequence < 0) return;
  const Sequence s = sequence_at(a.s, f.sequence);
  // (the first tile first: the most queries see it)
  const int c0 = f.nth * kOwnKeys, w0 = c0 + wave * 32, key = w0 + (lane & 31);
  const bool there = key < s.nk;
  // the first query that sees this lane's key, the wave's first and last, the block's first
  const auto first_of = [&](int k) { return a.causal ? std::max(0, k - (s.nk - s.nq)) : 0; };
  const int first = first_of(key), earliest = first_of(w0), latest = first_of(w0 + 31), begin = first_of(c0) / QT;
  const int end = (s.nq + QT - 1) / QT, span = c0 < s.nk ? std::max(0, end - begin) : 0, steps = span * a.group;
  const int64_t qstride = a.q_row * R::SIZE, gstride = static_cast<int64_t>(a.heads) * a.d * R::SIZE;
  const auto queries_of_head = [&](int head) {
    return reinterpret_cast<const char *>(static_cast<const T *>(a.q) + head * a.q_head);
  };
  const auto gradients_of = [&](int head) {
    return reinterpret_cast<const char *>(static_cast<const T *>(a.dout) + static_cast<int64_t>(head) * a.d);
  };
  const auto issue = [&](int step, int g, int t) {
    lds_char *to = (lds_char *)lds + (step & 1) * 2 * TILE;
    const int head = kv * a.group + g;
    const int64_t q0 = s.q0 + t * QT;
    const int n = s.nq - t * QT;
    fetch_tile<T, DP, QT, 256>(queries_of_head(head) + q0 * qstride, qstride, n, a.d, a.dma & 4, to, threadIdx.x);
    fetch_tile<T, DP, QT, 256>(gradients_of(head) + q0 * gstride, gstride, n, a.d, a.dma & 4, to + TILE, threadIdx.x);
    // (rows past the last: zeros, of which every product is zero)
    const int64_t bytes = std::min(n, QT) * 4;
    const uint32_t at = lane < QT ? lane * 4 : kOutOfRange;
    const int64_t row = head * a.s.rows + q0;
    if (wave == 0) load_lds_word(buffer(a.stats + row, bytes), at, rows[step & 1][0]);
    if (wave == 1) load_lds_word(buffer(a.delta + row, bytes), at, rows[step & 1][1]);
    if (sizeof(T) == 4 && wave == 2)
      load_lds_word(buffer(a.stats + a.heads * a.s.rows + row, bytes), at, rows[step & 1][2]);
  };
  int g = 0, t = begin;  // of the step to be issued
  const auto advance = [&] {
    if (++t == end) {
      t = begin;
      ++g;
    }
  };
  if (steps > 0) issue(0, g, t);
  advance();
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
  int now = begin, at_head = 0;  // of the step at hand
  for (int step = 0; step < steps; ++step) {
    wait_loads_and_meet<0>();
    if (step + 1 < steps) {
      issue(step + 1, g, t);
      advance();
    }
    const int q0 = now * QT, of_head = at_head;
    if (++now == end) {
      now = begin;
      ++at_head;
    }
    // (the same for the whole block, which then stays together)
    const bool hides = a.causal && q0 < first_of(std::min(c0 + kOwnKeys, s.nk) - 1);
    if (w0 >= s.nk && !hides) continue;
    lds_char *tiles = (lds_char *)lds + (step & 1) * 2 * TILE;
#pragma unroll
    for (int u = 0; u < QT / 32; ++u) {
      const int r0 = q0 + 32 * u;
      if ((r0 + 32 <= earliest || r0 >= s.nq) && !hides) continue;  // (hidden from all keys, or past the last)
      lds_char *qt = tiles + 32 * u * R::PITCH, *gt = qt + TILE;
      floatx16 p{}, dp{};
#pragma unroll
      for (int st = 0; st < DP / 16; ++st) {
        mma(p, row_frag<T, DP>(qt, 0, st), k[st]);
        mma(dp, row_frag<T, DP>(gt, 0, st), v[st]);
      }
      const bool whole = r0 >= latest;
      const int mine = first - r0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float *at = &rows[step & 1][0][32 * u + 8 * x + 4 * h];
        const floatx4_t base = *reinterpret_cast<const floatx4_t *>(at);
        const floatx4_t delta = *reinterpret_cast<const floatx4_t *>(at + 64);
        floatx4_t by{};
        if constexpr (sizeof(T) == 4) by = *reinterpret_cast<const floatx4_t *>(at + 128);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float w = weight(p[4 * x + y], a.scale2, Stat<T>{base[y], by[y]});
          const bool seen = whole || 8 * x + y >= mine - 4 * h;
          dp[4 * x + y] = seen ? w * (dp[4 * x + y] - delta[y]) : 0.f;
          p[4 * x + y] = seen ? w : 0.f;
        }
      }
      const Frag<T> pf[2] = {as_operand<T>(p, 0), as_operand<T>(p, 1)}, ds[2] = {as_operand<T>(dp, 0), as_operand<T>(dp, 1)};
      bool found = false;
      if (hides) {
        __syncthreads();  // (every wave has the scores)
        const bool x = clear_not_finite<T, DP, 32, 256>(qt, threadIdx.x), y = clear_not_finite<T, DP, 32, 256>(gt, threadIdx.x);
        found = __syncthreads_or(x || y);
      }
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) mma(av[n], col_frag<T, DP>(gt, 16 * st, n), pf[st]);
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) mma(ak[n], col_frag<T, DP>(qt, 16 * st, n), ds[st]);
      if (found) {
        const int head = kv * a.group + of_head, n = std::min(s.nq - r0, 32);
        const auto sees = [&](int x) { return x >= mine; };
        add_not_finite<T, DP>(av, gradients_of(head) + (s.q0 + r0) * gstride, gstride, n, a.d, sees);
        add_not_finite<T, DP>(ak, queries_of_head(head) + (s.q0 + r0) * qstride, qstride, n, a.d, sees);
      }
    }
  }
  // (keys that are none, in the room behind the others, get zeros)
  if (!there) {
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) ak[n] = av[n] = floatx16{};
  }
  const int64_t to = ((s.k0 + key) * a.kv_heads + kv) * a.d;
  if (dk) store_column<T, DP>(dk + to, a.d, key < s.room, ak, a.scale);
  if (dv) store_column<T, DP>(dv + to, a.d, key < s.room, av, 1.f);
}

int arguments(const spira_hip_attention_t &x, Args &a, int size);

template <class T, int DP> static int launch(const Args &a, hipStream_t stream) {
  if (a.s.rows > 0) {
    const int64_t blocks = (a.s.rows * a.group / kColumns + a.s.count) * a.kv_heads;
    SPIRA_HIP_REQUIRE(launchable(blocks, 256), "attention: too many tiles for a launch");
    hipLaunchKernelGGL((queries_kernel<T, DP>), dim3(blocks), dim3(256), 0, stream, a);
    SPIRA_HIP_LAUNCH_CHECK();
  }
  if (a.s.keys > 0 && (a.dk || a.dv)) {
    const int64_t blocks = (a.s.keys / kOwnKeys + a.s.count) * a.kv_heads;
    SPIRA_HIP_REQUIRE(launchable(blocks, 256), "attention: too many tiles for a launch");
    hipLaunchKernelGGL((keys_kernel<T, DP>), dim3(blocks), dim3(256), 0, stream, a);
    SPIRA_HIP_LAUNCH_CHECK();
  }
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
  const size_t need = static_cast<size_t>(x->rows) * x->heads * sizeof(float);
  SPIRA_HIP_REQUIRE(workspace_bytes >= need && (workspace || need == 0), "attention: workspace too small");
  a.out = out;
  a.dout = dout;
  a.stats = const_cast<float *>(stats);
  a.delta = static_cast<float *>(workspace);
  a.dq = dqueries;
  a.dk = dkey;
  a.dv = dvalue;
  if (!attention::dma_rows(dout, static_cast<int64_t>(x->heads) * x->head_dim, x->head_dim, x->head_dim, size, 64))
    a.dma &= ~4;
  return with_type(x->dtype, [&](auto t) -> int {
    return attention::with_width(x->head_dim, [&](auto W) -> int {
      return attention::launch<decltype(t), decltype(W)::value>(a, stream);
    });
  });
}

}  // extern "C"
