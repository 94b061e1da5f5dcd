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
//
// 16384 uneven packed tokens, 16 heads of 64 on 4, causal, bf16: dq 191 us (three products
// a pair, 830 TFLOP/s), bound by the exponentials and the products in turn.
#include "attention.hpp"

#include <algorithm>

namespace spira_hip {

namespace attention {

// ---------------------------------------------------------------------------
// queries: delta and dq; columns as in the forward pass
// ---------------------------------------------------------------------------
// a lane's column on its way: its query, its output's gradient, and dq (this half's
// share, without the scale)
template <class T, int DP> struct QueryColumn {
  using R = Rows<T, DP>;
  Frag<T> q[DP / 16], g[DP / 16];
  float delta;
  Stat<T> stat;
  Lift<T> lift;  // of ds, and so of dq
  floatx16 acc[DP / 32];

  // query i of sequence s, of this head; `there`: delta is to be written
  __device__ __forceinline__ void load(const Args &a, const Sequence &s, int i, int head, bool there) {
    const int64_t at = (s.q0 + i) * a.heads + head;
    const T *row = static_cast<const T *>(a.q) + (s.q0 + i) * a.q_row + head * a.q_head;
    const T *grow = static_cast<const T *>(a.dout) + at * a.d, *orow = static_cast<const T *>(a.out) + at * a.d;
    // (the outputs with what their rounding left: without, delta's error doubles that of dq
    // and dk in sequences of some ten tokens, and adds a twentieth in long ones)
    const T *rest = a.rest ? static_cast<const T *>(a.rest) + at * a.d : nullptr;
    delta = 0;
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) {
      q[st] = load_frag(row, a.d, st);
      g[st] = load_frag(grow, a.d, st);
      const Frag<T> of = load_frag(orow, a.d, st), rf = load_frag(rest, a.d, st);
      T x[8], y[8], z[8];
      __builtin_memcpy(x, &g[st], sizeof(x));
      __builtin_memcpy(y, &of, sizeof(y));
      __builtin_memcpy(z, &rf, sizeof(z));
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += to_float(x[e]) * (to_float(y[e]) + to_float(z[e]));
    }
    delta += other_half(delta);
    const int64_t to = head * a.s.rows + s.q0 + i;
    if (there && lane_id() < 32) a.delta[to] = delta;
    stat = {a.stats[to], 1.f};
    if constexpr (sizeof(T) == 4) stat.by = a.stats[a.heads * a.s.rows + to];
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) acc[n] = floatx16{};
  }
  // ds, lifted, of 32 keys (MASKED: of which this lane's column sees the first `seen`)
  template <bool MASKED>
  __device__ __forceinline__ void gradients(const Args &a, const Reader<T, DP> &read, lds_char *kt, lds_char *vt, int seen,
                                            floatx16 &ds) const {
    floatx16 p{}, dp{};
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) mma(p, read.rows(kt, 0, st), q[st]);
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) mma(dp, read.rows(vt, 0, st), g[st]);
    const int mine = seen - 4 * (lane_id() >> 5);
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const float w = weight(p[x], a.scale2, stat) * (dp[x] - delta);
      ds[x] = !MASKED || 8 * (x / 4) + x % 4 < mine ? w : 0.f;
    }
  }
  // FINE (16 bits): with what the rounding of ds leaves.  Tiles on the mask's edge take it:
  // the rows that see few keys have their weights there, whose roundings do not average out.
  template <bool FINE> __device__ __forceinline__ void accumulate(const Reader<T, DP> &read, lds_char *kt, floatx16 &ds) {
    lift.fit(ds, acc);
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const Frag<T> f = as_operand<T>(ds, st);
      Frag<T> g;
      if constexpr (FINE && sizeof(T) == 2) g = rest_operand<T>(ds, st, f);
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) {
        const Frag<T> k = read.cols(kt, 16 * st, n);
        mma(acc[n], k, f);
        if constexpr (FINE && sizeof(T) == 2) mma(acc[n], k, g);
      }
    }
  }
};

template <class T, int DP, bool DMA>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void queries_kernel(const Args a) {
  using R = Rows<T, DP>;
  constexpr int KT = kKeys<T>, TILE = KT * R::PITCH;
  __shared__ __align__(1024) char lds[4 * TILE];
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6)), lane = lane_id();
  T *dq = static_cast<T *>(a.dq);
  if (dq)
    clear_uncovered(a.s.offsets, a.s.count, a.s.rows, dq, static_cast<int64_t>(a.heads) * a.d, blockIdx.x, gridDim.x);
  const int kv = blockIdx.x % a.kv_heads;
  const Found s = find_longest(a.s, blockIdx.x / a.kv_heads, Cut{false, a.group, kColumns});
  if (!s.there) return;
  const int total = s.nq * a.group, c0 = s.nth * kColumns, w0 = c0 + wave * 32;
  const int column = w0 + (lane & 31), j = column < total ? column : total - 1;
  const int i = j / a.group, head = kv * a.group + (j - i * a.group), limit = visible(a, s, i);
  // (without dq, delta alone)
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
  const bool there = column < total;
  QueryColumn<T, DP> c;
  c.load(a, s, i, head, there);
  const Reader<T, DP> read;
  const int whole = std::min(fewest / KT, steps);  // tiles that every column sees whole
  ring(whole, 0, [&](int t, auto STAGE) {
    constexpr int stage = decltype(STAGE)::value;
    wait_loads_and_meet<0>();
    if (t + 1 < steps) issue(t + 1, stage ^ 1);
    lds_char *kt = (lds_char *)lds + stage * 2 * TILE;
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) {
      floatx16 ds;
      c.template gradients<false>(a, read, kt + 32 * u * R::PITCH, kt + TILE + 32 * u * R::PITCH, 0, ds);
      c.template accumulate<false>(read, kt + 32 * u * R::PITCH, ds);
    }
  });
  // the others; the block stays together
  for (int t = whole; t < steps; ++t) {
    wait_loads_and_meet<0>();
    if (t + 1 < steps) issue(t + 1, (t + 1) & 1);
#pragma unroll 1
    for (int u = 0; u < KT / 32; ++u) {
      lds_char *kt = (lds_char *)lds + (t & 1) * 2 * TILE + 32 * u * R::PITCH;
      const int first = t * KT + 32 * u, seen = limit - first;
      floatx16 ds;
      c.template gradients<true>(a, read, kt, kt + TILE, seen, ds);
      bool found = false;
      if (a.causal) {
        __syncthreads();  // (every wave has the scores)
        found = __syncthreads_or(clear_not_finite<T, DP, 32, 256>(kt, threadIdx.x));
      }
      c.template accumulate<true>(read, kt, ds);
      if (found)
        add_not_finite<T, DP>(c.acc, keys + first * kstride, kstride, std::min(s.nk - first, 32), a.d,
                              [&](int x) { return x < seen; });
    }
  }
  if (dq) store_column<T, DP>(dq + ((s.q0 + i) * a.heads + head) * a.d, a.d, there, c.acc, a.scale * c.lift.lower());
}

// Few columns: a block's waves share 32 of them and take the keys' tiles in turn, each
// on its own, and add up their dq in order.
template <class T, int DP, bool DMA>
__global__ __launch_bounds__(64 * 2, 1) void few_queries_kernel(const Args a) {
  using R = Rows<T, DP>;
  constexpr int KT = 32, TILE = KT * R::PITCH, NW = 2, LOADS = 2 * KT * R::CPR / 64;
  static_assert(32 * kSumPitch<DP> * 4 <= 4 * TILE, "a wave's sums take its stages' place");
  __shared__ __align__(1024) char lds[NW][4 * TILE];
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6)), lane = lane_id();
  lds_char *own = (lds_char *)lds[wave];
  T *dq = static_cast<T *>(a.dq);
  if (dq)
    clear_uncovered(a.s.offsets, a.s.count, a.s.rows, dq, static_cast<int64_t>(a.heads) * a.d, blockIdx.x, gridDim.x);
  const int kv = blockIdx.x % a.kv_heads;
  const Found s = find_longest(a.s, blockIdx.x / a.kv_heads, Cut{false, a.group, 32});
  if (!s.there) return;
  const int total = s.nq * a.group, w0 = s.nth * 32, column = w0 + (lane & 31), j = column < total ? column : total - 1;
  const int i = j / a.group, head = kv * a.group + (j - i * a.group), limit = visible(a, s, i);
  const int fewest = visible(a, s, w0 / a.group), end = dq ? visible(a, s, std::min(w0 + 31, total - 1) / a.group) : 0;
  const int steps = (end + KT - 1) / KT;
  const int64_t kstride = a.k_row * R::SIZE, vstride = a.v_row * R::SIZE;
  const char *keys = reinterpret_cast<const char *>(static_cast<const T *>(a.k) + s.k0 * a.k_row + kv * a.k_head);
  const char *values = reinterpret_cast<const char *>(static_cast<const T *>(a.v) + s.k0 * a.v_row + kv * a.v_head);
  const Fetch<T, DP, KT, 64, DMA> fetch_keys(kstride, a.d, lane), fetch_values(vstride, a.d, lane);
  const auto issue = [&](int t, int stage) {
    lds_char *to = own + stage * 2 * TILE;
    const int64_t n = t < steps ? s.nk - t * KT : 0;
    fetch_keys(keys + t * (KT * kstride), n, to);
    fetch_values(values + t * (KT * vstride), n, to + TILE);
  };
  issue(wave, 0);
  QueryColumn<T, DP> c;
  c.load(a, s, i, head, column < total && wave == 0);
  const Reader<T, DP> read;
  for (int t = wave, stage = 0; t < steps; t += NW, stage ^= 1) {
    issue(t + NW, stage ^ 1);
    // until this tile's loads have landed (the next one's are on their way)
    __builtin_amdgcn_s_waitcnt((LOADS & 15) | (7 << 4) | ((LOADS >> 4) << 14));
    asm volatile("" ::: "memory");
    lds_char *kt = own + stage * 2 * TILE;
    floatx16 ds;
    if (fewest >= (t + 1) * KT) {
      c.template gradients<false>(a, read, kt, kt + TILE, 0, ds);
      c.template accumulate<false>(read, kt, ds);
      continue;
    }
    const int seen = limit - t * KT;
    c.template gradients<true>(a, read, kt, kt + TILE, seen, ds);
    const bool found = a.causal && ballot(clear_not_finite<T, DP, KT, 64>(kt, lane)) != 0;
    c.template accumulate<true>(read, kt, ds);
    if (found)
      add_not_finite<T, DP>(c.acc, keys + t * (KT * kstride), kstride, std::min(s.nk - t * KT, KT), a.d,
                            [&](int x) { return x < seen; });
  }
  wait_loads();
  asm volatile("" ::: "memory");
  if (!dq) return;
  // (the waves' lifts are their own)
  if constexpr (std::is_same_v<T, _Float16>) {
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) c.acc[n][r] *= c.lift.lower();
  }
  put_sums<DP>(reinterpret_cast<float *>(lds[wave]), c.acc);
  __syncthreads();
  const int columns = std::min(32, total - w0);
  for (int k = threadIdx.x; k < columns * a.d; k += 64 * NW) {
    const int col = k / a.d, d = k - col * a.d, at_q = (w0 + col) / a.group, at_h = kv * a.group + (w0 + col - at_q * a.group);
    float v = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += reinterpret_cast<const float *>(lds[w])[col * kSumPitch<DP> + d];
    dq[((s.q0 + at_q) * a.heads + at_h) * a.d + d] = from_float<T>(v * a.scale);
  }
}

template <class T, int DP> static int launch(const Args &a, bool few, hipStream_t stream) {
  if (a.s.rows > 0) {
    int64_t blocks = (a.s.rows * a.group / kColumns + a.s.count) * a.kv_heads;
    if (few) blocks = (a.s.rows * a.group / 32 + a.s.count) * a.kv_heads;
    SPIRA_HIP_REQUIRE(launchable(blocks, 256), "attention: too many tiles for a launch");
    const auto kernel = few ? (a.dma & kKeysByDma ? few_queries_kernel<T, DP, true> : few_queries_kernel<T, DP, false>)
                            : (a.dma & kKeysByDma ? queries_kernel<T, DP, true> : queries_kernel<T, DP, false>);
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(few ? 128 : 256), 0, stream, a);
    SPIRA_HIP_LAUNCH_CHECK();
  }
  return kOk;
}

}  // namespace attention

}  // namespace spira_hip

using namespace spira_hip;

extern "C" {

int spira_hip_attention_backward(const spira_hip_attention_t *x, const void *out, const float *stats, const void *rest,
                                 const void *dout, void *dqueries, void *dkey, void *dvalue, void *workspace,
                                 size_t workspace_bytes, hipStream_t stream) {
  SPIRA_HIP_REQUIRE(x, "attention: null arguments");
  const int size = x->dtype == SPIRA_F32 ? 4 : 2;
  attention::Args a;
  if (int rc = attention::arguments(*x, a, size)) return rc;
  SPIRA_HIP_REQUIRE(x->rows == 0 || (out && stats && dout), "attention: null outputs of the forward pass");
  const size_t need = attention::delta_bytes(*x) + attention::key_sums_bytes(*x);
  SPIRA_HIP_REQUIRE(workspace_bytes >= need && (workspace || need == 0), "attention: workspace too small");
  a.out = out;
  a.dout = dout;
  a.stats = const_cast<float *>(stats);
  a.rest = x->dtype == SPIRA_F32 ? nullptr : const_cast<void *>(rest);
  a.delta = static_cast<float *>(workspace);
  a.partial = a.delta ? a.delta + attention::delta_bytes(*x) / sizeof(float) : nullptr;
  a.dq = dqueries;
  a.dk = dkey;
  a.dv = dvalue;
  if (!attention::dma_rows(dout, static_cast<int64_t>(x->heads) * x->head_dim, x->head_dim, x->head_dim, size))
    a.dma &= ~attention::kQueriesByDma;
  const int rc = with_type(x->dtype, [&](auto t) -> int {
    return attention::with_width(x->head_dim, [&](auto W) -> int {
      return attention::launch<decltype(t), decltype(W)::value>(a, attention::few_columns(*x), stream);
    });
  });
  // (delta is the first launch's)
  return rc ? rc : attention::key_gradients(*x, a, stream);
}

}  // extern "C"
