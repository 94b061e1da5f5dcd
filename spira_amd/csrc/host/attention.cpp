// Attention over rows of features and the norms of its heads in `_C`, forward and
// gradients (no counterparts in the reference).  Inputs may be views of one
// projection: rows and heads at any stride are read as they lie.
#include "rows.h"

namespace spira_host {

// t as the kernels read it: [rows, heads, dim], the values of a head consecutive
static Tensor strided(const Tensor &t) {
  return t.dim() == 3 && (t.size(2) == 1 || t.stride(2) == 1) ? t : t.contiguous();
}

static void require_heads(const Tensor &t, const char *name, const Tensor &x) {
  SPIRA_CHECK_ARG(t.is_cuda(), name, " must be a GPU tensor");
  SPIRA_CHECK_ARG(t.device() == x.device(), name, " must be on ", x.device());
  SPIRA_CHECK_ARG(t.scalar_type() == x.scalar_type(), name, " must be ", x.scalar_type(), ", got ", t.scalar_type());
  SPIRA_CHECK_ARG(t.dim() == 3, name, " must have the shape [rows, heads, values], got ", t.sizes());
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
static spira_hip_attention_t attention_arguments(const Tensor &q, const Tensor &k, const Tensor &v,
                                                 const Tensor &offsets, const Tensor &key_offsets,
                                                 const OptTensor &key_counts, bool causal, double scale) {
  require_heads(q, "queries", q);
  require_heads(k, "keys", q);
  require_heads(v, "values", q);
  const int dtype = row_dtype(q);
  SPIRA_CHECK_ARG(q.size(1) > 0 && k.size(1) > 0 && q.size(1) % k.size(1) == 0,
                  "attention: the number of query heads must be a multiple of the key heads', got ", q.size(1), " and ",
                  k.size(1));
  SPIRA_CHECK_ARG(q.size(2) > 0 && q.size(2) <= 128, "attention: needs heads of 1 to 128 values, got ", q.size(2));
  SPIRA_CHECK_ARG(k.size(2) == q.size(2), "keys must have heads of ", q.size(2), " values, got ", k.sizes());
  SPIRA_CHECK_ARG(v.sizes() == k.sizes(), "values must have the keys' shape ", k.sizes(), ", got ", v.sizes());
  SPIRA_CHECK_ARG(offsets.dim() == 1 && offsets.size(0) >= 2, "offsets must have the shape [sequences + 1], got ",
                  offsets.sizes());
  require(offsets, "offsets", q, torch::kInt, {-1});
  require(key_offsets, "key_offsets", q, torch::kInt, {offsets.size(0)});
  require(key_counts, "key_counts", q, torch::kInt, {offsets.size(0) - 1});
  SPIRA_CHECK_ARG(scale > 1e-38 && scale <= 1e38, "attention: the scale must be positive and finite, got ", scale);
  spira_hip_attention_t x{};
  x.rows = q.size(0);
  x.keys = k.size(0);
  SPIRA_CHECK_ARG(offsets.size(0) - 1 <= 65536, "attention: needs 1 to 65536 sequences, got ", offsets.size(0) - 1);
  SPIRA_CHECK_ARG(q.size(1) <= 65536, "attention: needs 1 to 65536 heads, got ", q.size(1));
  x.sequences = static_cast<int>(offsets.size(0) - 1);
  x.heads = static_cast<int>(q.size(1));
  x.kv_heads = static_cast<int>(k.size(1));
  x.head_dim = static_cast<int>(q.size(2));
  x.dtype = dtype;
  x.causal = causal;
  x.scale = static_cast<float>(scale);
  x.offsets = offsets.data_ptr<int32_t>();
  x.key_offsets = key_offsets.data_ptr<int32_t>();
  x.key_counts = static_cast<const int32_t *>(ptr(key_counts));
  x.queries = q.data_ptr();
  x.key = k.data_ptr();
  x.value = v.data_ptr();
  x.query_row = q.stride(0);
  x.query_head = q.stride(1);
  x.key_row = k.stride(0);
  x.key_head = k.stride(1);
  x.value_row = v.stride(0);
  x.value_head = v.stride(1);
  return x;
}

// (output, statistics of its rows and what rounding left of it, or None unless `train`)
static std::tuple<Tensor, OptTensor, OptTensor> attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &offsets,
                                               const Tensor &key_offsets, const OptTensor &key_counts, bool causal,
                                               double scale, bool train) {
  const spira_hip_attention_t x = attention_arguments(q, k, v, offsets, key_offsets, key_counts, causal, scale);
  const c10::DeviceGuard guard(q.device());
  Tensor out = like(q, q.sizes());
  OptTensor stats, rest;
  size_t bytes = 0;
  const bool full = q.scalar_type() == torch::kFloat;
  if (train) stats = floats(q, {full ? 2 : 1, q.size(1), q.size(0)});
  if (train && !full) rest = like(q, q.sizes());
  if (!train) check_rc(spira_hip_attention_workspace(&x, 0, &bytes), "attention");
  Tensor ws = bytes > 0 ? workspace(bytes, q.device()) : Tensor();
  check_rc(spira_hip_attention(&x, out.data_ptr(), stats ? stats->data_ptr<float>() : nullptr,
                               rest ? rest->data_ptr() : nullptr, bytes > 0 ? ws.data_ptr() : nullptr, bytes, current_stream()),
           "attention");
  return {out, stats, rest};
}

// (dq, dk, dv), each None unless it is in `need`
static std::array<OptTensor, 3> attention_backward(const Tensor &q, const Tensor &k, const Tensor &v,
                                                   const Tensor &offsets, const Tensor &key_offsets,
                                                   const OptTensor &key_counts, bool causal, double scale,
                                                   const Tensor &out, const Tensor &stats, const OptTensor &rest, const Tensor &dout,
                                                   int64_t need) {
  const spira_hip_attention_t x = attention_arguments(q, k, v, offsets, key_offsets, key_counts, causal, scale);
  require(dout, "gradient", q, q.scalar_type(), {q.size(0), q.size(1), q.size(2)});
  require(out, "output", q, q.scalar_type(), {q.size(0), q.size(1), q.size(2)});
  require(stats, "statistics", q, torch::kFloat, {q.scalar_type() == torch::kFloat ? 2 : 1, q.size(1), q.size(0)});
  require(rest, "rest", q, q.scalar_type(), {q.size(0), q.size(1), q.size(2)});
  const c10::DeviceGuard guard(q.device());
  std::array<OptTensor, 3> d;
  if (need & 1) d[0] = like(q, q.sizes());
  if (need & 2) d[1] = like(k, k.sizes());
  if (need & 4) d[2] = like(v, v.sizes());
  size_t bytes = 0;
  check_rc(spira_hip_attention_workspace(&x, 1, &bytes), "attention");
  Tensor ws = workspace(bytes, q.device());
  const auto at = [&](int i) { return d[i] ? d[i]->data_ptr() : nullptr; };
  check_rc(spira_hip_attention_backward(&x, out.data_ptr(), stats.data_ptr<float>(), ptr(rest), dout.data_ptr(), at(0),
                                        at(1), at(2), ws.data_ptr(), bytes, current_stream()),
           "attention");
  return d;
}

struct AttentionFunction : torch::autograd::Function<AttentionFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &offsets,
                        const Tensor &key_offsets, const OptTensor &key_counts, bool causal, double scale) {
    auto [out, stats, rest] = attention(q, k, v, offsets, key_offsets, key_counts, causal, scale, true);
    ctx->save_for_backward({q, k, v, offsets, key_offsets, given(key_counts), out, *stats, given(rest)});
    ctx->saved_data["need"] = int64_t(q.requires_grad()) | int64_t(k.requires_grad()) << 1 | int64_t(v.requires_grad()) << 2;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list d) {
    const variable_list v = ctx->get_saved_variables();
    auto g = attention_backward(v[0], v[1], v[2], v[3], v[4], maybe(v[5]), ctx->saved_data["causal"].toBool(),
                                ctx->saved_data["scale"].toDouble(), v[6], v[7], maybe(v[8]), dense(d[0]),
                                ctx->saved_data["need"].toInt());
    return once({given(g[0]), given(g[1]), given(g[2]), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, "attention");
  }
};

static Tensor attention_call(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &offsets,
                             const OptTensor &key_offsets, const OptTensor &key_counts, bool causal,
                             std::optional<double> scale) {
  SPIRA_CHECK_ARG(q.dim() == 3, "queries must have the shape [rows, heads, values], got ", q.sizes());
  const double by = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(std::max<int64_t>(q.size(2), 1)));
  SPIRA_CHECK_ARG(key_offsets || (k.dim() == 3 && k.size(0) == q.size(0)),
                  "attention: without offsets of their own the keys are as many as the queries, got ", k.sizes(), " and ",
                  q.sizes());
  const Tensor off = dense(offsets), key_off = key_offsets ? dense(*key_offsets) : off;
  const OptTensor oq = q, ok = k, ov = v;
  if (tracked("attention", {&oq, &ok, &ov}))
    return AttentionFunction::apply(strided(q), strided(k), strided(v), off, key_off, dense(key_counts), causal, by);
  return std::get<0>(attention(strided(q), strided(k), strided(v), off, key_off, dense(key_counts), causal, by, false));
}

// ---------------------------------------------------------------------------
// norms of the heads and their rotation
// ---------------------------------------------------------------------------
static spira_hip_heads_t heads_arguments(const Tensor &q, const Tensor &k, const OptTensor &wq, const OptTensor &wk,
                                         const OptTensor &positions, double base, bool interleaved, double eps) {
  require_heads(q, "queries", q);
  require_heads(k, "keys", q);
  spira_hip_heads_t x{};
  x.dtype = row_dtype(q);
  SPIRA_CHECK_ARG(q.size(1) > 0 && k.size(1) > 0 && q.size(1) <= 65536 && k.size(1) <= 65536,
                  "norm_rotate_heads: needs 1 to 65536 heads");
  SPIRA_CHECK_ARG(q.size(2) > 0 && q.size(2) <= 128, "norm_rotate_heads: needs heads of 1 to 128 values, got ", q.size(2));
  SPIRA_CHECK_ARG(k.size(0) == q.size(0) && k.size(2) == q.size(2), "keys must have the queries' rows and heads of ",
                  q.size(2), " values, got ", k.sizes());
  require(wq, "query_weight", q, q.scalar_type(), {q.size(2)});
  require(wk, "key_weight", q, q.scalar_type(), {q.size(2)});
  if (positions) {
    SPIRA_CHECK_ARG(positions->dim() == 1 || positions->dim() == 2, "positions must have the shape [rows] or [rows, axes], got ",
                    positions->sizes());
    x.axes = positions->dim() == 1 ? 1 : static_cast<int>(std::min<int64_t>(positions->size(1), 1 << 20));
    SPIRA_CHECK_ARG(x.axes > 0, "norm_rotate_heads: positions without an axis");
    if (positions->dim() == 1) require(positions, "positions", q, torch::kInt, {q.size(0)});
    else require(positions, "positions", q, torch::kInt, {q.size(0), -1});
    SPIRA_CHECK_ARG(q.size(2) % 2 == 0 && x.axes <= q.size(2) / 2,
                    "norm_rotate_heads: a rotation needs an even number of values and a pair for each axis, got ",
                    q.size(2), " values and ", x.axes, " axes");
    SPIRA_CHECK_ARG(base > 0 && base <= 1e300, "norm_rotate_heads: the base must be positive and finite, got ", base);
  }
  x.rows = q.size(0);
  x.heads = static_cast<int>(q.size(1));
  x.kv_heads = static_cast<int>(k.size(1));
  x.head_dim = static_cast<int>(q.size(2));
  x.interleaved = interleaved;
  x.eps = static_cast<float>(eps);
  x.base = base;
  x.queries = q.data_ptr();
  x.key = k.data_ptr();
  x.query_weight = ptr(wq);
  x.key_weight = ptr(wk);
  x.query_row = q.stride(0);
  x.query_head = q.stride(1);
  x.key_row = k.stride(0);
  x.key_head = k.stride(1);
  x.positions = static_cast<const int32_t *>(ptr(positions));
  return x;
}

static std::tuple<Tensor, Tensor> norm_rotate_heads(const Tensor &q, const Tensor &k, const OptTensor &wq,
                                                    const OptTensor &wk, const OptTensor &positions, double base,
                                                    bool interleaved, double eps) {
  const spira_hip_heads_t x = heads_arguments(q, k, wq, wk, positions, base, interleaved, eps);
  const c10::DeviceGuard guard(q.device());
  Tensor yq = like(q, q.sizes()), yk = like(k, k.sizes());
  check_rc(spira_hip_norm_rotate_heads(&x, yq.data_ptr(), yk.data_ptr(), current_stream()), "norm_rotate_heads");
  return {yq, yk};
}

struct HeadsFunction : torch::autograd::Function<HeadsFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const OptTensor &wq,
                               const OptTensor &wk, const OptTensor &positions, double base, bool interleaved,
                               double eps) {
    auto [yq, yk] = norm_rotate_heads(q, k, wq, wk, positions, base, interleaved, eps);
    ctx->save_for_backward({q, k, given(wq), given(wk), given(positions)});
    ctx->saved_data["need"] = int64_t(q.requires_grad()) | int64_t(k.requires_grad()) << 1 | int64_t(wants(wq)) << 2 |
                              int64_t(wants(wk)) << 3;
    ctx->saved_data["base"] = base;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    return {yq, yk};
  }
  static variable_list backward(AutogradContext *ctx, variable_list d) {
    const variable_list v = ctx->get_saved_variables();
    const Tensor &q = v[0], &k = v[1];
    const spira_hip_heads_t x =
        heads_arguments(q, k, maybe(v[2]), maybe(v[3]), maybe(v[4]), ctx->saved_data["base"].toDouble(),
                        ctx->saved_data["interleaved"].toBool(), ctx->saved_data["eps"].toDouble());
    const int64_t need = ctx->saved_data["need"].toInt();
    const c10::DeviceGuard guard(q.device());
    const OptTensor gq = dense(maybe(d[0])), gk = dense(maybe(d[1]));
    require(gq, "gradient", q, q.scalar_type(), {q.size(0), q.size(1), q.size(2)});
    require(gk, "gradient", q, q.scalar_type(), {k.size(0), k.size(1), k.size(2)});
    // (an output without a gradient: none of what it came from)
    variable_list g(8);
    if (gq && need & 1) g[0] = like(q, q.sizes());
    if (gk && need & 2) g[1] = like(k, k.sizes());
    if (gq && need & 4) g[2] = like(q, {q.size(2)});
    if (gk && need & 8) g[3] = like(q, {q.size(2)});
    size_t bytes = 0;
    check_rc(spira_hip_norm_rotate_heads_backward_workspace(&x, &bytes), "norm_rotate_heads");
    Tensor ws = workspace(bytes, q.device());
    const auto at = [&](int i) { return g[i].defined() ? g[i].data_ptr() : nullptr; };
    check_rc(spira_hip_norm_rotate_heads_backward(&x, ptr(gq), ptr(gk), at(0), at(1), at(2), at(3), ws.data_ptr(), bytes,
                                                  current_stream()),
             "norm_rotate_heads");
    return once(std::move(g), "norm_rotate_heads");
  }
};

static std::tuple<Tensor, Tensor> heads_call(const Tensor &q, const Tensor &k, const OptTensor &wq, const OptTensor &wk,
                                             const OptTensor &positions, double base, bool interleaved, double eps) {
  const OptTensor oq = q, ok = k;
  if (!tracked("norm_rotate_heads", {&oq, &ok, &wq, &wk}))
    return norm_rotate_heads(strided(q), strided(k), dense(wq), dense(wk), dense(positions), base, interleaved, eps);
  const variable_list v = HeadsFunction::apply(strided(q), strided(k), dense(wq), dense(wk), dense(positions), base,
                                               interleaved, eps);
  return {v[0], v[1]};
}

void register_attention(pybind11::module_ &m) {
  m.def("attention", &attention_call);
  m.def("norm_rotate_heads", &heads_call);
}

}  // namespace spira_host
