// Row operators of `_C`: products grouped by expert, the router and the sum of
// its experts' rows, the gated residual norm and dropout, forward and gradients
// (no counterparts in the reference).  Outputs and workspaces come from the
// caching allocator on the current stream; nothing is read back on the host.
#include "rows.h"

namespace spira_host {

struct Linear {
  int64_t rows, groups, ci, co;
};

static Linear check_linear(const Tensor &x, const Tensor &w, const Tensor &offsets, const OptTensor &sources) {
  require(x, "features", x, x.scalar_type(), {-1, -1});
  (void)row_dtype(x);
  require(w, "weight", x, x.scalar_type(), {-1, x.size(1), -1});
  require(offsets, "offsets", x, torch::kInt, {w.size(0) + 1});
  require(sources, "rows", x, torch::kInt, {-1});
  Linear l{sources ? sources->size(0) : x.size(0), w.size(0), w.size(1), w.size(2)};
  SPIRA_CHECK_ARG(l.groups > 0 && l.ci > 0 && l.co > 0, "weight must not be empty");
  SPIRA_CHECK_ARG(l.ci <= (1 << 20) && l.co <= (1 << 20), "weight is too wide");
  SPIRA_CHECK_ARG(l.groups <= 32767, "grouped_linear: needs 1 to 32767 groups");
  return l;
}

static Tensor grouped_linear(const Tensor &x, const Tensor &w, const Tensor &offsets, const OptTensor &sources,
                             const OptTensor &bias, bool relu) {
  const Linear l = check_linear(x, w, offsets, sources);
  require(bias, "bias", x, x.scalar_type(), {l.groups, l.co});
  const c10::DeviceGuard guard(x.device());
  Tensor y = like(x, {l.rows, l.co});
  check_rc(spira_hip_grouped_linear(l.rows, l.groups, offsets.data_ptr<int32_t>(),
                                    static_cast<const int32_t *>(ptr(sources)), x.size(0), x.data_ptr(), l.ci,
                                    w.data_ptr(), ptr(bias), l.co, row_dtype(x), relu, y.data_ptr(), current_stream()),
           "grouped_linear");
  return y;
}

// (dx, dw, dbias) from dy; y: the outputs of a relu.  With slots (the rows of
// each token), dx is summed per token.
static std::tuple<OptTensor, OptTensor, OptTensor> grouped_linear_backward(
    const Tensor &x, const Tensor &w, const Tensor &offsets, const OptTensor &sources, const OptTensor &slots,
    const OptTensor &y, const Tensor &dy, bool need_dx, bool need_dw, bool need_db) {
  const Linear l = check_linear(x, w, offsets, sources);
  const int dtype = row_dtype(x);
  const auto *off = offsets.data_ptr<int32_t>();
  require(dy, "gradient", x, x.scalar_type(), {l.rows, l.co});
  require(y, "output", x, x.scalar_type(), {l.rows, l.co});
  SPIRA_CHECK_ARG(sources.has_value() == slots.has_value(), "rows and slots come together");
  require(slots, "slots", x, torch::kInt, {x.size(0), -1});
  const c10::DeviceGuard guard(x.device());
  OptTensor dx, dw, db;
  Tensor dz = dy;
  if (y || need_db) {
    if (y) dz = like(x, {l.rows, l.co});
    if (need_db) db = like(x, {l.groups, l.co});
    size_t bytes = 0;
    check_rc(spira_hip_grouped_linear_activation_gradient_workspace(l.rows, l.groups, l.co, dtype, &bytes),
             "grouped_linear");
    Tensor ws = workspace(bytes, x.device());
    check_rc(spira_hip_grouped_linear_activation_gradient(l.rows, l.groups, off, dy.data_ptr(), ptr(y), l.co, dtype,
                                                          dz.data_ptr(), db ? db->data_ptr() : nullptr, ws.data_ptr(),
                                                          bytes, current_stream()),
             "grouped_linear");
  }
  if (need_dx) {
    dx = like(x, x.sizes());
    if (!slots) {
      check_rc(spira_hip_grouped_linear_rows_gradient(l.rows, l.groups, off, dz.data_ptr(), l.co, w.data_ptr(), l.ci,
                                                      dtype, dx->data_ptr(), current_stream()),
               "grouped_linear");
    } else if (slots->size(1) > 0) {
      size_t bytes = 0;
      check_rc(spira_hip_grouped_linear_tokens_gradient_workspace(l.rows, slots->size(1), l.ci, &bytes),
               "grouped_linear");
      Tensor ws = workspace(bytes, x.device());
      check_rc(spira_hip_grouped_linear_tokens_gradient(l.rows, l.groups, off, slots->data_ptr<int32_t>(), x.size(0),
                                                        slots->size(1), dz.data_ptr(), l.co, w.data_ptr(), l.ci, dtype,
                                                        dx->data_ptr(), ws.data_ptr(), bytes, current_stream()),
               "grouped_linear");
    } else {
      dx->zero_();
    }
  }
  if (need_dw) {
    dw = like(w, w.sizes());
    size_t bytes = 0;
    check_rc(spira_hip_grouped_linear_weights_gradient_workspace(l.rows, l.groups, l.ci, l.co, &bytes),
             "grouped_linear");
    Tensor ws = workspace(bytes, x.device());
    check_rc(spira_hip_grouped_linear_weights_gradient(l.rows, l.groups, off,
                                                       static_cast<const int32_t *>(ptr(sources)), x.size(0),
                                                       x.data_ptr(), l.ci, dz.data_ptr(), l.co, dtype, dw->data_ptr(),
                                                       ws.data_ptr(), bytes, current_stream()),
             "grouped_linear");
  }
  return {dx, dw, db};
}

static std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> route(const Tensor &logits, int64_t k, bool renormalize) {
  require(logits, "logits", logits, logits.scalar_type(), {-1, -1});
  const int dtype = row_dtype(logits);
  const int64_t tokens = logits.size(0), experts = logits.size(1);
  SPIRA_CHECK_ARG(experts > 0 && experts <= 512, "route_experts: needs 1 to 512 experts, got ", experts);
  SPIRA_CHECK_ARG(k > 0 && k <= 16 && k <= experts, "route_experts: needs 1 to 16 choices of ", experts,
                  " experts, got ", k);
  const c10::DeviceGuard guard(logits.device());
  size_t bytes = 0;
  check_rc(spira_hip_route_workspace(tokens, experts, k, &bytes), "route_experts");
  Tensor weights = floats(logits, {tokens, k}), chosen = empty_i32({tokens, k}, logits.device());
  Tensor offsets = empty_i32({experts + 1}, logits.device()), rows = empty_i32({tokens * k}, logits.device());
  Tensor slots = empty_i32({tokens, k}, logits.device()), ws = workspace(bytes, logits.device());
  check_rc(spira_hip_route(logits.data_ptr(), tokens, experts, k, dtype, renormalize, weights.data_ptr<float>(),
                           chosen.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(), rows.data_ptr<int32_t>(),
                           slots.data_ptr<int32_t>(), ws.data_ptr(), bytes, current_stream()),
           "route_experts");
  return {weights, chosen, offsets, rows, slots};
}

static Tensor route_backward(const Tensor &logits, const Tensor &weights, const Tensor &chosen, const Tensor &dweights,
                             bool renormalize) {
  require(logits, "logits", logits, logits.scalar_type(), {-1, -1});
  const int dtype = row_dtype(logits);
  require(chosen, "experts", logits, torch::kInt, {logits.size(0), -1});
  require(weights, "weights", logits, torch::kFloat, {logits.size(0), chosen.size(1)});
  require(dweights, "gradient", logits, torch::kFloat, {logits.size(0), chosen.size(1)});
  const c10::DeviceGuard guard(logits.device());
  Tensor d = like(logits, logits.sizes());
  check_rc(spira_hip_route_backward(logits.data_ptr(), logits.size(0), logits.size(1), chosen.size(1), dtype,
                                    renormalize, weights.data_ptr<float>(), chosen.data_ptr<int32_t>(),
                                    dweights.data_ptr<float>(), d.data_ptr(), current_stream()),
           "route_experts");
  return d;
}

static void check_combine(const Tensor &h, const Tensor &slots, const Tensor &weights) {
  require(h, "features", h, h.scalar_type(), {-1, -1});
  (void)row_dtype(h);
  require(slots, "slots", h, torch::kInt, {-1, -1});
  require(weights, "weights", h, torch::kFloat, {slots.size(0), slots.size(1)});
  SPIRA_CHECK_ARG(slots.size(1) > 0 && h.size(1) > 0, "combine_experts: no choices or no channels");
}

static Tensor combine(const Tensor &h, const Tensor &slots, const Tensor &weights) {
  check_combine(h, slots, weights);
  const c10::DeviceGuard guard(h.device());
  Tensor y = like(h, {slots.size(0), h.size(1)});
  check_rc(spira_hip_combine(h.data_ptr(), h.size(0), slots.data_ptr<int32_t>(), weights.data_ptr<float>(),
                             slots.size(0), slots.size(1), h.size(1), row_dtype(h), y.data_ptr(), current_stream()),
           "combine_experts");
  return y;
}

static std::tuple<OptTensor, OptTensor> combine_backward(const Tensor &h, const Tensor &rows, const Tensor &slots,
                                                         const Tensor &weights, const Tensor &dy, bool need_dh,
                                                         bool need_dw) {
  check_combine(h, slots, weights);
  require(rows, "rows", h, torch::kInt, {h.size(0)});
  require(dy, "gradient", h, h.scalar_type(), {slots.size(0), h.size(1)});
  const c10::DeviceGuard guard(h.device());
  OptTensor dh, dw;
  if (need_dh) dh = like(h, h.sizes());
  if (need_dw) dw = floats(h, weights.sizes());
  check_rc(spira_hip_combine_backward(h.data_ptr(), h.size(0), rows.data_ptr<int32_t>(), slots.data_ptr<int32_t>(),
                                      weights.data_ptr<float>(), dy.data_ptr(), slots.size(0), slots.size(1),
                                      h.size(1), row_dtype(h), dh ? dh->data_ptr() : nullptr,
                                      dw ? dw->data_ptr<float>() : nullptr, current_stream()),
           "combine_experts");
  return {dh, dw};
}

struct NormShape {
  int64_t n, c;
  int gate_form;
};

static NormShape check_norm(const Tensor &x, const OptTensor &h, const OptTensor &weight, const OptTensor &gate,
                            const OptTensor &next_weight) {
  const auto type = x.scalar_type();
  require(x, "residual", x, type, {-1, -1});
  (void)row_dtype(x);
  const int64_t n = x.size(0), c = x.size(1);
  SPIRA_CHECK_ARG(c > 0 && c <= 16384, "gated_residual_norm: needs 1 to 16384 channels, got ", c);
  require(h, "update", x, type, {n, c});
  require(weight, "weight", x, type, {c});
  require(next_weight, "next_weight", x, type, {c});
  SPIRA_CHECK_ARG(h || next_weight, "gated_residual_norm: neither an update nor a next norm");
  SPIRA_CHECK_ARG(h || (!weight && !gate), "gated_residual_norm: a weight or gate without an update");
  int form = 0;
  if (gate) {
    form = gate->dim() == 1 ? 1 : gate->dim() == 2 && gate->size(1) == 1 && c > 1 ? 2 : 3;
    if (form == 1) require(*gate, "gate", x, type, {c});
    else require(*gate, "gate (of two dimensions)", x, type, {n, form == 2 ? 1 : c});
  }
  return {n, c, form};
}

// (r or None without an update, next or None, 1 / root mean squares of the
// update and of r, or None unless `train`)
static std::tuple<OptTensor, OptTensor, OptTensor, OptTensor> gated_residual_norm(
    const Tensor &x, const OptTensor &h, const OptTensor &weight, const OptTensor &gate, bool gate_sigmoid,
    double scale, const OptTensor &next_weight, double eps, bool train) {
  const NormShape s = check_norm(x, h, weight, gate, next_weight);
  const c10::DeviceGuard guard(x.device());
  OptTensor r, next, inv_h, inv_r;
  if (h) r = like(x, x.sizes());
  if (next_weight) next = like(x, x.sizes());
  if (train && weight) inv_h = floats(x, {s.n});
  if (train && next_weight) inv_r = floats(x, {s.n});
  const auto at = [](OptTensor &t) { return t ? t->data_ptr() : nullptr; };
  check_rc(spira_hip_gated_residual_norm(x.data_ptr(), ptr(h), s.n, s.c, row_dtype(x), ptr(weight), ptr(gate),
                                         s.gate_form, gate_sigmoid, scale, ptr(next_weight), eps, at(r), at(next),
                                         static_cast<float *>(at(inv_h)), static_cast<float *>(at(inv_r)),
                                         current_stream()),
           "gated_residual_norm");
  return {r, next, inv_h, inv_r};
}

// (dx, dh, dweight, dgate, dnext_weight), each None unless it is in `need`
static std::vector<OptTensor> gated_residual_norm_backward(
    const Tensor &x, const OptTensor &h, const OptTensor &weight, const OptTensor &gate, bool gate_sigmoid,
    double scale, const OptTensor &next_weight, const OptTensor &inv_h, const OptTensor &inv_r, const OptTensor &dr,
    const OptTensor &dnext, const std::array<bool, 5> &need) {
  const NormShape s = check_norm(x, h, weight, gate, next_weight);
  const auto type = x.scalar_type();
  require(inv_h, "inverse root mean squares", x, torch::kFloat, {s.n});
  require(inv_r, "inverse root mean squares", x, torch::kFloat, {s.n});
  require(dr, "gradient", x, type, {s.n, s.c});
  require(dnext, "gradient", x, type, {s.n, s.c});
  SPIRA_CHECK_ARG((!weight || inv_h) && (!dnext || (inv_r && next_weight)),
                  "gated_residual_norm: the forward pass kept nothing for a gradient");
  const c10::DeviceGuard guard(x.device());
  std::vector<OptTensor> d(5);
  if (need[0]) d[0] = like(x, x.sizes());
  if (need[1] && h) d[1] = like(x, x.sizes());
  if (need[2] && weight) d[2] = like(x, {s.c});
  if (need[3] && gate) d[3] = like(x, gate->sizes());
  if (need[4] && next_weight) d[4] = dnext ? like(x, {s.c}) : torch::zeros({s.c}, x.options());
  size_t bytes = 0;
  check_rc(spira_hip_gated_residual_norm_backward_workspace(s.n, s.c, row_dtype(x), &bytes), "gated_residual_norm");
  Tensor ws = workspace(bytes, x.device());
  const auto at = [&](int i) { return d[i] ? d[i]->data_ptr() : nullptr; };
  check_rc(spira_hip_gated_residual_norm_backward(
               x.data_ptr(), ptr(h), s.n, s.c, row_dtype(x), ptr(weight), ptr(gate), s.gate_form, gate_sigmoid, scale,
               ptr(next_weight), static_cast<const float *>(ptr(inv_h)), static_cast<const float *>(ptr(inv_r)),
               ptr(dr), ptr(dnext), at(0), at(1), at(2), at(3), at(4), ws.data_ptr(), bytes, current_stream()),
           "gated_residual_norm");
  return d;
}

static Tensor dropout(const Tensor &x, double p, uint64_t seed, uint64_t offset, const OptTensor &residual) {
  require_device(x, "features");
  const int dtype = row_dtype(x);
  SPIRA_CHECK_ARG(p >= 0.0 && p <= 1.0, "dropout: p must be in [0, 1], got ", p);
  if (residual) {
    require_device(*residual, "residual");
    SPIRA_CHECK_ARG(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() &&
                        residual->device() == x.device(),
                    "residual must have the features' shape, type and device");
  }
  const c10::DeviceGuard guard(x.device());
  Tensor y = like(x, x.sizes());
  check_rc(spira_hip_dropout(x.data_ptr(), ptr(residual), x.numel(), dtype, p, seed, offset, y.data_ptr(),
                             current_stream()),
           "dropout");
  return y;
}

// (loss, counts, mean probabilities, what the gradient needs)
static std::tuple<Tensor, Tensor, Tensor, Tensor> balance(const Tensor &logits, const Tensor &offsets) {
  require(logits, "logits", logits, logits.scalar_type(), {-1, -1});
  const int dtype = row_dtype(logits);
  const int64_t tokens = logits.size(0), experts = logits.size(1);
  SPIRA_CHECK_ARG(experts > 0 && experts <= 512, "balance_loss: needs 1 to 512 experts, got ", experts);
  require(offsets, "offsets", logits, torch::kInt, {experts + 1});
  const c10::DeviceGuard guard(logits.device());
  size_t bytes = 0;
  check_rc(spira_hip_balance_workspace(tokens, experts, &bytes), "balance_loss");
  Tensor loss = floats(logits, {}), counts = empty_i32({experts}, logits.device()), mean = floats(logits, {experts});
  Tensor kept = floats(logits, {experts + 1}), ws = workspace(bytes, logits.device());
  check_rc(spira_hip_balance(logits.data_ptr(), tokens, experts, dtype, offsets.data_ptr<int32_t>(),
                             loss.data_ptr<float>(), counts.data_ptr<int32_t>(), mean.data_ptr<float>(),
                             kept.data_ptr<float>(), ws.data_ptr(), bytes, current_stream()),
           "balance_loss");
  return {loss, counts, mean, kept};
}

static Tensor balance_backward(const Tensor &logits, const Tensor &kept, const Tensor &dloss) {
  require(logits, "logits", logits, logits.scalar_type(), {-1, -1});
  require(kept, "sums", logits, torch::kFloat, {logits.size(1) + 1});
  require(dloss, "gradient", logits, torch::kFloat, {});
  const c10::DeviceGuard guard(logits.device());
  Tensor d = like(logits, logits.sizes());
  check_rc(spira_hip_balance_backward(logits.data_ptr(), logits.size(0), logits.size(1), row_dtype(logits),
                                      kept.data_ptr<float>(), dloss.data_ptr<float>(), d.data_ptr(), current_stream()),
           "balance_loss");
  return d;
}

// ---------------------------------------------------------------------------
// Gradients.  The functions above take contiguous tensors and know nothing of
// autograd; those below are what Python calls.  (In C++: with Python's autograd
// functions a training step of a small operator was bound by the host, 104 us
// where its kernels take 23.)
// ---------------------------------------------------------------------------
struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const OptTensor &bias,
                        const Tensor &offsets, const OptTensor &rows, const OptTensor &slots, bool relu) {
    Tensor y = grouped_linear(x, w, offsets, rows, bias, relu);
    ctx->save_for_backward({x, w, offsets, given(rows), given(slots), relu ? y : Tensor()});
    ctx->saved_data["need"] = int64_t(x.requires_grad()) | int64_t(w.requires_grad()) << 1 | int64_t(wants(bias)) << 2;
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list d) {
    const variable_list v = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    auto [dx, dw, db] = grouped_linear_backward(v[0], v[1], v[2], maybe(v[3]), maybe(v[4]), maybe(v[5]), dense(d[0]),
                                                need & 1, need & 2, need & 4);
    return once({given(dx), given(dw), given(db), Tensor(), Tensor(), Tensor(), Tensor()}, "grouped_linear");
  }
};

static Tensor grouped_linear_call(const Tensor &x, const Tensor &w, const Tensor &offsets, const OptTensor &rows,
                                  const OptTensor &slots, const OptTensor &bias, bool relu) {
  if (slots) {
    SPIRA_CHECK_ARG(rows && slots->dim() == 2 && x.dim() == 2 && slots->size(0) == x.size(0) &&
                        slots->numel() == rows->numel(),
                    "grouped_linear: routes of ", slots->sizes(), " choices do not fit features of ", x.sizes());
  }
  const OptTensor ox = x, ow = w;
  if (tracked("grouped_linear", {&ox, &ow, &bias}))
    return LinearFunction::apply(dense(x), dense(w), dense(bias), dense(offsets), dense(rows), dense(slots), relu);
  return grouped_linear(dense(x), dense(w), dense(offsets), dense(rows), dense(bias), relu);
}

struct RouteFunction : torch::autograd::Function<RouteFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &logits, int64_t k, bool renormalize) {
    auto [weights, chosen, offsets, rows, slots] = route(logits, k, renormalize);
    ctx->save_for_backward({logits, weights, chosen});
    ctx->saved_data["renormalize"] = renormalize;
    ctx->mark_non_differentiable({chosen, offsets, rows, slots});
    ctx->set_materialize_grads(false);  // (four of zeros, for the integers)
    return {weights, chosen, offsets, rows, slots};
  }
  static variable_list backward(AutogradContext *ctx, variable_list d) {
    const variable_list v = ctx->get_saved_variables();
    if (!d[0].defined()) return {Tensor(), Tensor(), Tensor()};  // (what follows had no gradient of the weights)
    return once({route_backward(v[0], v[1], v[2], dense(d[0]), ctx->saved_data["renormalize"].toBool()), Tensor(),
                 Tensor()},
                "route_experts");
  }
};

static std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> route_call(const Tensor &logits, int64_t k,
                                                                     bool renormalize) {
  const OptTensor l = logits;
  if (!tracked("route_experts", {&l})) return route(dense(logits), k, renormalize);
  const variable_list v = RouteFunction::apply(dense(logits), k, renormalize);
  return {v[0], v[1], v[2], v[3], v[4]};
}

struct CombineFunction : torch::autograd::Function<CombineFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &h, const Tensor &weights, const Tensor &rows,
                        const Tensor &slots) {
    ctx->save_for_backward({h, weights, rows, slots});
    ctx->saved_data["need"] = int64_t(h.requires_grad()) | int64_t(weights.requires_grad()) << 1;
    return combine(h, slots, weights);
  }
  static variable_list backward(AutogradContext *ctx, variable_list d) {
    const variable_list v = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    auto [dh, dw] = combine_backward(v[0], v[2], v[3], v[1], dense(d[0]), need & 1, need & 2);
    return once({given(dh), given(dw), Tensor(), Tensor()}, "combine_experts");
  }
};

static Tensor combine_call(const Tensor &h, const Tensor &weights, const Tensor &rows, const Tensor &slots) {
  // (a slot past the features' rows would count as none)
  SPIRA_CHECK_ARG(h.dim() == 2 && rows.numel() == h.size(0) && slots.numel() == rows.numel(),
                  "combine_experts: routes of ", slots.sizes(), " choices do not fit features of ", h.sizes());
  const OptTensor oh = h, ow = weights;
  if (tracked("combine_experts", {&oh, &ow})) return CombineFunction::apply(dense(h), dense(weights), dense(rows), dense(slots));
  return combine(dense(h), dense(slots), dense(weights));
}

struct NormFunction : torch::autograd::Function<NormFunction> {
  // (the outputs that there are: r, next)
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const OptTensor &h, const OptTensor &weight,
                               const OptTensor &gate, const OptTensor &next_weight, bool gate_sigmoid, double scale,
                               double eps) {
    auto [r, next, inv_h, inv_r] = gated_residual_norm(x, h, weight, gate, gate_sigmoid, scale, next_weight, eps, true);
    ctx->save_for_backward(
        {x, given(h), given(weight), given(gate), given(next_weight), given(inv_h), given(inv_r)});
    ctx->saved_data["need"] = int64_t(x.requires_grad()) | int64_t(wants(h)) << 1 | int64_t(wants(weight)) << 2 |
                              int64_t(wants(gate)) << 3 | int64_t(wants(next_weight)) << 4;
    ctx->saved_data["gate_sigmoid"] = gate_sigmoid;
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    variable_list out;
    if (r) out.push_back(*r);
    if (next) out.push_back(*next);
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list d) {
    const variable_list v = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    Tensor dr = v[1].defined() ? d[0] : Tensor(), dn = v[4].defined() ? d.back() : Tensor();
    auto g = gated_residual_norm_backward(
        v[0], maybe(v[1]), maybe(v[2]), maybe(v[3]), ctx->saved_data["gate_sigmoid"].toBool(),
        ctx->saved_data["scale"].toDouble(), maybe(v[4]), maybe(v[5]), maybe(v[6]), dense(maybe(dr)), dense(maybe(dn)),
        {bool(need & 1), bool(need & 2), bool(need & 4), bool(need & 8), bool(need & 16)});
    variable_list out;
    for (const OptTensor &t : g) out.push_back(given(t));
    out.resize(8);
    return once(std::move(out), "gated_residual_norm");
  }
};

static std::tuple<OptTensor, OptTensor> norm_call(const Tensor &x, const OptTensor &h, const OptTensor &weight,
                                                  const OptTensor &gate, bool gate_sigmoid, double scale,
                                                  const OptTensor &next_weight, double eps) {
  const OptTensor ox = x;
  if (!tracked("gated_residual_norm", {&ox, &h, &weight, &gate, &next_weight})) {
    auto out = gated_residual_norm(dense(x), dense(h), dense(weight), dense(gate), gate_sigmoid, scale,
                                   dense(next_weight), eps, false);
    return {std::get<0>(out), std::get<1>(out)};
  }
  const variable_list v = NormFunction::apply(dense(x), dense(h), dense(weight), dense(gate), dense(next_weight),
                                              gate_sigmoid, scale, eps);
  return {h ? OptTensor(v[0]) : std::nullopt, next_weight ? OptTensor(v.back()) : std::nullopt};
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &residual, double p, int64_t seed,
                        int64_t offset) {
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["need"] = int64_t(x.requires_grad()) | int64_t(wants(residual)) << 1;
    return dropout(x, p, static_cast<uint64_t>(seed), static_cast<uint64_t>(offset), residual);
  }
  static variable_list backward(AutogradContext *ctx, variable_list d) {
    const int64_t need = ctx->saved_data["need"].toInt();
    Tensor dx;
    if (need & 1)
      dx = dropout(dense(d[0]), ctx->saved_data["p"].toDouble(), static_cast<uint64_t>(ctx->saved_data["seed"].toInt()),
                   static_cast<uint64_t>(ctx->saved_data["offset"].toInt()), std::nullopt);
    // (the residual's gradient is the output's own, of any order)
    variable_list own = once({dx}, "dropout");
    return {own[0], need & 2 ? d[0] : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

static Tensor dropout_call(const Tensor &x, double p, uint64_t seed, uint64_t offset, const OptTensor &residual) {
  const OptTensor ox = x;
  if (tracked("dropout", {&ox, &residual}))
    return DropoutFunction::apply(dense(x), dense(residual), p, static_cast<int64_t>(seed),
                                  static_cast<int64_t>(offset));
  return dropout(dense(x), p, seed, offset, dense(residual));
}

struct BalanceFunction : torch::autograd::Function<BalanceFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &offsets) {
    auto [loss, counts, mean, kept] = balance(logits, offsets);
    ctx->save_for_backward({logits, kept});
    ctx->mark_non_differentiable({counts, mean});
    ctx->set_materialize_grads(false);
    return {loss, counts, mean};
  }
  static variable_list backward(AutogradContext *ctx, variable_list d) {
    const variable_list v = ctx->get_saved_variables();
    if (!d[0].defined()) return {Tensor(), Tensor()};
    return once({balance_backward(v[0], v[1], dense(d[0])), Tensor()}, "balance_loss");
  }
};

static std::tuple<Tensor, Tensor, Tensor> balance_call(const Tensor &logits, const Tensor &offsets) {
  const OptTensor l = logits;
  if (!tracked("balance_loss", {&l})) {
    auto out = balance(dense(logits), dense(offsets));
    return {std::get<0>(out), std::get<1>(out), std::get<2>(out)};
  }
  const variable_list v = BalanceFunction::apply(dense(logits), dense(offsets));
  return {v[0], v[1], v[2]};
}

void register_experts(pybind11::module_ &m) {
  m.def("grouped_linear", &grouped_linear_call);
  m.def("route_experts", &route_call);
  m.def("combine_experts", &combine_call);
  m.def("gated_residual_norm", &norm_call);
  m.def("dropout", &dropout_call);
  m.def("balance_loss", &balance_call);
}

}  // namespace spira_host
