// torch_seam.cpp — titan:: operators around a block's FFN: counter-based dropout and the residual seam with its
// norms, over the C ABI of liblbk.so (include/lbk.h).  Same conventions as torch_ops.cpp.
#include "torch_util.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

Tensor or_undefined(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor or_none(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
const void* vptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ------------------------------------------------------------------ random numbers
const int64_t* check_random(double p, const OptTensor& seed, int64_t stream, const Tensor& x, const char* op) {
  TORCH_CHECK(p >= 0.0 && p <= 1.0, "titan::", op, ": p must lie in [0, 1], got ", p);
  TORCH_CHECK(stream >= 0 && stream <= UINT32_MAX, "titan::", op, ": stream must be a 32-bit number, got ", stream);
  if (!seed.has_value() || !seed->defined()) return nullptr;
  check_with(*seed, x, op, "seed");
  TORCH_CHECK(seed->scalar_type() == at::kLong && seed->numel() == 1, "titan::", op, ": seed must be one int64, got ",
              seed->scalar_type(), " ", seed->sizes());
  return seed->data_ptr<int64_t>();
}

Tensor dropout(const Tensor& x_, double p, const OptTensor& seed_tensor, int64_t seed, int64_t stream) {
  const char* op = "counter_dropout";
  check_gpu(x_, op, "x");
  const int32_t dt = elem_type(x_.scalar_type(), op, "x");
  TORCH_CHECK(x_.dim() >= 1, "titan::", op, ": x must be [..., F]");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x_.device());
  const int64_t* sp = check_random(p, seed_tensor, stream, x_, op);
  const int32_t F = dim32(x_.size(-1), op, "x's features");
  Tensor y = at::empty(x_.sizes(), x_.options());
  if (x_.numel() == 0) return y;
  const bool rows = x_.dim() == 2 && x_.stride(1) == 1 && x_.stride(0) >= F;
  const Tensor x = rows ? x_ : x_.contiguous();
  const int64_t N = x.numel() / F;
  LBK_CALL("counter_dropout", lbk_dropout(x.data_ptr(), dt, N, F, rows && N > 1 ? x.stride(0) : F, p, sp, seed, (uint32_t)stream,
                                          y.data_ptr(), cur_stream(x)));
  return y;
}

Tensor call_dropout(const Tensor& x, double p, const OptTensor& seed_tensor, int64_t seed, int64_t stream) {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("titan::counter_dropout", "").typed<decltype(dropout)>();
  return op.call(x, p, seed_tensor, seed, stream);
}

struct Dropout : public torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, const OptTensor& seed_tensor, int64_t seed, int64_t stream) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({or_undefined(seed_tensor)});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["stream"] = stream;
    return call_dropout(x, p, seed_tensor, seed, stream);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list r(5);
    const BelowAutograd below;
    if (grads[0].defined())
      r[0] = call_dropout(grads[0], ctx->saved_data["p"].toDouble(), or_none(ctx->get_saved_variables()[0]),
                          ctx->saved_data["seed"].toInt(), ctx->saved_data["stream"].toInt());
    return r;
  }
};

Tensor dropout_autograd(const Tensor& x, double p, const OptTensor& seed_tensor, int64_t seed, int64_t stream) {
  no_tangents("counter_dropout", x);
  if (at::GradMode::is_enabled() && x.requires_grad()) return Dropout::apply(x, p, seed_tensor, seed, stream);
  at::AutoDispatchBelowADInplaceOrView below;
  return call_dropout(x, p, seed_tensor, seed, stream);
}

// ------------------------------------------------------------------ the seam
struct SeamOptions {
  double residual_scale, eps, p;
  int64_t seed, stream;
};

// the operands as the kernels take them, and the C struct over them (valid while this lives)
struct Seam {
  Tensor post, gate, pre;
  lbk_seam s;
};

Seam make_seam(const Tensor& h, const Tensor& y, const OptTensor& post, const OptTensor& gate, const OptTensor& pre,
               const SeamOptions& o, const OptTensor& seed, const char* op) {
  const int32_t th = elem_type(h.scalar_type(), op, "h"), ty = elem_type(y.scalar_type(), op, "y");
  check_with(y, h, op, "y");
  TORCH_CHECK(h.dim() == 2 && y.sizes() == h.sizes(), "titan::", op, ": h and y must be one [N, d], got ", h.sizes(), " and ", y.sizes());
  TORCH_CHECK(th == ty || th == LBK_FP32, "titan::", op, ": h is ", h.scalar_type(), ", y ", y.scalar_type(),
              "; h must be of y's type or fp32");
  TORCH_CHECK(h.size(1) >= 8 && h.size(1) <= 8192, "titan::", op, ": d must lie between 8 and 8192, got ", h.size(1));
  TORCH_CHECK(o.eps >= 0, "titan::", op, ": eps must not be negative, got ", o.eps);
  const int64_t N = h.size(0), d = h.size(1);
  Seam r;
  r.post = opt_bias(post, d, h, op, "post_scale");
  r.pre = opt_bias(pre, d, h, op, "pre_scale");
  lbk_seam& s = r.s;
  s = lbk_seam{};
  if (gate.has_value() && gate->defined()) {
    check_with(*gate, h, op, "gate");
    s.gate_type = elem_type(gate->scalar_type(), op, "gate");
    TORCH_CHECK((gate->dim() == 1 || gate->dim() == 2) && gate->size(-1) == d, "titan::", op, ": gate must be [", d, "] or [G, ",
                d, "], got ", gate->sizes());
    s.gate_rows = gate->dim() == 2 ? gate->size(0) : 1;
    TORCH_CHECK(s.gate_rows > 0 && N % s.gate_rows == 0, "titan::", op, ": ", N, " rows are not shared evenly by a gate of ",
                s.gate_rows, " rows");
    r.gate = gate->contiguous();
    s.gate = r.gate.data_ptr();
  }
  s.N = N, s.d = dim32(d, op, "features"), s.state_type = th, s.type = ty;
  s.post_scale = fptr(r.post), s.pre_scale = fptr(r.pre);
  s.residual_scale = (float)o.residual_scale, s.eps = (float)o.eps;
  s.p = o.p, s.seed_dev = check_random(o.p, seed, o.stream, h, op), s.seed = o.seed, s.stream_id = (uint32_t)o.stream;
  return r;
}

using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;
using Five = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

// (h', n, rs_post, rs_pre), what the call has none of empty
Four seam_fwd_impl(const Tensor& h_, const Tensor& y_, const OptTensor& post, const OptTensor& gate, const OptTensor& pre,
                   const SeamOptions& o, const OptTensor& seed, bool train, const char* op) {
  check_gpu(h_, op, "h");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(h_.device());
  const Seam s = make_seam(h_, y_, post, gate, pre, o, seed, op);
  const Tensor h = h_.contiguous(), y = y_.contiguous();
  Tensor hn = at::empty(h.sizes(), h.options()), n = s.pre.defined() ? at::empty(y.sizes(), y.options()) : at::empty({0}, y.options());
  const auto f32 = h.options().dtype(at::kFloat);
  Tensor r1, r2;
  if (train) r1 = at::empty({s.post.defined() ? h.size(0) : 0}, f32), r2 = at::empty({s.pre.defined() ? h.size(0) : 0}, f32);
  const int st = lbk_residual_norm_fwd(&s.s, h.data_ptr(), y.data_ptr(), hn.data_ptr(), s.pre.defined() ? n.data_ptr() : nullptr,
                                       train && s.post.defined() ? r1.data_ptr<float>() : nullptr,
                                       train && s.pre.defined() ? r2.data_ptr<float>() : nullptr, cur_stream(h));
  TORCH_CHECK(st == LBK_OK, "titan::", op, ": ", lbk_status_string(st), " (status ", st, ")");
  return {hn, n, r1, r2};
}

std::tuple<Tensor, Tensor> seam_fwd(const Tensor& h, const Tensor& y, const OptTensor& post, const OptTensor& gate, const OptTensor& pre,
                                    double scale, double eps, double p, const OptTensor& seed_tensor, int64_t seed, int64_t stream) {
  auto [hn, n, r1, r2] = seam_fwd_impl(h, y, post, gate, pre, {scale, eps, p, seed, stream}, seed_tensor, false, "residual_norm");
  return {hn, n};
}

Four seam_fwd_train(const Tensor& h, const Tensor& y, const OptTensor& post, const OptTensor& gate, const OptTensor& pre, double scale,
                    double eps, double p, const OptTensor& seed_tensor, int64_t seed, int64_t stream) {
  return seam_fwd_impl(h, y, post, gate, pre, {scale, eps, p, seed, stream}, seed_tensor, true, "residual_norm_fwd_train");
}

// (dh, dy, d_post, d_gate, d_pre): d_post and d_pre in fp32, the others like their tensors; those not wanted come
// back empty
Five seam_bwd(const OptTensor& dh_, const OptTensor& dn_, const Tensor& h_, const Tensor& y_, const Tensor& r1_, const Tensor& r2_,
              const OptTensor& post, const OptTensor& gate, const OptTensor& pre, double scale, double eps, double p,
              const OptTensor& seed_tensor, int64_t seed, int64_t stream, std::array<bool, 5> want) {
  const char* op = "residual_norm_bwd";
  check_gpu(h_, op, "h");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(h_.device());
  const Seam s = make_seam(h_, y_, post, gate, pre, {scale, eps, p, seed, stream}, seed_tensor, op);
  const Tensor h = h_.contiguous(), y = y_.contiguous();
  Tensor dhn = or_undefined(dh_), dn = or_undefined(dn_);
  const std::tuple<Tensor*, const Tensor*, const char*> grads[] = {{&dhn, &h, "gradient of h"}, {&dn, &y, "gradient of n"}};
  for (const auto& [t, like, name] : grads) {
    if (!t->defined()) continue;
    check_with(*t, h, op, name);
    TORCH_CHECK(t->scalar_type() == like->scalar_type() && t->sizes() == like->sizes(), "titan::", op, ": the ", name, " must be ",
                like->scalar_type(), " ", like->sizes(), ", got ", t->scalar_type(), " ", t->sizes());
    *t = t->contiguous();
  }
  TORCH_CHECK(!dn.defined() || s.pre.defined(), "titan::", op, ": a gradient of n without pre_scale");
  TORCH_CHECK((!want[2] || s.post.defined()) && (!want[3] || s.gate.defined()) && (!want[4] || s.pre.defined()), "titan::", op,
              ": a gradient is wanted of an operand that is not there");
  const std::tuple<const Tensor*, const Tensor*, const char*> stats[] = {{&r1_, &s.post, "rs_post"}, {&r2_, &s.pre, "rs_pre"}};
  for (const auto& [r, norm, name] : stats) {
    if (!norm->defined()) continue;
    check_with(*r, h, op, name);
    TORCH_CHECK(r->scalar_type() == at::kFloat && r->numel() == h.size(0), "titan::", op, ": ", name, " must be fp32 [", h.size(0),
                "], got ", r->scalar_type(), " ", r->sizes());
  }
  const Tensor r1 = s.post.defined() ? r1_.contiguous() : Tensor(), r2 = s.pre.defined() ? r2_.contiguous() : Tensor();
  const auto f32 = h.options().dtype(at::kFloat);
  const Tensor* like[] = {&h, &y, &s.post, &s.gate, &s.pre};
  Tensor d[5];
  void* q[5];
  for (int k = 0; k < 5; ++k) {
    d[k] = want[k] ? at::empty(like[k]->sizes(), like[k]->options()) : at::empty({0}, f32);
    q[k] = want[k] ? d[k].data_ptr() : nullptr;
  }
  const size_t wsb = want[2] || want[3] || want[4] ? lbk_residual_norm_bwd_workspace_bytes(&s.s) : 0;
  Tensor ws = wsb ? workspace(wsb, h) : Tensor();
  LBK_CALL("residual_norm_bwd",
           lbk_residual_norm_bwd(&s.s, h.data_ptr(), y.data_ptr(), fptr(r1), fptr(r2), vptr(dhn), vptr(dn), q[0], q[1],
                                 static_cast<float*>(q[2]), q[3], static_cast<float*>(q[4]), wsb ? ws.data_ptr() : nullptr, wsb,
                                 cur_stream(h)));
  return {d[0], d[1], d[2], d[3], d[4]};
}

Four call_seam_fwd_train(const Tensor& h, const Tensor& y, const OptTensor& post, const OptTensor& gate, const OptTensor& pre,
                         double scale, double eps, double p, const OptTensor& seed_tensor, int64_t seed, int64_t stream) {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("titan::residual_norm_fwd_train", "").typed<decltype(seam_fwd_train)>();
  return op.call(h, y, post, gate, pre, scale, eps, p, seed_tensor, seed, stream);
}
Five call_seam_bwd(const OptTensor& dhn, const OptTensor& dn, const Tensor& h, const Tensor& y, const Tensor& r1, const Tensor& r2,
                   const OptTensor& post, const OptTensor& gate, const OptTensor& pre, double scale, double eps, double p,
                   const OptTensor& seed_tensor, int64_t seed, int64_t stream, std::array<bool, 5> want) {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("titan::residual_norm_bwd", "").typed<decltype(seam_bwd)>();
  return op.call(dhn, dn, h, y, r1, r2, post, gate, pre, scale, eps, p, seed_tensor, seed, stream, want);
}

struct SeamTrain : public torch::autograd::Function<SeamTrain> {
  static variable_list forward(AutogradContext* ctx, const Tensor& h, const Tensor& y, const OptTensor& post, const OptTensor& gate,
                               const OptTensor& pre, double scale, double eps, double p, const OptTensor& seed_tensor, int64_t seed,
                               int64_t stream) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [hn, n, r1, r2] = call_seam_fwd_train(h, y, post, gate, pre, scale, eps, p, seed_tensor, seed, stream);
    ctx->save_for_backward({h, y, r1, r2, or_undefined(post), or_undefined(gate), or_undefined(pre), or_undefined(seed_tensor)});
    for (const auto& [k, v] : {std::pair<const char*, double>{"scale", scale}, {"eps", eps}, {"p", p}}) ctx->saved_data[k] = v;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["stream"] = stream;
    ctx->set_materialize_grads(false);
    if (!pre.has_value() || !pre->defined()) ctx->mark_non_differentiable({n});
    return {hn, n};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list r(11);
    if (!grads[0].defined() && !grads[1].defined()) return r;
    const BelowAutograd below;
    const auto s = ctx->get_saved_variables();
    auto& v = ctx->saved_data;
    std::array<bool, 5> want;
    size_t input = 0;                     // inputs are counted over the tensors that are there
    for (int k = 0; k < 5; ++k) want[k] = (k < 2 || s[2 + k].defined()) && ctx->needs_input_grad(input++);
    auto [dh, dy, dpost, dgate, dpre] = call_seam_bwd(
        or_none(grads[0]), s[6].defined() ? or_none(grads[1]) : OptTensor(), s[0], s[1], s[2], s[3], or_none(s[4]), or_none(s[5]),
        or_none(s[6]), v["scale"].toDouble(), v["eps"].toDouble(), v["p"].toDouble(), or_none(s[7]), v["seed"].toInt(), v["stream"].toInt(), want);
    if (want[0]) r[0] = dh;
    if (want[1]) r[1] = dy;
    if (want[2]) r[2] = dpost.to(s[4].scalar_type()).reshape(s[4].sizes());
    if (want[3]) r[3] = dgate;
    if (want[4]) r[4] = dpre.to(s[6].scalar_type()).reshape(s[6].sizes());
    return r;
  }
};

using Two = std::tuple<Tensor, Tensor>;

Two seam_autograd(const Tensor& h, const Tensor& y, const OptTensor& post, const OptTensor& gate, const OptTensor& pre, double scale,
                  double eps, double p, const OptTensor& seed_tensor, int64_t seed, int64_t stream) {
  no_tangents("residual_norm", h, y, post, gate, pre);
  if (at::GradMode::is_enabled() &&
      (h.requires_grad() || y.requires_grad() || needs_grad(post) || needs_grad(gate) || needs_grad(pre))) {
    auto r = SeamTrain::apply(h, y, post, gate, pre, scale, eps, p, seed_tensor, seed, stream);
    return {r[0], r[1]};
  }
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("titan::residual_norm", "").typed<decltype(seam_fwd)>();
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(h, y, post, gate, pre, scale, eps, p, seed_tensor, seed, stream);
}

// for the shape functions: the operators' results are contiguous, whatever the arguments' strides
Tensor rows_like(const Tensor& x) { return at::empty(x.sizes(), x.options()); }

}  // namespace

#define SEAM_ARGS \
  "Tensor? post_scale, Tensor? gate, Tensor? pre_scale, float residual_scale, float eps, float p, Tensor? seed_tensor, int seed, int stream"

TORCH_LIBRARY_FRAGMENT(titan, m) {
  m.def("counter_dropout(Tensor x, float p, Tensor? seed_tensor, int seed, int stream) -> Tensor");
  m.def("residual_norm(Tensor h, Tensor y, " SEAM_ARGS ") -> (Tensor, Tensor)");
  m.def("residual_norm_fwd_train(Tensor h, Tensor y, " SEAM_ARGS ") -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("residual_norm_bwd(Tensor? grad_h, Tensor? grad_n, Tensor h, Tensor y, Tensor rs_post, Tensor rs_pre, " SEAM_ARGS
        ", bool[5] want) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(titan, CUDA, m) {
  m.impl("counter_dropout", &dropout);
  m.impl("residual_norm", &seam_fwd);
  m.impl("residual_norm_fwd_train", &seam_fwd_train);
  m.impl("residual_norm_bwd", &seam_bwd);
}

TORCH_LIBRARY_IMPL(titan, Autograd, m) {
  m.impl("counter_dropout", &dropout_autograd);
  m.impl("residual_norm", &seam_autograd);
  for (const char* name : {"residual_norm_fwd_train", "residual_norm_bwd"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}

TORCH_LIBRARY_IMPL(titan, Meta, m) {
  m.impl("counter_dropout", [](const Tensor& x, double, const OptTensor&, int64_t, int64_t) {
    dim32(x.size(-1), "counter_dropout", "x's features");
    return rows_like(x);
  });
  auto two = [](const Tensor& h, const Tensor& y, const OptTensor&, const OptTensor&, const OptTensor& pre, double, double, double,
                const OptTensor&, int64_t, int64_t) {
    dim32(h.size(1), "residual_norm", "features");
    return std::make_tuple(rows_like(h), pre.has_value() && pre->defined() ? rows_like(y) : at::empty({0}, y.options()));
  };
  m.impl("residual_norm", two);
  m.impl("residual_norm_fwd_train", [two](const Tensor& h, const Tensor& y, const OptTensor& post, const OptTensor& gate, const OptTensor& pre,
                                          double a, double b, double c, const OptTensor& s, int64_t e, int64_t f) {
    auto [hn, n] = two(h, y, post, gate, pre, a, b, c, s, e, f);
    auto stat = [&](const OptTensor& t) {
      return at::empty({t.has_value() && t->defined() ? h.size(0) : 0}, h.options().dtype(at::kFloat));
    };
    return std::make_tuple(hn, n, stat(post), stat(pre));
  });
  m.impl("residual_norm_bwd",
         [](const OptTensor&, const OptTensor&, const Tensor& h, const Tensor& y, const Tensor&, const Tensor&, const OptTensor& post,
            const OptTensor& gate, const OptTensor& pre, double, double, double, const OptTensor&, int64_t, int64_t, std::array<bool, 5> want) {
           const auto f32 = h.options().dtype(at::kFloat);
           auto vec = [&](bool w, const OptTensor& t) { return w ? at::empty(t->sizes(), f32) : at::empty({0}, f32); };
           return std::make_tuple(want[0] ? rows_like(h) : at::empty({0}, f32), want[1] ? rows_like(y) : at::empty({0}, f32),
                                  vec(want[2], post), want[3] ? rows_like(*gate) : at::empty({0}, f32), vec(want[4], pre));
         });
}
