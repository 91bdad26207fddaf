// torch_ffn.cpp — titan:: operators on weights in microscaled 4-bit floating point and of the dense
// gated FFN, over the C ABI of liblbk.so (include/lbk.h).  Same conventions as torch_ops.cpp.
#include "torch_util.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<at::Tensor>;

int32_t elem_type(at::ScalarType t, const char* op, const char* name) {
  TORCH_CHECK(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat, "titan::", op, ": ", name,
              " must be bf16, fp16 or fp32, got ", t);
  return t == at::kBFloat16 ? LBK_BF16 : t == at::kHalf ? LBK_FP16 : LBK_FP32;
}

// contiguous and 16-byte aligned (a view may start anywhere in its storage)
Tensor dense16(const Tensor& t) {
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) & 15 ? c.clone() : c;
}

void check_with(const Tensor& t, const Tensor& x, const char* op, const char* name) {
  check_gpu(t, op, name);
  TORCH_CHECK(t.device() == x.device(), "titan::", op, ": ", name, " is on ", t.device(), ", the input on ", x.device());
}

// of a weight [R, K, ...]
void check_slots(const Tensor& t, const char* op) {
  dim32(t.size(0), op, "block rows");
  dim32(t.size(1), op, "slots of a row");
}

// ------------------------------------------------------------------ quantisation
std::tuple<Tensor, Tensor> mx_quantize(const Tensor& x_) {
  const char* op = "mx_quantize";
  check_gpu(x_, op, "x");
  const int32_t dt = elem_type(x_.scalar_type(), op, "x");
  TORCH_CHECK(x_.dim() == 2 && x_.size(1) > 0 && x_.size(1) % 32 == 0, "titan::", op,
              ": x must be [N, F] with F a multiple of 32, got ", x_.sizes());
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x_.device());
  const int64_t N = x_.size(0), per16 = dt == LBK_FP32 ? 4 : 8;
  const int32_t F = dim32(x_.size(1), op, "x's features");
  const bool rows = x_.stride(1) == 1 && x_.stride(0) >= F && x_.stride(0) % per16 == 0 &&
                    (reinterpret_cast<uintptr_t>(x_.data_ptr()) & 15) == 0;
  const Tensor x = rows ? x_ : dense16(x_);
  Tensor codes = at::empty({N, F / 2}, x.options().dtype(at::kByte)), scales = at::empty({N, F / 32}, codes.options());
  LBK_CALL("mx_quantize", lbk_mx_quantize(x.data_ptr(), dt, N, F, N > 1 ? x.stride(0) : F, codes.data_ptr<uint8_t>(),
                                          scales.data_ptr<uint8_t>(), cur_stream(x)));
  return {codes, scales};
}

Tensor mx_dequantize(const Tensor& codes_, const Tensor& scales_, at::ScalarType dtype) {
  const char* op = "mx_dequantize";
  check_gpu(codes_, op, "codes");
  check_with(scales_, codes_, op, "scales");
  const int32_t dt = elem_type(dtype, op, "dtype");
  TORCH_CHECK(codes_.scalar_type() == at::kByte && scales_.scalar_type() == at::kByte, "titan::", op,
              ": codes and scales must be uint8");
  TORCH_CHECK(codes_.dim() == 2 && scales_.dim() == 2 && codes_.size(1) > 0 && codes_.size(1) == 16 * scales_.size(1) &&
                  codes_.size(0) == scales_.size(0),
              "titan::", op, ": codes must be [N, F/2] and scales [N, F/32], got ", codes_.sizes(), " and ", scales_.sizes());
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(codes_.device());
  const int64_t N = codes_.size(0);
  const int32_t F = dim32(2 * codes_.size(1), op, "features");
  const Tensor codes = dense16(codes_), scales = scales_.contiguous();
  Tensor out = at::empty({N, F}, codes.options().dtype(dtype));
  LBK_CALL("mx_dequantize", lbk_mx_dequantize(codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), N, F, dt,
                                              out.data_ptr(), cur_stream(codes)));
  return out;
}

std::tuple<Tensor, Tensor> mx_quantize_tiles(const Tensor& v_) {
  const char* op = "mx_quantize_tiles";
  check_gpu(v_, op, "values");
  const int32_t dt = elem_type(v_.scalar_type(), op, "values");
  TORCH_CHECK(v_.dim() == 4 && v_.size(2) == v_.size(3), "titan::", op, ": values must be [R, K, B, B], got ", v_.sizes());
  TORCH_CHECK(v_.size(2) == 32 || v_.size(2) == 64, "titan::", op,
              ": B must be 32 or 64 (a group of 32 inputs lies in one tile), got ", v_.size(2));
  check_slots(v_, op);
  const int32_t R = (int32_t)v_.size(0), K = (int32_t)v_.size(1), B = (int32_t)v_.size(2);
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(v_.device());
  const Tensor v = v_.contiguous();
  Tensor codes = at::empty({R, K, B, B / 2}, v.options().dtype(at::kByte)),
         scales = at::empty({R, K, B, B / 32}, codes.options());
  LBK_CALL("mx_quantize_tiles", lbk_mx_quantize_tiles(v.data_ptr(), dt, R, K, B, codes.data_ptr<uint8_t>(),
                                                      scales.data_ptr<uint8_t>(), cur_stream(v)));
  return {codes, scales};
}

// codes [R, K, B, B/2], scales [R, K, B, B/32] (made contiguous in place)
void check_mx_tiles(Tensor& c, Tensor& s, const char* op, const char* name) {
  check_gpu(c, op, name);
  check_with(s, c, op, name);
  TORCH_CHECK(c.scalar_type() == at::kByte && s.scalar_type() == at::kByte, "titan::", op, ": ", name,
              " codes and scales must be uint8");
  TORCH_CHECK(c.dim() == 4 && (c.size(2) == 32 || c.size(2) == 64) && c.size(3) * 2 == c.size(2), "titan::", op, ": ", name,
              " codes must be [R, K, B, B/2] with B 32 or 64, got ", c.sizes());
  TORCH_CHECK(s.dim() == 4 && s.size(0) == c.size(0) && s.size(1) == c.size(1) && s.size(2) == c.size(2) &&
                  s.size(3) * 32 == c.size(2),
              "titan::", op, ": ", name, " scales must be [R, K, B, B/32], got ", s.sizes());
  check_slots(c, op);
  c = dense16(c);
  s = dense16(s);
}

Tensor mx_dequantize_tiles(const Tensor& codes_, const Tensor& scales_, at::ScalarType dtype) {
  const char* op = "mx_dequantize_tiles";
  Tensor c = codes_, s = scales_;
  const int32_t dt = elem_type(dtype, op, "dtype");
  check_gpu(c, op, "codes");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(c.device());
  check_mx_tiles(c, s, op, "weight");
  const int32_t R = (int32_t)c.size(0), K = (int32_t)c.size(1), B = (int32_t)c.size(2);
  Tensor v = at::empty({R, K, B, B}, c.options().dtype(dtype));
  LBK_CALL("mx_dequantize_tiles", lbk_mx_dequantize_tiles(c.data_ptr<uint8_t>(), s.data_ptr<uint8_t>(), R, K, B, dt, v.data_ptr(),
                                                          cur_stream(c)));
  return v;
}

// ------------------------------------------------------------------ products
lbk_bell_mx make_mx(Tensor& c, Tensor& s, Tensor& ci, const Tensor& x, const char* op, const char* name) {
  check_with(c, x, op, name);
  check_with(ci, x, op, name);
  check_mx_tiles(c, s, op, name);
  TORCH_CHECK(ci.scalar_type() == at::kInt, "titan::", op, ": ", name, " col_indices must be int32");
  TORCH_CHECK(ci.dim() == 2 && ci.size(0) == c.size(0) && ci.size(1) == c.size(1), "titan::", op, ": ", name,
              " col_indices must be [R, K] matching codes, got ", ci.sizes());
  ci = ci.contiguous();
  return lbk_bell_mx{c.data_ptr<uint8_t>(), s.data_ptr<uint8_t>(), ci.data_ptr<int32_t>(), (int32_t)c.size(0),
                     (int32_t)c.size(1), (int32_t)c.size(2)};
}

Tensor x2d16(const Tensor& x, const char* op) {
  if (x.dim() == 2) dim32(x.size(1), op, "x's features");      // ahead of a copy
  return dense16(check_x2d(x, op));
}

Tensor matmul_mx(const Tensor& x_, const Tensor& c_, const Tensor& s_, const Tensor& ci_, const OptTensor& bias_) {
  const char* op = "block_ell_matmul_mx";
  check_gpu(x_, op, "x");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x_.device());
  Tensor c = c_, s = s_, ci = ci_, x = x2d16(x_, op);
  const lbk_bell_mx w = make_mx(c, s, ci, x, op, "weight");
  const int64_t N = x.size(0), O = (int64_t)w.R * w.B;
  const int32_t F = (int32_t)x.size(1);
  TORCH_CHECK(F > 0 && F % w.B == 0, "titan::", op, ": in_features ", F, " not a multiple of B=", w.B);
  const Tensor bias = opt_bias(bias_, O, x, op, "bias");
  Tensor y = at::empty({N, O}, x.options());
  const size_t wsb = lbk_mx_matmul_workspace_bytes(N, F, &w);
  Tensor ws = wsb ? workspace(wsb, x) : Tensor();
  LBK_CALL("block_ell_matmul_mx", lbk_mx_matmul_bf16(bf(x), N, F, &w, fptr(bias), bfm(y),
                                                     wsb ? ws.data_ptr() : nullptr, wsb, cur_stream(x)));
  return y;
}

Tensor swiglu_mx(const Tensor& x_, const Tensor& cg_, const Tensor& sg_, const Tensor& ig_, const OptTensor& bg_,
                 const Tensor& cu_, const Tensor& su_, const Tensor& iu_, const OptTensor& bu_, const Tensor& cd_,
                 const Tensor& sd_, const Tensor& id_, const OptTensor& bd_, bool add_residual) {
  const char* op = "block_ell_swiglu_fwd_mx";
  check_gpu(x_, op, "x");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x_.device());
  Tensor x = x2d16(x_, op), cg = cg_, sg = sg_, ig = ig_, cu = cu_, su = su_, iu = iu_, cd = cd_, sd = sd_, id = id_;
  const lbk_bell_mx g = make_mx(cg, sg, ig, x, op, "gate"), u = make_mx(cu, su, iu, x, op, "up"),
                    d = make_mx(cd, sd, id, x, op, "down");
  const int64_t N = x.size(0), F = (int64_t)g.R * g.B;
  const int32_t D = (int32_t)x.size(1);
  TORCH_CHECK(g.B == u.B && g.B == d.B, "titan::", op, ": the three weights must have one tile size");
  TORCH_CHECK(g.R == u.R && g.R > 0, "titan::", op, ": gate and up must have the same (non-zero) output features");
  TORCH_CHECK(D > 0 && (int64_t)d.R * d.B == D, "titan::", op, ": down's ", (int64_t)d.R * d.B,
              " output features are not d_model=", D);
  const Tensor bg = opt_bias(bg_, F, x, op, "b_gate"), bu = opt_bias(bu_, F, x, op, "b_up"),
               bd = opt_bias(bd_, D, x, op, "b_down");
  Tensor out = at::empty({N, D}, x.options());
  const size_t wsb = lbk_mx_swiglu_workspace_bytes(N, D, &g, &u, &d);
  Tensor ws = workspace(wsb, x);
  LBK_CALL("block_ell_swiglu_fwd_mx",
           lbk_mx_swiglu_fwd_bf16(bf(x), N, D, &g, &u, &d, fptr(bg), fptr(bu), fptr(bd), add_residual ? 1 : 0,
                                  bfm(out), ws.data_ptr(), wsb, cur_stream(x)));
  return out;
}

// ------------------------------------------------------------------ dense gated FFN
struct Gated {
  Tensor x, wg, wu, wd;
  int64_t N, D, F;
  int32_t dt, act;
};

Gated make_gated(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, c10::string_view act, const char* op) {
  check_gpu(x, op, "x");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "titan::", op, ": x must be bf16 or fp16");
  TORCH_CHECK(x.dim() == 2, "titan::", op, ": x must be 2D [N, d_model], got ", x.sizes());
  TORCH_CHECK(act == "silu" || act == "gelu", "titan::", op, ": activation must be 'silu' or 'gelu', got '", act, "'");
  const std::pair<const Tensor*, const char*> ws[] = {{&wg, "w_gate"}, {&wu, "w_up"}, {&wd, "w_down"}};
  for (const auto& [w, name] : ws) {
    check_with(*w, x, op, name);
    TORCH_CHECK(w->scalar_type() == x.scalar_type(), "titan::", op, ": ", name, " is ", w->scalar_type(), ", x is ",
                x.scalar_type());
    TORCH_CHECK(w->dim() == 2, "titan::", op, ": ", name, " must be 2D [out, in], got ", w->sizes());
  }
  const int64_t D = x.size(1), F = wg.size(0);
  TORCH_CHECK(wg.size(1) == D && wu.sizes() == wg.sizes() && wd.size(0) == D && wd.size(1) == F, "titan::", op,
              ": w_gate and w_up must be [d_ff, d_model] and w_down [d_model, d_ff]; got ", wg.sizes(), ", ", wu.sizes(), ", ",
              wd.sizes(), " for d_model=", D);
  TORCH_CHECK(D > 0 && F > 0 && D % 8 == 0 && F % 8 == 0, "titan::", op, ": d_model=", D, " and d_ff=", F,
              " must be multiples of 8");
  dim32(D, op, "x's features"), dim32(F, op, "hidden features");
  return {dense16(x), dense16(wg), dense16(wu), dense16(wd), x.size(0), D, F,
          x.scalar_type() == at::kHalf ? LBK_FP16 : LBK_BF16, act == "gelu" ? LBK_GELU : LBK_SILU};
}

using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;

Four gated_fwd_impl(const Tensor& x_, const Tensor& wg, const Tensor& wu, const Tensor& wd, c10::string_view act,
                    bool add_residual, bool train, const char* op) {
  check_gpu(x_, op, "x");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x_.device());
  const Gated a = make_gated(x_, wg, wu, wd, act, op);
  Tensor out = at::empty({a.N, a.D}, a.x.options()), h, g, u;
  if (train) {
    h = at::empty({a.N, a.F}, a.x.options());
    g = at::empty({a.N, 3 * a.F}, a.x.options().dtype(at::kByte));
    u = at::empty({a.N, 3 * a.F}, g.options());
  }
  const size_t wsb = lbk_gated_fwd_workspace_bytes(a.N, (int32_t)a.D, (int32_t)a.F, train ? 1 : 0);
  Tensor ws = wsb ? workspace(wsb, a.x) : Tensor();
  const int st = lbk_gated_fwd(a.dt, a.act, a.x.data_ptr(), a.N, (int32_t)a.D, (int32_t)a.F, a.wg.data_ptr(), a.wu.data_ptr(),
                               a.wd.data_ptr(), add_residual ? 1 : 0, out.data_ptr(), train ? h.data_ptr() : nullptr,
                               train ? g.data_ptr<uint8_t>() : nullptr, train ? u.data_ptr<uint8_t>() : nullptr, wsb ? ws.data_ptr() : nullptr,
                               wsb, cur_stream(a.x));
  TORCH_CHECK(st == LBK_OK, "titan::", op, ": ", lbk_status_string(st), " (status ", st, ")");
  return {out, h, g, u};
}

Tensor gated_fwd(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, c10::string_view act, bool add_residual) {
  return std::get<0>(gated_fwd_impl(x, wg, wu, wd, act, add_residual, false, "gated_ffn_fwd"));
}

// (out, h, u act'(g), act(g)), the factors in 24 bits (include/lbk.h)
Four gated_fwd_train(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, c10::string_view act,
                     bool add_residual) {
  return gated_fwd_impl(x, wg, wu, wd, act, add_residual, true, "gated_ffn_fwd_train");
}

// (dx, dw_gate, dw_up, dw_down) from gated_fwd_train's factors and h; those not wanted come back empty
Four gated_bwd(const Tensor& dy_, const Tensor& x_, const Tensor& g_, const Tensor& u_, const Tensor& h_, const Tensor& wg,
               const Tensor& wu, const Tensor& wd, bool add_residual, std::array<bool, 4> want) {
  const char* op = "gated_ffn_bwd";
  check_gpu(x_, op, "x");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x_.device());
  const Gated a = make_gated(x_, wg, wu, wd, "silu", op);     // the factors hold the activation
  const std::pair<const Tensor*, const char*> ts[] = {{&dy_, "grad_out"}, {&g_, "gate_factor"}, {&u_, "up_factor"}, {&h_, "h"}};
  for (const auto& [t, name] : ts) {
    check_with(*t, x_, op, name);
    const bool factor = t == &g_ || t == &u_;
    const auto type = factor ? at::kByte : x_.scalar_type();
    const int64_t cols = factor ? 3 * a.F : t == &dy_ ? a.D : a.F;
    TORCH_CHECK(t->scalar_type() == type && t->dim() == 2 && t->size(0) == a.N && t->size(1) == cols, "titan::", op, ": ", name,
                " must be ", type, " [", a.N, ", ", cols, "], got ", t->scalar_type(), " ", t->sizes());
  }
  const Tensor dy = dense16(dy_), g = dense16(g_), u = dense16(u_), h = dense16(h_);
  Tensor r[4];
  const Tensor* like[] = {&a.x, &a.wg, &a.wu, &a.wd};
  void* p[4];
  for (int k = 0; k < 4; ++k) {
    r[k] = want[k] ? at::empty(like[k]->sizes(), a.x.options()) : at::empty({0}, a.x.options());
    p[k] = want[k] ? r[k].data_ptr() : nullptr;
  }
  const size_t wsb = lbk_gated_bwd_workspace_bytes(a.N, (int32_t)a.D, (int32_t)a.F);
  Tensor ws = workspace(wsb, a.x);
  LBK_CALL("gated_ffn_bwd",
           lbk_gated_bwd(a.dt, dy.data_ptr(), a.x.data_ptr(), g.data_ptr<uint8_t>(), u.data_ptr<uint8_t>(), h.data_ptr(), a.N, (int32_t)a.D,
                         (int32_t)a.F, a.wg.data_ptr(), a.wu.data_ptr(), a.wd.data_ptr(), add_residual ? 1 : 0, p[0], p[1],
                         p[2], p[3], ws.data_ptr(), wsb, cur_stream(a.x)));
  return {r[0], r[1], r[2], r[3]};
}

Four call_gated_fwd_train(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, c10::string_view act,
                          bool add_residual) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("titan::gated_ffn_fwd_train", "")
                             .typed<decltype(gated_fwd_train)>();
  return op.call(x, wg, wu, wd, act, add_residual);
}

Four call_gated_bwd(const Tensor& dy, const Tensor& x, const Tensor& g, const Tensor& u, const Tensor& h, const Tensor& wg,
                    const Tensor& wu, const Tensor& wd, bool add_residual, std::array<bool, 4> want) {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("titan::gated_ffn_bwd", "").typed<decltype(gated_bwd)>();
  return op.call(dy, x, g, u, h, wg, wu, wd, add_residual, want);
}

struct GatedTrain : public torch::autograd::Function<GatedTrain> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu,
                        const Tensor& wd, c10::string_view act, bool add_residual) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, h, g, u] = call_gated_fwd_train(x, wg, wu, wd, act, add_residual);
    ctx->save_for_backward({x, g, u, h, wg, wu, wd});
    ctx->saved_data["res"] = add_residual;
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list r(6);
    if (!grads[0].defined()) return r;
    const auto s = ctx->get_saved_variables();
    std::array<bool, 4> want;
    for (int k = 0; k < 4; ++k) want[k] = ctx->needs_input_grad(k);
    auto d = call_gated_bwd(grads[0].to(s[0].scalar_type()), s[0], s[1], s[2], s[3], s[4], s[5], s[6],
                            ctx->saved_data["res"].toBool(), want);
    if (want[0]) r[0] = std::get<0>(d);
    if (want[1]) r[1] = std::get<1>(d);
    if (want[2]) r[2] = std::get<2>(d);
    if (want[3]) r[3] = std::get<3>(d);
    return r;
  }
};

Tensor gated_train(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, c10::string_view act,
                   bool add_residual) {
  return std::get<0>(call_gated_fwd_train(x, wg, wu, wd, act, add_residual));
}
Tensor gated_train_autograd(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, c10::string_view act,
                            bool add_residual) {
  return GatedTrain::apply(x, wg, wu, wd, act, add_residual);
}

// for the shape functions: the operators' results are contiguous, whatever x's strides
Tensor rows_like(const Tensor& x) { return at::empty(x.sizes(), x.options()); }

}  // namespace

TORCH_LIBRARY_FRAGMENT(titan, m) {
  m.def("mx_quantize(Tensor x) -> (Tensor, Tensor)");
  m.def("mx_dequantize(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
  m.def("mx_quantize_tiles(Tensor values) -> (Tensor, Tensor)");
  m.def("mx_dequantize_tiles(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
  m.def("block_ell_matmul_mx(Tensor x, Tensor codes, Tensor scales, Tensor col_indices, Tensor? bias=None) -> Tensor");
  m.def("block_ell_swiglu_fwd_mx(Tensor x, Tensor c_gate, Tensor s_gate, Tensor ci_gate, Tensor? b_gate, "
        "Tensor c_up, Tensor s_up, Tensor ci_up, Tensor? b_up, Tensor c_down, Tensor s_down, Tensor ci_down, "
        "Tensor? b_down, bool add_residual) -> Tensor");
  m.def("gated_ffn_fwd(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, str activation, bool add_residual) -> Tensor");
  m.def("gated_ffn_fwd_train(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, str activation, bool add_residual) "
        "-> (Tensor, Tensor, Tensor, Tensor)");
  m.def("gated_ffn_bwd(Tensor grad_out, Tensor x, Tensor gate_factor, Tensor up_factor, Tensor h, Tensor w_gate, "
        "Tensor w_up, Tensor w_down, bool add_residual, bool[4] want) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("gated_ffn_train(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, str activation, bool add_residual) -> Tensor");
}

TORCH_LIBRARY_IMPL(titan, CUDA, m) {
  m.impl("mx_quantize", &mx_quantize);
  m.impl("mx_dequantize", &mx_dequantize);
  m.impl("mx_quantize_tiles", &mx_quantize_tiles);
  m.impl("mx_dequantize_tiles", &mx_dequantize_tiles);
  m.impl("block_ell_matmul_mx", &matmul_mx);
  m.impl("block_ell_swiglu_fwd_mx", &swiglu_mx);
  m.impl("gated_ffn_fwd", &gated_fwd);
  m.impl("gated_ffn_fwd_train", &gated_fwd_train);
  m.impl("gated_ffn_bwd", &gated_bwd);
  m.impl("gated_ffn_train", &gated_train);
}

TORCH_LIBRARY_IMPL(titan, Autograd, m) {
  m.impl("gated_ffn_train", &gated_train_autograd);
  for (const char* name : {"mx_quantize", "mx_dequantize", "mx_quantize_tiles", "mx_dequantize_tiles", "block_ell_matmul_mx",
                           "block_ell_swiglu_fwd_mx", "gated_ffn_fwd", "gated_ffn_fwd_train", "gated_ffn_bwd"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}

TORCH_LIBRARY_IMPL(titan, Meta, m) {
  m.impl("mx_quantize", [](const Tensor& x) {
    dim32(x.size(1), "mx_quantize", "x's features");
    const auto o = x.options().dtype(at::kByte);
    return std::make_tuple(at::empty({x.size(0), x.size(1) / 2}, o), at::empty({x.size(0), x.size(1) / 32}, o));
  });
  m.impl("mx_dequantize", [](const Tensor& c, const Tensor&, at::ScalarType t) {
    return at::empty({c.size(0), dim32(2 * c.size(1), "mx_dequantize", "features")}, c.options().dtype(t));
  });
  m.impl("mx_quantize_tiles", [](const Tensor& v) {
    check_slots(v, "mx_quantize_tiles");
    const auto o = v.options().dtype(at::kByte);
    return std::make_tuple(at::empty({v.size(0), v.size(1), v.size(2), v.size(2) / 2}, o),
                           at::empty({v.size(0), v.size(1), v.size(2), v.size(2) / 32}, o));
  });
  m.impl("mx_dequantize_tiles", [](const Tensor& c, const Tensor&, at::ScalarType t) {
    check_slots(c, "mx_dequantize_tiles");
    return at::empty({c.size(0), c.size(1), c.size(2), c.size(2)}, c.options().dtype(t));
  });
  m.impl("block_ell_matmul_mx", [](const Tensor& x, const Tensor& c, const Tensor&, const Tensor&, const OptTensor&) {
    dim32(x.size(1), "block_ell_matmul_mx", "x's features");
    check_slots(c, "block_ell_matmul_mx");
    return at::empty({x.size(0), c.size(0) * c.size(2)}, x.options());
  });
  m.impl("block_ell_swiglu_fwd_mx",
         [](const Tensor& x, const Tensor& cg, const Tensor&, const Tensor&, const OptTensor&, const Tensor& cu, const Tensor&,
            const Tensor&, const OptTensor&, const Tensor& cd, const Tensor&, const Tensor&, const OptTensor&, bool) {
           dim32(x.size(1), "block_ell_swiglu_fwd_mx", "x's features");
           for (const Tensor& c : {cg, cu, cd}) check_slots(c, "block_ell_swiglu_fwd_mx");
           return rows_like(x);
         });
  auto gated_dims = [](const Tensor& x, const Tensor& wg, const char* op) {
    dim32(x.size(1), op, "x's features");
    dim32(wg.size(0), op, "hidden features");
  };
  auto like_x = [gated_dims](const Tensor& x, const Tensor& wg, const Tensor&, const Tensor&, c10::string_view, bool) {
    gated_dims(x, wg, "gated_ffn_fwd");
    return rows_like(x);
  };
  m.impl("gated_ffn_fwd", like_x);
  m.impl("gated_ffn_train", like_x);
  m.impl("gated_ffn_fwd_train", [](const Tensor& x, const Tensor& wg, const Tensor&, const Tensor&, c10::string_view, bool) {
    auto factor = [&]() { return at::empty({x.size(0), 3 * wg.size(0)}, x.options().dtype(at::kByte)); };
    return std::make_tuple(rows_like(x), at::empty({x.size(0), wg.size(0)}, x.options()), factor(), factor());
  });
  m.impl("gated_ffn_bwd", [](const Tensor&, const Tensor& x, const Tensor&, const Tensor&, const Tensor&, const Tensor& wg,
                             const Tensor& wu, const Tensor& wd, bool, std::array<bool, 4> want) {
    auto d = [&](int k, const Tensor& t) { return want[k] ? at::empty(t.sizes(), x.options()) : at::empty({0}, x.options()); };
    return std::make_tuple(d(0, x), d(1, wg), d(2, wu), d(3, wd));
  });
}
