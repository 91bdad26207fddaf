// torch_adapter.cpp — titan:: operators of low-rank adapters beside a shared projection, over the C ABI of liblbk.so
// (include/lbk.h).  Same conventions as torch_ops.cpp.
#include "torch_util.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

Tensor adapter_plan(const Tensor& ids_, int64_t n) {
  const char* op = "adapter_plan";
  check_gpu(ids_, op, "ids");
  TORCH_CHECK(ids_.scalar_type() == at::kInt || ids_.scalar_type() == at::kLong, "titan::", op, ": ids must be int32 or int64, got ",
              ids_.scalar_type());
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(ids_.device());
  const size_t bytes = n < 1 || n > INT32_MAX ? 0 : lbk_adapter_plan_bytes(ids_.numel(), (int32_t)n);
  TORCH_CHECK(bytes > 0, "titan::", op, ": ", ids_.numel(), " tokens and ", n, " adapters; up to 2^30 and 1 .. 4096 are taken");
  const Tensor ids = ids_.contiguous();
  Tensor plan = at::empty({(int64_t)bytes / 4}, ids.options().dtype(at::kInt));
  LBK_CALL("adapter_plan", lbk_adapter_plan(ids.data_ptr(), (int32_t)ids.element_size(), ids.numel(), (int32_t)n, plan.data_ptr(), bytes,
                                            cur_stream(ids)));
  return plan;
}

// rows as the kernels take them: features consecutive, rows and the start on 16 bytes
bool rows16(const Tensor& t) {
  return t.stride(1) == 1 && (t.size(0) < 2 || (t.stride(0) >= t.size(1) && t.stride(0) % 8 == 0)) &&
         (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}
Tensor as_rows16(const Tensor& t) {
  if (t.numel() == 0 || rows16(t)) return t;
  const Tensor c = t.contiguous();
  return rows16(c) ? c : c.clone();
}
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

Tensor dense16(const Tensor& t) {
  const Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) & 15 ? c.clone() : c;
}

// the weights, scales and plan as the kernels take them, and the C struct over them (valid while this lives)
struct Adapter {
  Tensor a, b, scales, plan;
  lbk_adapter d;
};

Adapter make_adapter(const Tensor& x, const Tensor& out, const Tensor& a, const Tensor& b, const Tensor& plan, const OptTensor& scales,
                     const char* op, const char* out_name) {
  check_gpu(x, op, "x");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "titan::", op, ": x must be bf16 or fp16, got ", x.scalar_type());
  const std::pair<const Tensor*, const char*> ts[] = {{&out, out_name}, {&a, "a"}, {&b, "b"}};
  for (const auto& [t, name] : ts) {
    check_with(*t, x, op, name);
    TORCH_CHECK(t->scalar_type() == x.scalar_type(), "titan::", op, ": ", name, " is ", t->scalar_type(), ", x is ", x.scalar_type());
  }
  TORCH_CHECK(x.dim() == 2 && out.dim() == 2 && out.size(0) == x.size(0), "titan::", op, ": x and ", out_name,
              " must be [N, in] and [N, out], got ", x.sizes(), " and ", out.sizes());
  TORCH_CHECK(a.dim() == 3 && b.dim() == 3 && a.size(0) == b.size(0) && a.size(1) == b.size(2) && a.size(2) == x.size(1) &&
                  b.size(1) == out.size(1),
              "titan::", op, ": a and b must be [n, rank, ", x.size(1), "] and [n, ", out.size(1), ", rank], got ", a.sizes(), " and ", b.sizes());
  const int64_t n = a.size(0), r = a.size(1), in = a.size(2), of = b.size(1);
  TORCH_CHECK(n >= 1 && n <= 4096 && r >= 1 && r <= 256, "titan::", op, ": ", n, " adapters of rank ", r, "; 1 .. 4096 and 1 .. 256 are taken");
  TORCH_CHECK(in >= 8 && of >= 8 && in % 8 == 0 && of % 8 == 0, "titan::", op, ": features ", in, " and ", of, " must be multiples of 8");
  check_with(plan, x, op, "plan");
  const int64_t words = (int64_t)(lbk_adapter_plan_bytes(x.size(0), (int32_t)n) / 4);
  TORCH_CHECK(words > 0, "titan::", op, ": ", x.size(0), " tokens, more than 2^30");
  TORCH_CHECK(plan.scalar_type() == at::kInt && plan.dim() == 1 && plan.size(0) == words && plan.is_contiguous(), "titan::", op,
              ": the plan is not one of ", x.size(0), " tokens and ", n, " adapters");
  Adapter r_;
  r_.a = dense16(a), r_.b = dense16(b), r_.plan = dense16(plan);
  r_.scales = opt_bias(scales, n, x, op, "scales");
  r_.d = lbk_adapter{r_.a.data_ptr(), r_.b.data_ptr(), fptr(r_.scales), r_.plan.data_ptr<int32_t>(), x.size(0), (int32_t)n, (int32_t)r,
                     dim32(in, op, "x's features"), dim32(of, op, "out's features"), x.scalar_type() == at::kHalf ? LBK_FP16 : LBK_BF16};
  return r_;
}

// adds into `out`, which may be y
void add_into(const Adapter& k, const Tensor& x_, const Tensor& y_, Tensor& out, Tensor* planes, const char* op) {
  if (x_.size(0) == 0) return;
  const Tensor x = as_rows16(x_), y = as_rows16(y_);
  if (planes) *planes = workspace(lbk_adapter_planes_bytes(&k.d), x);
  const size_t wsb = lbk_adapter_add_workspace_bytes(&k.d);
  Tensor ws = workspace(wsb, x);
  const int st = lbk_adapter_add(&k.d, x.data_ptr(), ld(x), y.data_ptr(), ld(y), out.data_ptr(), ld(out), planes ? planes->data_ptr() : nullptr,
                                 ws.data_ptr(), wsb, cur_stream(x));
  TORCH_CHECK(st == LBK_OK, "titan::", op, ": ", lbk_status_string(st), " (status ", st, ")");
}

Tensor adapter_add(const Tensor& y, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& plan, const OptTensor& scales) {
  const char* op = "adapter_add";
  check_gpu(x, op, "x");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
  const Adapter k = make_adapter(x, y, a, b, plan, scales, op, "y");
  Tensor out = at::empty(y.sizes(), y.options());
  add_into(k, x, y, out, nullptr, op);
  return out;
}

void adapter_add_(Tensor y, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& plan, const OptTensor& scales) {
  const char* op = "adapter_add_";
  check_gpu(x, op, "x");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
  const Adapter k = make_adapter(x, y, a, b, plan, scales, op, "y");
  TORCH_CHECK(y.numel() == 0 || rows16(y), "titan::", op, ": y must have consecutive features and rows on 16 bytes, got strides ", y.strides());
  if (!y.is_inference()) y.unsafeGetTensorImpl()->bump_version();
  add_into(k, x, y, y, nullptr, op);
}

// (out, planes): what the backward needs of a x
std::tuple<Tensor, Tensor> adapter_add_fwd_train(const Tensor& y, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& plan,
                                                 const OptTensor& scales) {
  const char* op = "adapter_add_fwd_train";
  check_gpu(x, op, "x");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
  const Adapter k = make_adapter(x, y, a, b, plan, scales, op, "y");
  Tensor out = at::empty(y.sizes(), y.options()), planes = at::empty({0}, y.options().dtype(at::kByte));
  add_into(k, x, y, out, &planes, op);
  return {out, planes};
}

using Three = std::tuple<Tensor, Tensor, Tensor>;

// (dx, da, db); those not wanted come back empty
Three adapter_add_bwd(const Tensor& dout_, const Tensor& x_, const Tensor& a, const Tensor& b, const Tensor& plan, const Tensor& planes_,
                      const OptTensor& scales, std::array<bool, 3> want) {
  const char* op = "adapter_add_bwd";
  check_gpu(x_, op, "x");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x_.device());
  const Adapter k = make_adapter(x_, dout_, a, b, plan, scales, op, "grad_out");
  check_with(planes_, x_, op, "planes");
  TORCH_CHECK(planes_.scalar_type() == at::kByte && (!want[2] || planes_.numel() >= (int64_t)lbk_adapter_planes_bytes(&k.d)), "titan::", op,
              ": planes are not adapter_add_fwd_train's");
  const Tensor x = as_rows16(x_), dout = as_rows16(dout_), planes = dense16(planes_);
  const Tensor* like[] = {&x_, &a, &b};
  Tensor d[3];
  void* q[3];
  for (int j = 0; j < 3; ++j) {
    d[j] = want[j] ? at::empty(like[j]->sizes(), x.options()) : at::empty({0}, x.options());
    q[j] = want[j] ? d[j].data_ptr() : nullptr;
  }
  const size_t wsb = lbk_adapter_bwd_workspace_bytes_for(&k.d, want[0], want[1], want[2]);
  Tensor ws = workspace(wsb, x);
  LBK_CALL("adapter_add_bwd", lbk_adapter_bwd(&k.d, x.data_ptr(), ld(x), dout.data_ptr(), ld(dout), want[2] ? planes.data_ptr() : nullptr, q[0],
                                              q[1], q[2], ws.data_ptr(), wsb, cur_stream(x)));
  return {d[0], d[1], d[2]};
}

std::tuple<Tensor, Tensor> call_fwd_train(const Tensor& y, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& plan, const OptTensor& scales) {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("titan::adapter_add_fwd_train", "").typed<decltype(adapter_add_fwd_train)>();
  return op.call(y, x, a, b, plan, scales);
}
Three call_bwd(const Tensor& dout, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& plan, const Tensor& planes,
               const OptTensor& scales, std::array<bool, 3> want) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("titan::adapter_add_bwd", "").typed<decltype(adapter_add_bwd)>();
  return op.call(dout, x, a, b, plan, planes, scales, want);
}

struct AdapterTrain : public torch::autograd::Function<AdapterTrain> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& plan,
                        const OptTensor& scales) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, planes] = call_fwd_train(y, x, a, b, plan, scales);
    ctx->save_for_backward({x, a, b, plan, planes, scales.has_value() ? *scales : Tensor()});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list r(6);
    if (!grads[0].defined()) return r;
    const BelowAutograd below;
    const auto s = ctx->get_saved_variables();
    const std::array<bool, 3> want = {ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->needs_input_grad(3)};
    const Tensor dout = grads[0].to(s[0].scalar_type());
    if (ctx->needs_input_grad(0)) r[0] = dout;
    if (want[0] || want[1] || want[2]) {
      auto d = call_bwd(dout, s[0], s[1], s[2], s[3], s[4], s[5].defined() ? OptTensor(s[5]) : OptTensor(), want);
      if (want[0]) r[1] = std::get<0>(d);
      if (want[1]) r[2] = std::get<1>(d);
      if (want[2]) r[3] = std::get<2>(d);
    }
    return r;
  }
};

Tensor adapter_add_autograd(const Tensor& y, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& plan, const OptTensor& scales) {
  no_tangents("adapter_add", y, x, a, b, scales);
  if (at::GradMode::is_enabled()) {
    TORCH_CHECK(!needs_grad(scales), "titan::adapter_add: scales have no gradient");
    if (y.requires_grad() || x.requires_grad() || a.requires_grad() || b.requires_grad()) return AdapterTrain::apply(y, x, a, b, plan, scales);
  }
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("titan::adapter_add", "").typed<decltype(adapter_add)>();
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(y, x, a, b, plan, scales);
}
void adapter_add_inplace_autograd(Tensor y, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& plan, const OptTensor& scales) {
  no_tangents("adapter_add_", y, x, a, b, scales);
  TORCH_CHECK(!at::GradMode::is_enabled() ||
                  !(y.requires_grad() || x.requires_grad() || a.requires_grad() || b.requires_grad() || needs_grad(scales)),
              "titan::adapter_add_ has no gradient");
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("titan::adapter_add_", "").typed<decltype(adapter_add_)>();
  at::AutoDispatchBelowADInplaceOrView below;
  op.call(y, x, a, b, plan, scales);
}

}  // namespace

#define ADAPTER_ARGS "Tensor x, Tensor a, Tensor b, Tensor plan, Tensor? scales"

TORCH_LIBRARY_FRAGMENT(titan, m) {
  m.def("adapter_plan(Tensor ids, int n_adapters) -> Tensor");
  m.def("adapter_add(Tensor y, " ADAPTER_ARGS ") -> Tensor");
  m.def("adapter_add_(Tensor(a!) y, " ADAPTER_ARGS ") -> ()");
  m.def("adapter_add_fwd_train(Tensor y, " ADAPTER_ARGS ") -> (Tensor, Tensor)");
  m.def("adapter_add_bwd(Tensor grad_out, Tensor x, Tensor a, Tensor b, Tensor plan, Tensor planes, Tensor? scales, bool[3] want) "
        "-> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(titan, CUDA, m) {
  m.impl("adapter_plan", &adapter_plan);
  m.impl("adapter_add", &adapter_add);
  m.impl("adapter_add_", &adapter_add_);
  m.impl("adapter_add_fwd_train", &adapter_add_fwd_train);
  m.impl("adapter_add_bwd", &adapter_add_bwd);
}

TORCH_LIBRARY_IMPL(titan, Autograd, m) {
  m.impl("adapter_plan", torch::CppFunction::makeFallthrough());      // whole numbers
  m.impl("adapter_add", &adapter_add_autograd);
  m.impl("adapter_add_", &adapter_add_inplace_autograd);
  for (const char* name : {"adapter_add_fwd_train", "adapter_add_bwd"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}

TORCH_LIBRARY_IMPL(titan, Meta, m) {
  m.impl("adapter_plan", [](const Tensor& ids, int64_t n) {
    const size_t bytes = n < 1 || n > INT32_MAX ? 0 : lbk_adapter_plan_bytes(ids.numel(), (int32_t)n);
    TORCH_CHECK(bytes > 0, "titan::adapter_plan: ", ids.numel(), " tokens and ", n, " adapters; up to 2^30 and 1 .. 4096 are taken");
    return at::empty({(int64_t)bytes / 4}, ids.options().dtype(at::kInt));
  });
  auto add = [](const Tensor& y, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptTensor&) {
    return at::empty(y.sizes(), y.options());
  };
  m.impl("adapter_add", add);
  m.impl("adapter_add_", [](Tensor, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptTensor&) {});
  m.impl("adapter_add_fwd_train", [add](const Tensor& y, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& plan, const OptTensor& scales) {
    lbk_adapter d{};
    d.N = x.size(0), d.n = (int32_t)a.size(0), d.rank = (int32_t)a.size(1), d.in_features = (int32_t)a.size(2);
    d.out_features = (int32_t)b.size(1), d.type = LBK_BF16;
    const int64_t bytes = x.size(0) == 0 ? 0 : std::max<int64_t>(1, (int64_t)lbk_adapter_planes_bytes(&d));
    return std::make_tuple(add(y, x, a, b, plan, scales), at::empty({bytes}, y.options().dtype(at::kByte)));
  });
  m.impl("adapter_add_bwd", [](const Tensor&, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor&, const Tensor&, const OptTensor&,
                               std::array<bool, 3> want) {
    auto d = [&](int k, const Tensor& t) { return want[k] ? at::empty(t.sizes(), x.options()) : at::empty({0}, x.options()); };
    return std::make_tuple(d(0, x), d(1, a), d(2, b));
  });
}
