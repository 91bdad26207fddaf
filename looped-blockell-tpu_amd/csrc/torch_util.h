// torch_util.h — what the operator registrations (torch_ops.cpp, torch_ffn.cpp, torch_seam.cpp, torch_adapter.cpp)
// share: the current stream, status codes as errors, argument checks, workspaces.
#pragma once

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <cstdint>
#include <vector>

#include "lbk.h"

namespace {

inline void* cur_stream(const at::Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

#define LBK_CALL(opname, expr)                                                                    \
  do {                                                                                            \
    const int _st = (expr);                                                                       \
    TORCH_CHECK(_st == LBK_OK, "titan::" opname ": ", lbk_status_string(_st), " (status ", _st, ")"); \
  } while (0)

inline const uint16_t* bf(const at::Tensor& t) { return reinterpret_cast<const uint16_t*>(t.data_ptr()); }
inline uint16_t* bfm(at::Tensor& t) { return reinterpret_cast<uint16_t*>(t.data_ptr()); }

inline void check_gpu(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda(), "titan::", op, ": ", name, " must be a GPU (HIP) tensor");
}

inline void check_with(const at::Tensor& t, const at::Tensor& x, const char* op, const char* name) {
  check_gpu(t, op, name);
  TORCH_CHECK(t.device() == x.device(), "titan::", op, ": ", name, " is on ", t.device(), ", the input on ", x.device());
}

inline int32_t elem_type(at::ScalarType t, const char* op, const char* name) {
  TORCH_CHECK(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat, "titan::", op, ": ", name,
              " must be bf16, fp16 or fp32, got ", t);
  return t == at::kBFloat16 ? LBK_BF16 : t == at::kHalf ? LBK_FP16 : LBK_FP32;
}

// a size as the C ABI's 32-bit argument
inline int32_t dim32(int64_t n, const char* op, const char* what) {
  TORCH_CHECK(n <= INT32_MAX, "titan::", op, ": ", what, " are ", n, ", more than 2^31 - 1");
  return (int32_t)n;
}

inline at::Tensor check_x2d(const at::Tensor& x, const char* op) {
  check_gpu(x, op, "x");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, "titan::", op, ": x must be bf16");
  TORCH_CHECK(x.dim() == 2, "titan::", op, ": x must be 2D [N, d_model], got ", x.sizes());
  return x.contiguous();
}

inline at::Tensor workspace(size_t bytes, const at::Tensor& like) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 1)}, like.options().dtype(at::kByte));
}

// optional fp32 bias of `n` elements on x's device (made contiguous), or undefined
inline at::Tensor opt_bias(const c10::optional<at::Tensor>& b, int64_t n, const at::Tensor& x, const char* op,
                    const char* name) {
  if (!b.has_value() || !b->defined()) return at::Tensor();
  check_gpu(*b, op, name);
  TORCH_CHECK(b->numel() == n, "titan::", op, ": ", name, " must have ", n, " elements, got ", b->numel());
  if (b->scalar_type() == at::kFloat && b->device() == x.device() && b->is_contiguous()) return *b;
  return b->to(x.device(), at::kFloat).contiguous();
}
inline bool needs_grad(const c10::optional<at::Tensor>& t) { return t.has_value() && t->defined() && t->requires_grad(); }

// Forward-mode derivatives: refused, as an operator below autograd would return its result without the tangent.
inline bool has_tangent(const at::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
inline bool has_tangent(const c10::optional<at::Tensor>& t) { return t.has_value() && has_tangent(*t); }
template <class... T>
inline void no_tangents(const char* op, const T&... operands) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(operands) || ...), "titan::", op, " has no forward-mode derivative");
}

// For a backward that calls operators: past the Autograd key, whose fallback boxes every argument, unless a graph of the
// gradients is asked for (which those operators then refuse or, having a formula, record).
struct BelowAutograd {
  c10::optional<at::AutoDispatchBelowADInplaceOrView> guard;
  BelowAutograd() {
    if (!at::GradMode::is_enabled()) guard.emplace();
  }
};

inline const float* fptr(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

}  // namespace
