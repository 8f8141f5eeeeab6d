// Shared by the calls of the operators that take fp16, bf16 and fp32 with any strides (torch_state_space.cpp, torch_attention.cpp): checks, copies where a
// kernel wants them, what autograd is told.
#pragma once

#include "torch_call.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int float_code(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return RFA_BF16;
  if (t.scalar_type() == at::kHalf) return RFA_F16;
  if (t.scalar_type() == at::kFloat) return RFA_F32;
  raise(PyExc_TypeError, "rfa_b200: unsupported dtype " + dtype_name(t) + " (fp16, bf16 and fp32 only)");
}
void same_dtype(const char* what, const Tensor& x, std::initializer_list<const Tensor*> others) {
  for (const Tensor* t : others)
    if (t->scalar_type() != x.scalar_type())
      raise(PyExc_TypeError, std::string(what) + ": expected tensors of one dtype, got " + dtype_name(x) + " and " + dtype_name(*t));
}
void need_shape(const char* what, const char* name, const Tensor& t, at::IntArrayRef shape) {
  if (t.sizes() != shape) {
    std::string want = "[";
    for (size_t i = 0; i < shape.size(); ++i) want += (i ? ", " : "") + std::to_string(shape[i]);
    raise(PyExc_AssertionError, std::string(what) + ": " + name + " is " + shape_name(t) + ", expected " + want + "]");
  }
}
void need_f32(const char* what, const char* name, const Tensor& t) {
  if (t.scalar_type() != at::kFloat) raise(PyExc_TypeError, std::string(what) + ": " + name + " must be fp32, got " + dtype_name(t));
}
// A gradient that a caller hands in: of the shape that it is the gradient of, and on its device.
void need_grad(const char* what, const char* name, const OptTensor& g, at::IntArrayRef shape, const Tensor& x) {
  if (!g) return;
  need_shape(what, name, *g, shape);
  require_device(x, {&*g});
}
// Activations are taken with any strides but along the channels.
Tensor unit_last(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// A contiguous copy where a tensor is not contiguous or, being a state that kernels take in 16-byte words, not aligned.
Tensor packed(const Tensor& t) {
  Tensor c = t.contiguous();
  return aligned(c) ? c : c.clone();
}
OptTensor packed(const OptTensor& t) { return t ? OptTensor(packed(*t)) : t; }
const void* maybe(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
void* maybe_out(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
const float* maybe_f(const OptTensor& t) { return t ? t->data_ptr<float>() : nullptr; }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor plain(const OptTensor& t) { return t ? *t : Tensor(); }
Tensor scratch(size_t bytes, const Tensor& like) { return fresh({static_cast<int64_t>(std::max<size_t>(bytes, 16))}, like, at::kByte); }
int as_int(const char* what, int64_t n) {
  if (n > INT_MAX) raise(PyExc_ValueError, std::string(what) + ": a size of " + std::to_string(n));
  return static_cast<int>(n);
}
OptTensor mask_of(const char* what, const OptTensor& mask, int64_t B, int64_t T, const Tensor& like) {
  if (!mask) return mask;
  need_shape(what, "key_padding_mask", *mask, {B, T});
  return mask_bytes(mask, B * T, like);
}
// A kernel wrote to it: autograd is to notice where an earlier graph keeps it.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
bool wants(const OptTensor& t) { return t && t->requires_grad(); }
template <class... Ts> bool records(const Ts&... ts) {      // decided in front of a node, whose own forward records nothing
  return at::GradMode::is_enabled() && (wants(OptTensor(ts)) || ...);
}
void once(const char* what) {
  if (at::GradMode::is_enabled()) raise(PyExc_RuntimeError, std::string(what) + ": the backward pass is not differentiable (create_graph)");
}

}  // namespace
