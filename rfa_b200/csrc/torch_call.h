// Shared by the tensor-level calls (torch_ops.cpp, torch_state_space.cpp): checks, errors of the Python types, the device guard, allocation.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>
#include <string>
#include <tuple>

#include "../../include/rfa_b200.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

// The calls run without the interpreter lock (see the module's end); what touches Python objects takes it.
[[noreturn]] void raise(PyObject* type, const std::string& msg) {
  py::gil_scoped_acquire lock;
  PyErr_SetString(type, msg.c_str());
  throw py::error_already_set();
}
std::string attr_name(const Tensor& t, const char* attr) {
  py::gil_scoped_acquire lock;
  return py::str(py::cast(t).attr(attr)).cast<std::string>();
}
std::string dtype_name(const Tensor& t) { return attr_name(t, "dtype"); }
std::string shape_name(const Tensor& t) { return attr_name(t, "shape"); }

void require_cuda(const Tensor& t) {
  if (!t.is_cuda())
    raise(PyExc_RuntimeError, "rfa_b200 kernels take CUDA tensors only (there is no CPU path); got a " + t.device().str() + " tensor");
}
void* ptr(const Tensor& t) {
  require_cuda(t);
  if (!t.is_contiguous()) raise(PyExc_ValueError, "rfa_b200: tensor must be contiguous");
  return t.data_ptr();
}
void* ptr(const OptTensor& t) { return t ? ptr(*t) : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
float* fptr(const OptTensor& t) { return static_cast<float*>(ptr(t)); }
const uint8_t* bptr(const OptTensor& t) { return static_cast<const uint8_t*>(ptr(t)); }

int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kHalf) return RFA_F16;
  if (t.scalar_type() == at::kFloat) return RFA_F32;
  raise(PyExc_TypeError, "rfa_b200: unsupported dtype " + dtype_name(t) + " (fp16 and fp32 only)");
}
template <class... T>
void require_half(const T&... ts) {
  for (const Tensor* t : {&ts...})
    if (t->scalar_type() != at::kHalf) raise(PyExc_TypeError, "rfa_b200: this kernel is fp16-only, got " + dtype_name(*t));
}
// A kernel launched on x's device must not be handed another device's addresses.
void require_device(const Tensor& x, std::initializer_list<const Tensor*> others) {
  for (const Tensor* t : others)
    if (t->device() != x.device())
      raise(PyExc_RuntimeError, "rfa_b200: expected all tensors on " + x.device().str() + ", got one on " + t->device().str());
}
void require(bool ok, const std::string& msg = "") {
  if (!ok) raise(PyExc_AssertionError, msg);
}
void rank(const Tensor& t, int64_t n) {
  if (t.dim() != n) raise(PyExc_ValueError, "rfa_b200: expected a tensor of " + std::to_string(n) + " dimensions, got " + shape_name(t));
}
int64_t rows_of(const Tensor& x, int64_t H, int64_t d) {
  if (H * d == 0) raise(PyExc_ZeroDivisionError, "rfa_b200: the matrices are empty");
  return x.numel() / (H * d);
}
std::string shapes(const Tensor& a, const Tensor& b) { return "(" + shape_name(a) + ", " + shape_name(b) + ")"; }

int64_t status_error(int status, const char* what) {
  if (status == 0) {      // a bounded wait of an earlier kernel ran out: synchronise and clear, so that it is reported once
    const int code = rfa_status_peek();
    rfa_debug_status();
    raise(PyExc_RuntimeError, std::string("rfa_b200: a bounded wait inside a kernel launched before or by ") + what + " ran out (site code " +
                                  std::to_string(code) + "); results computed since are invalid");
  }
  raise(status < 0 && status != RFA_EDEVICE ? PyExc_ValueError : PyExc_RuntimeError,
        std::string(what) + " failed with status " + std::to_string(status) + ": " + rfa_last_error());
}
void check(int status, const char* what) {
  if (status != 0 || rfa_status_peek() != 0) status_error(status, what);
}

// Makes the tensor's device current for the call and, on first use of a device, switches on the status mirror.
struct Call {
  c10::cuda::CUDAGuard guard;
  rfa_stream_t stream;
  explicit Call(const Tensor& t) : guard((require_cuda(t), t.device())) {
    static std::atomic<bool> watched[64];
    const int i = t.device().index();
    stream = c10::cuda::getCurrentCUDAStream(i).stream();
    if (i >= 64 || !watched[i].load(std::memory_order_acquire)) {
      const int s = rfa_status_mirror_enable();
      if (s != 0) raise(PyExc_RuntimeError, "rfa_status_mirror_enable failed with status " + std::to_string(s) + ": " + rfa_last_error());
      watched[i].store(true, std::memory_order_release);
    }
  }
};

Tensor fresh(at::IntArrayRef shape, const Tensor& like, at::ScalarType dtype) { return at::empty(shape, like.options().dtype(dtype).requires_grad(false)); }
Tensor fresh_zeros(at::IntArrayRef shape, const Tensor& like) { return at::zeros(shape, like.options().dtype(at::kFloat).requires_grad(false)); }
Tensor fresh_like(const Tensor& t) { return fresh(t.sizes(), t, t.scalar_type()); }
Tensor f32(const Tensor& t) { return t.contiguous().to(at::kFloat); }
OptTensor f32(const OptTensor& t) { return t ? OptTensor(f32(*t)) : t; }

Tensor workspace(int64_t T, int64_t BH, int64_t K, int64_t d, const Tensor& like) {
  const int64_t n = static_cast<int64_t>(rfa_causal_workspace_bytes(T, static_cast<int>(BH), static_cast<int>(K), static_cast<int>(d)));
  return fresh({std::max<int64_t>(n, 256)}, like, at::kByte);
}

// A mask as bytes, non-zero = masked.  Booleans are taken as they are.
OptTensor mask_bytes(const OptTensor& mask, int64_t n, const Tensor& like) {
  if (!mask) return mask;
  Tensor m = mask->to(like.device()).reshape({-1});
  if (m.scalar_type() != at::kBool) m = m.ne(0);
  m = m.contiguous();
  require(m.numel() == n, "(" + std::to_string(m.numel()) + ", " + std::to_string(n) + ")");
  return m;
}

// A padding mask [B, T] (any shape that views as one).
OptTensor pad_bytes(const OptTensor& pad, int64_t B, int64_t T, const Tensor& like) {
  return pad ? mask_bytes(pad->reshape({B, T}), B * T, like) : pad;
}

}  // namespace
