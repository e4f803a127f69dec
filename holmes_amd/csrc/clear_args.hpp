// What the Python sides of the cleartext operators share (clear_bind.cpp, window_bind.cpp): reading arguments, refusing them,
// making outputs.  Each is a module of its own, so everything here is internal to the file that includes it.
#pragma once
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "../../include/holmes_ckks.h"

namespace {

using at::ScalarType;
using at::Tensor;

int type_of(ScalarType t) {
  return t == at::kBFloat16 ? HCK_BF16 : t == at::kHalf ? HCK_F16 : t == at::kFloat ? HCK_F32 : -1;
}

[[noreturn]] void refuse(const std::string& message) {
  PyErr_SetString(PyExc_ValueError, message.c_str());
  throw python_error();
}
void need(bool condition, const char* message) {
  if (!condition) refuse(message);
}

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw torch::TypeError(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

// Nothing here has a backward pass, nor a forward one, and a result without one would pass for a constant.
void no_gradient(const Tensor& t, const char* name) {
  if (t.requires_grad() && c10::GradMode::is_enabled())
    refuse(std::string(name) + " require a gradient, which this call does not have: detach them, or call it under torch.no_grad()");
  if (t._fw_grad(/*level=*/0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    refuse(std::string(name) + " have a tangent (forward-mode derivatives), which this call does not pass on: detach them");
}

long long whole(PyObject* o) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw python_error();
  return x;
}

PyObject* wrap(Tensor t) { return THPVariable_Wrap(std::move(t)); }
PyObject* none() { return Py_NewRef(Py_None); }

// (A launch goes to the current device, whatever the stream: each call makes its tensors' device that first.)
void* stream_of(at::DeviceIndex index) { return (void*)c10::hip::getCurrentHIPStream(index).stream(); }

Tensor make(at::IntArrayRef size, ScalarType type, at::Device device) {
  return at::detail::empty_cuda(size, type, device, std::nullopt);
}

// A pool: its bytes, pages, key heads, head dimension and device, as the first five arguments.
struct Pool {
  PyObject* buf;
  int64_t pages;
  int heads, dim;
  at::Device device;
  explicit Pool(PyObject* const* a)
      : buf(a[0]), pages(whole(a[1])), heads((int)whole(a[2])), dim((int)whole(a[3])),
        device(at::kCUDA, (at::DeviceIndex)whole(a[4])) {}
  // The address of its bytes.  They are a tensor that a program can replace or resize: asked for at each call.
  void* at() const {
    const Tensor& t = tensor(buf, "the pool's buf");
    const int64_t bytes = pages * heads * (int64_t)hck_kv4_page_bytes(dim);
    need(t.scalar_type() == at::kByte && t.device() == device && t.numel() == bytes && t.is_contiguous() &&
             t.storage_offset() + bytes <= (int64_t)t.storage().nbytes(),
         "the pool's buf must be its pages' bytes, contiguous uint8 on the pool's device");
    return t.data_ptr();
  }
};

// Contiguous along axis i; of one element or none the stride says nothing.
bool dense(const Tensor& t, int i) { return t.size(i) <= 1 || t.stride(i) == 1 || t.numel() == 0; }

void count(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) throw torch::TypeError(std::to_string(n) + " arguments instead of " + std::to_string(want));
}

}  // namespace
