// What the native per-layer launches (py_torch.cpp, py_fp8.cpp) share: torch
// tensors as the kernels read them, and a step's packed words.
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>

#include <cstdint>
#include <cstring>

#include "mvattn.h"

#define FASTCALL(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL

namespace {

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MV_DTYPE_F32;
    case at::kHalf: return MV_DTYPE_F16;
    case at::kBFloat16: return MV_DTYPE_BF16;
    default: return -1;
  }
}

const at::Tensor* plain(PyObject* o) {  // a torch.Tensor, no subclass
  return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}

bool sized(const at::Tensor& t, std::initializer_list<int64_t> s) {
  return t.sizes() == at::IntArrayRef(s.begin(), s.size());
}

// [T, H, D] rows as the kernels read them: D contiguous, 16-byte aligned.
struct Rows {
  void* p;
  int64_t st, sh;
};
bool aligned_rows(const at::Tensor& t, Rows& r) {
  const int64_t eb = t.element_size();
  r = {t.data_ptr(), t.stride(0), t.stride(1)};
  return t.stride(2) == 1 && r.st * eb % 16 == 0 && r.sh * eb % 16 == 0 &&
         reinterpret_cast<uintptr_t>(r.p) % 16 == 0;
}

// The two caches of one layer: the pool layout, contiguous, of `like`'s type and device.
bool caches_ok(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& like) {
  return kc.dim() == 4 && kc.sizes() == vc.sizes() && kc.scalar_type() == like.scalar_type() &&
         vc.scalar_type() == like.scalar_type() && kc.device() == like.device() &&
         vc.device() == like.device() && kc.is_contiguous() && vc.is_contiguous();
}

PyObject* none() { Py_RETURN_NONE; }
PyObject* status(int rc) { return PyLong_FromLong(rc); }
void* address(PyObject* o) { return o == Py_None ? nullptr : PyLong_AsVoidPtr(o); }

// A step's packed words (the layouts are _hip.py's): little-endian 64-bit
// integers, a double where noted.
struct Words {
  const char* p = nullptr;
  Words(PyObject* o, Py_ssize_t count) {
    char* b;
    Py_ssize_t n;
    if (PyBytes_AsStringAndSize(o, &b, &n) == 0 && n == 8 * count) p = b;
    PyErr_Clear();
  }
  int64_t i(int k) const {
    int64_t v;
    std::memcpy(&v, p + 8 * k, 8);
    return v;
  }
  double f(int k) const {
    double v;
    std::memcpy(&v, p + 8 * k, 8);
    return v;
  }
  template <class T>
  T* ptr(int k) const { return reinterpret_cast<T*>(i(k)); }
};

}  // namespace
