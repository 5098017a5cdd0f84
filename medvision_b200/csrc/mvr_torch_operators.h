// What the host paths of the operators behind the roi modules and of an encoder's blocks share: checks of arguments, streams, gradients
// that are taken once, arguments from Python.
#pragma once
#include <Python.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/mvr.h"
#include "mvr_torch.h"

namespace {

using mvr_host::check;
using mvr_host::type_name;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

int head_code(at::ScalarType t) {
  return t == at::kFloat ? MVR_F32 : t == at::kHalf ? MVR_F16 : t == at::kBFloat16 ? MVR_BF16 : -1;
}
int index_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MVR_INDEX_F32;
    case at::kHalf: return MVR_INDEX_F16;
    case at::kDouble: return MVR_INDEX_F64;
    case at::kBFloat16: return MVR_INDEX_BF16;
    case at::kInt: return MVR_INDEX_I32;
    case at::kLong: return MVR_INDEX_I64;
    case at::kShort: return MVR_INDEX_I16;
    case at::kByte: return MVR_INDEX_U8;
    default: return -1;
  }
}

// Types and shapes are looked at before the device, so that a wrong call fails alike on every machine.
void check_cuda(const char* what, const at::Tensor& t) { TORCH_CHECK(t.is_cuda(), what, " is not implemented on CPU"); }
void check_type(const char* what, const at::Tensor& t) {
  TORCH_CHECK(head_code(t.scalar_type()) >= 0, "\"", what, "\" not implemented for '", type_name(t.scalar_type()), "'");
}
void check_like(const at::Tensor& t, const at::Tensor& like) {
  TORCH_CHECK(t.device() == like.device(), "expected all tensors to be on the same CUDA device");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), "expected scalar type torch.", type_name(like.scalar_type()), " but found torch.",
              type_name(t.scalar_type()));
}
void check_tangent(const char* what, const at::Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !torch::autograd::impl::get_autograd_meta(t) || !t._fw_grad(/*level=*/0).defined(), what,
                              " has no forward-mode derivative");
}

void* stream_of(const at::Tensor& t) { return (void*)c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
void* data_or_null(const at::Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }

// The gradients were computed without a graph of their own: asking for one (create_graph) ends in an error, not in a silent 0.
void once_differentiable(const char* what, variable_list& results, const variable_list& from) {
  if (!at::GradMode::is_enabled()) return;
  bool any = false;
  for (const at::Tensor& t : from) any |= t.defined() && t.requires_grad();
  if (!any) return;
  for (at::Tensor& r : results) {
    if (!r.defined()) continue;
    r = r.detach();
    auto node = std::make_shared<torch::autograd::Error>(std::string("the gradients of ") + what + " cannot be differentiated again",
                                                         torch::autograd::collect_next_edges(from));
    torch::autograd::set_history(r, node);
  }
}

// ---- arguments from Python ------------------------------------------------------------------------------
const at::Tensor& tensor_arg(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a Tensor, not %s", name, Py_TYPE(o)->tp_name);
    throw python_error();
  }
  return THPVariable_Unpack(o);
}
at::Tensor optional_tensor(PyObject* o, const char* name) { return o == Py_None ? at::Tensor() : tensor_arg(o, name); }

double number_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
// A whole number of 64 bits with a sign.
int64_t whole_arg(PyObject* o, const char* name) {
  PyObject* index = PyNumber_Index(o);
  if (!index) throw python_error();
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(index, &overflow);
  Py_DECREF(index);
  if (overflow != 0) {
    PyErr_Format(PyExc_ValueError, "%s must fit 64 bits", name);
    throw python_error();
  }
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

void expect(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    throw python_error();
  }
}

#define FAST(f) (PyCFunction)(void (*)(void)) f, METH_FASTCALL

}  // namespace
