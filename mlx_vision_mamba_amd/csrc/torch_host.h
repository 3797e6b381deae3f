// What the parts of the C++ host path share: error types, checks and small
// helpers over torch and the C ABI.  Part of torch_ext.cpp's one translation
// unit.
#pragma once

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>
#include <initializer_list>
#include <string>
#include <vector>

#include "mvm_scan.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ----------------------------------------------------------------- errors

// a negative status of the library; becomes _lib.ScanError in Python
struct StatusError : std::runtime_error {
  int64_t code;
  explicit StatusError(int64_t c)
      : std::runtime_error("libmvm_scan error " + std::to_string(c) + ": " + mvm_last_error()), code(c) {}
};

int64_t check(int64_t rc) {
  if (rc < 0) throw StatusError(rc);
  return rc;
}

[[noreturn]] void bad_value(const std::string& msg) { throw py::value_error(msg); }

std::string shape_str(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

// sets the Python error that stands for e (with the GIL held)
void set_scan_error(const StatusError& e) {
  const std::string msg = e.what();
  const py::object cls = py::module_::import("mlx_vision_mamba_amd._lib").attr("ScanError");
  const auto cut = msg.find(": ");
  const py::object exc = cls(e.code, msg.substr(cut == std::string::npos ? 0 : cut + 2));
  PyErr_SetObject(cls.ptr(), exc.ptr());
}

// Runs f with torch's exception translation, and StatusError as ScanError
template <typename F>
auto guarded(F&& f) -> decltype(f()) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const StatusError& e) {
    set_scan_error(e);
    throw py::error_already_set();
  }
  END_HANDLE_TH_ERRORS_PYBIND
}

// Runs a Function's backward: the autograd engine carries its exceptions from
// its own threads to the caller's, but hands a C++ one over as RuntimeError.
// Library refusals and ValueErrors travel as the Python exceptions they are.
template <typename F>
variable_list in_backward(F&& f) {
  python_error err;
  try {
    return f();
  } catch (const StatusError& e) {
    py::gil_scoped_acquire gil;
    set_scan_error(e);
    err.persist();
  } catch (const py::builtin_exception& e) {
    py::gil_scoped_acquire gil;
    e.set_error();
    err.persist();
  }
  throw python_error(std::move(err));
}

// ---------------------------------------------------------------- helpers

const float* fp(const Tensor& t) { return t.defined() ? static_cast<const float*>(t.const_data_ptr()) : nullptr; }
float* fpm(const Tensor& t) { return t.defined() ? static_cast<float*>(t.mutable_data_ptr()) : nullptr; }

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

Tensor empty_like_opts(at::IntArrayRef sizes, const Tensor& like, at::ScalarType dt = at::kFloat) {
  return at::empty(sizes, like.options().dtype(dt).requires_grad(false));
}

Tensor workspace(int64_t nbytes, const Tensor& like) {
  return empty_like_opts({std::max<int64_t>(nbytes, 1)}, like, at::kByte);
}

void check_device(std::initializer_list<const Tensor*> ts) {
  const auto dev = (*ts.begin())->device();
  TORCH_CHECK(dev.is_cuda(), "mlx_vision_mamba_amd scans run only on the GPU (HIP); got tensors on ", dev,
              ". There is no CPU fallback.");
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->defined() || t->device() == dev, "all scan tensors must be on ", dev, "; got one on ",
                t->device());
}

// true when no two elements of t share memory: ordered by stride, each
// dimension's stride clears the span of the smaller ones
bool no_overlap(const Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> v;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) != 1) v.emplace_back(t.stride(i), t.size(i));
  std::sort(v.begin(), v.end());
  int64_t span = 1;
  for (const auto& p : v) {
    if (p.first < span) return false;
    span = p.first * p.second;
  }
  return true;
}

bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0; }

// The gradients `out` of a Function whose backward is raw launches, as they
// leave it.  Under create_graph they would have no history, and a derivative
// through them would silently lack this Function's part: they get a node that
// raises instead, on the paths to the Function's inputs and to the incoming
// gradients.  (The gradients themselves are right and may be used.)
variable_list once_differentiable(variable_list out, const variable_list& grads, const char* what) {
  if (!at::GradMode::is_enabled()) return out;
  auto edges = torch::autograd::collect_next_edges(grads);
  if (const auto node = torch::autograd::get_current_node())
    for (const auto& e : node->next_edges())
      if (e.is_valid()) edges.push_back(e);
  const auto err = std::make_shared<torch::autograd::Error>(std::string(what) + " is not twice differentiable",
                                                            std::move(edges));
  for (Tensor& t : out)
    if (t.defined()) {
      t = t.detach();
      torch::autograd::create_gradient_edge(t, err);
    }
  return out;
}

}  // namespace
