// What the parts of the C++ host path share: error types, checks and small
// helpers over torch and the C ABI.  Part of torch_ext.cpp's one translation
// unit.
#pragma once

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/extension.h>

#include <algorithm>
#include <initializer_list>
#include <string>
#include <unordered_set>
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

bool is_capturing(void* stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  // (the null stream is never captured, and not to be asked while another is)
  return stream != nullptr && hipStreamIsCapturing(static_cast<hipStream_t>(stream), &status) == hipSuccess &&
         status == hipStreamCaptureStatusActive;
}

// In a Function's backward: while it is captured into a graph, what takes gradients from it, directly or through other
// nodes, must be part of the capture or join it.  A leaf's gradient accumulator, which an eager graph of the same leaf
// keeps alive, runs on the stream that it was made on; the engine draws that stream into the capture, and waits for it
// again only where the accumulator runs (backward(), not grad()).  The null stream cannot be drawn into one.  Either
// ends the process when the capture ends: refused here.
void check_captured_edges(const Tensor& like, const char* what) {
  if (!like.is_cuda() || !is_capturing(stream_of(like))) return;
  const auto node = torch::autograd::get_current_node();
  if (node == nullptr) return;
  const c10::Stream here = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(like.device().index()).unwrap();
  const auto* exec = torch::autograd::get_current_graph_task_exec_info();
  const bool accumulates = exec == nullptr || exec->empty();
  std::vector<const torch::autograd::Node*> todo{node.get()};
  std::unordered_set<const torch::autograd::Node*> seen{node.get()};
  while (!todo.empty()) {
    const auto* from = todo.back();
    todo.pop_back();
    for (const auto& edge : from->next_edges()) {
      torch::autograd::Node* next = edge.function.get();
      if (next == nullptr || !seen.insert(next).second) continue;
      bool runs = true;  // (else its gradient is handed out in front of it, or not asked for)
      if (!accumulates) {
        const auto info = exec->find(next);
        if (info == exec->end() || !info->second.should_execute()) continue;
        runs = info->second.needed_;
      }
      const auto s = next->stream();
      if (s.has_value() && *s != here && s->device() == here.device()) {
        void* const other = c10::hip::HIPStreamMasqueradingAsCUDA(*s).stream();
        const bool waited_for = accumulates || (runs && next->num_outputs() > 0);
        if (!is_capturing(other) && (other == nullptr || !waited_for))
          throw std::runtime_error(std::string("the backward of ") + what + " is captured into a graph, but an eager graph "
                                   "of its inputs is alive on another stream: delete that graph's outputs before the "
                                   "capture");
      }
      if (runs) todo.push_back(next);
    }
  }
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
