// Host-side helper of the Python binding: one pass over a Python list of tensors
// that validates it against a tensor table and writes the per-call pointer and
// mode arrays the C ABI takes (yafsdp_gather_in / yafsdp_scatter_out).
//
// The same checks written in Python cost about 0.6 us per tensor (five
// interpreter-level passes); a parameter group with 1,400 tensors then spends
// longer on the host than its kernel runs.  This pass takes about 10 ns per
// tensor.  It moves no tensor data; the kernels and the C ABI stay free of torch
// types (the list calls reach the ABI through addresses that the binding passes).
// Any list it does not accept is handed back to the Python checks, which raise
// the descriptive error.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <algorithm>
#include <cstdint>
#include <utility>
#include <vector>

#include "../../include/yafsdp_hip.h"

namespace {

constexpr int kModeSkip = 0, kModeCopy = 1;
constexpr int64_t kRejected = -1000;  // let the Python checks explain

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}

// tensors: list/tuple of Tensor or None.  modes: None, or list/tuple of ints (0 skip, 1 copy, 2 add).
// numels_addr: int64[n] expected element counts.  ptrs_addr: uint64[n] out.  modes_addr: uint8[n] out.
// Returns the dtype code shared by the live tensors, -1 if every tensor is skipped, kRejected otherwise.
int64_t fill(py::handle tensors, py::handle modes, uint64_t numels_addr, uint64_t ptrs_addr, uint64_t modes_addr,
             bool want_cuda, int64_t device_index) {
  PyObject* seq = tensors.ptr();
  if (!PyList_Check(seq) && !PyTuple_Check(seq)) return kRejected;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  PyObject** items = PySequence_Fast_ITEMS(seq);
  PyObject** mode_items = nullptr;
  if (!modes.is_none()) {
    PyObject* m = modes.ptr();
    if ((!PyList_Check(m) && !PyTuple_Check(m)) || PySequence_Fast_GET_SIZE(m) != n) return kRejected;
    mode_items = PySequence_Fast_ITEMS(m);
  }
  const auto* numels = reinterpret_cast<const int64_t*>(numels_addr);
  auto* ptrs = reinterpret_cast<uint64_t*>(ptrs_addr);
  auto* out_modes = reinterpret_cast<uint8_t*>(modes_addr);
  int code = -1;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = items[i];
    int mode = kModeCopy;
    if (mode_items != nullptr) {
      const long v = PyLong_AsLong(mode_items[i]);
      if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return kRejected;
      }
      if (v < 0 || v > 2) return kRejected;
      mode = static_cast<int>(v);
    }
    if (o == Py_None) mode = kModeSkip;
    out_modes[i] = static_cast<uint8_t>(mode);
    if (mode == kModeSkip) {
      ptrs[i] = 0;
      continue;
    }
    if (!THPVariable_Check(o)) return kRejected;
    const at::Tensor& t = THPVariable_Unpack(o);
    const int c = dtype_code(t.scalar_type());
    if (c < 0 || (code >= 0 && c != code)) return kRejected;
    code = c;
    if (t.numel() != numels[i] || !t.is_contiguous()) return kRejected;
    const auto dev = t.device();
    if (want_cuda ? !(dev.is_cuda() && dev.index() == device_index) : !dev.is_cpu()) return kRejected;
    ptrs[i] = reinterpret_cast<uint64_t>(t.data_ptr());
  }
  return code;
}

// True if every tensor of the list (None entries aside) is contiguous.
bool all_contiguous(py::handle tensors) {
  PyObject* seq = tensors.ptr();
  if (!PyList_Check(seq) && !PyTuple_Check(seq)) throw py::type_error("expected a list or tuple of tensors");
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  PyObject** items = PySequence_Fast_ITEMS(seq);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = items[i];
    if (o == Py_None) continue;
    if (!THPVariable_Check(o)) throw py::type_error("expected a list or tuple of tensors");
    if (!THPVariable_Unpack(o).is_contiguous()) return false;
  }
  return true;
}

// ---- lists of tensors (yafsdp_list_norm / _clip / _scale / _adamw) ---------------------------------------------
// A plain torch.Tensor or Parameter in one of the path's dtypes on the wanted kind of device; anything else (wrapper
// subclasses among them) is left to the Python side.
inline const at::Tensor* plain_tensor(PyObject* o, bool want_cuda, int64_t& device_index) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided || t.is_neg()) return nullptr;
  const auto dev = t.device();
  if (want_cuda ? !dev.is_cuda() : !dev.is_cpu()) return nullptr;
  if (device_index == -2) device_index = dev.index();
  return dev.index() == device_index ? &t : nullptr;
}

struct ListEntries {
  std::vector<yafsdp_list_entry> entries;  // None left out
  int64_t device_index = -2;

  // False if the list is not accepted as it stands.  Elementwise and order-free passes: any dense layout will do,
  // whatever its dimension order.
  bool collect(py::handle tensors, bool want_cuda) {
    PyObject* seq = tensors.ptr();
    if (!PyList_Check(seq) && !PyTuple_Check(seq)) return false;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    PyObject** items = PySequence_Fast_ITEMS(seq);
    entries.reserve(size_t(n));
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (items[i] == Py_None) continue;
      const at::Tensor* t = plain_tensor(items[i], want_cuda, device_index);
      if (t == nullptr) return false;
      const int code = dtype_code(t->scalar_type());
      if (code < 0 || !t->is_non_overlapping_and_dense()) return false;
      entries.push_back(yafsdp_list_entry{t->numel() ? t->data_ptr() : nullptr, t->numel(), code, 0});
    }
    return !entries.empty();
  }
};

// (entries, count, device index) of a list of tensors; None if the list is not accepted as it stands.
py::object list_entries(py::handle tensors, bool want_cuda) {
  ListEntries l;
  if (!l.collect(tensors, want_cuda)) return py::none();
  return py::make_tuple(
      py::bytes(reinterpret_cast<const char*>(l.entries.data()), l.entries.size() * sizeof(yafsdp_list_entry)),
      l.entries.size(), l.device_index);
}

struct AdamwEntries {
  std::vector<yafsdp_adamw_entry> entries;  // positions without a gradient and empty ones left out
  int64_t device_index = -2;
  int grad_code = -1, out_code = 0;

  // Five parallel lists; `outs`: None for "no 16-bit copies".  False if not accepted as they stand.
  bool collect(py::handle params, py::handle grads, py::handle exp_avgs, py::handle exp_avg_sqs, py::handle outs,
               bool want_cuda) {
    const bool has_out = !outs.is_none();
    PyObject* seqs[5] = {params.ptr(), grads.ptr(), exp_avgs.ptr(), exp_avg_sqs.ptr(), outs.ptr()};
    const int lists = has_out ? 5 : 4;
    PyObject** items[5] = {};
    Py_ssize_t n = -1;
    for (int k = 0; k < lists; ++k) {
      if (!PyList_Check(seqs[k]) && !PyTuple_Check(seqs[k])) return false;
      if (n >= 0 && PySequence_Fast_GET_SIZE(seqs[k]) != n) return false;
      n = PySequence_Fast_GET_SIZE(seqs[k]);
      items[k] = PySequence_Fast_ITEMS(seqs[k]);
    }
    entries.reserve(size_t(n));
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (items[1][i] == Py_None) continue;
      const at::Tensor* t[5] = {};
      for (int k = 0; k < lists; ++k) {
        t[k] = plain_tensor(items[k][i], want_cuda, device_index);
        if (t[k] == nullptr || t[k]->numel() != t[0]->numel() || !t[k]->is_contiguous()) return false;
      }
      for (int k : {0, 2, 3})
        if (t[k]->scalar_type() != at::kFloat) return false;
      const int g = dtype_code(t[1]->scalar_type());
      if (g < 0 || (grad_code >= 0 && g != grad_code)) return false;
      grad_code = g;
      if (has_out) {
        const int o = dtype_code(t[4]->scalar_type());
        if (o <= 0 || (out_code > 0 && o != out_code)) return false;
        out_code = o;
      }
      const int64_t numel = t[0]->numel();
      if (numel == 0) continue;
      entries.push_back(yafsdp_adamw_entry{static_cast<float*>(t[0]->data_ptr()), t[1]->data_ptr(),
                                           static_cast<float*>(t[2]->data_ptr()), static_cast<float*>(t[3]->data_ptr()),
                                           has_out ? t[4]->data_ptr() : nullptr, numel});
    }
    return grad_code >= 0;
  }
};

// (entries, count, device index, gradient dtype code, 16-bit copy's dtype code or 0); None if not accepted.
py::object adamw_entries(py::handle params, py::handle grads, py::handle exp_avgs, py::handle exp_avg_sqs,
                         py::handle outs, bool want_cuda) {
  AdamwEntries l;
  if (!l.collect(params, grads, exp_avgs, exp_avg_sqs, outs, want_cuda)) return py::none();
  return py::make_tuple(
      py::bytes(reinterpret_cast<const char*>(l.entries.data()), l.entries.size() * sizeof(yafsdp_adamw_entry)),
      l.entries.size(), l.device_index, l.grad_code, l.out_code);
}

// What an in-place torch op does to its tensors' version counters (the kernels write behind autograd's back).  With
// `where` (a list of the same length) only positions that are not None there.
void bump_versions(py::handle tensors, py::handle where) {
  PyObject* seqs[2] = {tensors.ptr(), where.is_none() ? tensors.ptr() : where.ptr()};
  for (PyObject* s : seqs)
    if (!PyList_Check(s) && !PyTuple_Check(s)) throw py::type_error("expected a list or tuple of tensors");
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seqs[0]);
  if (PySequence_Fast_GET_SIZE(seqs[1]) != n) throw py::type_error("expected lists of one length");
  PyObject** items = PySequence_Fast_ITEMS(seqs[0]);
  PyObject** on = PySequence_Fast_ITEMS(seqs[1]);
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (items[i] == Py_None || on[i] == Py_None) continue;
    if (!THPVariable_Check(items[i])) throw py::type_error("expected a list or tuple of tensors");
    const at::Tensor& t = THPVariable_Unpack(items[i]);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
}

// Whether two tensors of the list share a byte (0.3 us per tensor in Python); None if the list holds anything but plain
// dense tensors.
py::object any_shared(py::handle tensors) {
  PyObject* seq = tensors.ptr();
  if (!PyList_Check(seq) && !PyTuple_Check(seq)) return py::none();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  PyObject** items = PySequence_Fast_ITEMS(seq);
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  spans.reserve(size_t(n));
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!THPVariable_CheckExact(items[i])) return py::none();
    const at::Tensor& t = THPVariable_Unpack(items[i]);
    if (t.layout() != at::kStrided || !t.is_non_overlapping_and_dense()) return py::none();
    if (t.numel() == 0) continue;
    const uintptr_t at = reinterpret_cast<uintptr_t>(t.data_ptr());
    spans.emplace_back(at, at + t.nbytes());
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i - 1].second > spans[i].first) return py::bool_(true);
  return py::bool_(false);
}

// ---- whole calls, for lists on the current device ---------------------------------------------------------------
// What the Python binding does through ctypes in 5-6 us (entries as bytes, two torch.empty, argument conversion) takes
// about 2 us here.  `fn` / `ws_fn`: addresses of the ABI's entry point and of its workspace size.
inline at::Tensor scratch(uint64_t ws_fn, int64_t count, int64_t device_index) {
  const size_t bytes = reinterpret_cast<size_t (*)(int64_t)>(ws_fn)(count);
  return at::empty({int64_t(bytes)}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, c10::DeviceIndex(device_index)));
}

// yafsdp_list_norm / yafsdp_list_clip: (status, [norm, coefficient] tensor), or None if the list is not accepted.
py::object list_norm(uint64_t fn, uint64_t ws_fn, py::handle tensors, int64_t device_index, uint64_t stream, int norm,
                     double max_norm) {
  ListEntries l;
  if (!l.collect(tensors, true) || l.device_index != device_index) return py::none();
  const int64_t count = int64_t(l.entries.size());
  const at::Tensor ws = scratch(ws_fn, count, device_index);
  at::Tensor out = at::empty({2}, ws.options().dtype(at::kFloat));
  int status;
  {
    py::gil_scoped_release release;
    status = reinterpret_cast<decltype(&yafsdp_list_norm)>(fn)(l.entries.data(), count, norm, max_norm, ws.data_ptr(),
                                                               size_t(ws.numel()), out.data_ptr<float>(),
                                                               reinterpret_cast<void*>(stream));
  }
  return py::make_tuple(status, out);
}

// yafsdp_list_adamw: its status, or None if the lists are not accepted.
py::object list_adamw(uint64_t fn, uint64_t ws_fn, py::handle params, py::handle grads, py::handle exp_avgs,
                      py::handle exp_avg_sqs, py::handle outs, int64_t device_index, uint64_t stream, double lr,
                      double beta1, double beta2, double eps, double weight_decay, int64_t step, uint64_t grad_scale,
                      int flags) {
  AdamwEntries l;
  if (!l.collect(params, grads, exp_avgs, exp_avg_sqs, outs, true) || l.device_index != device_index) return py::none();
  const int64_t count = int64_t(l.entries.size());
  at::Tensor ws;
  if (reinterpret_cast<size_t (*)(int64_t)>(ws_fn)(count) > 0) ws = scratch(ws_fn, count, device_index);
  int status;
  {
    py::gil_scoped_release release;
    status = reinterpret_cast<decltype(&yafsdp_list_adamw)>(fn)(
        l.entries.data(), count, l.grad_code, l.out_code, lr, beta1, beta2, eps, weight_decay, step,
        reinterpret_cast<const float*>(grad_scale), flags, ws.defined() ? ws.data_ptr() : nullptr,
        ws.defined() ? size_t(ws.numel()) : 0, reinterpret_cast<void*>(stream));
  }
  return py::int_(status);
}

}  // namespace

PYBIND11_MODULE(_tensorlist, m) {
  m.attr("REJECTED") = kRejected;
  m.def("fill", &fill, "validate a tensor list against a table and write its pointer / mode arrays");
  m.def("all_contiguous", &all_contiguous);
  m.def("list_entries", &list_entries, "yafsdp_list_entry array of a list of tensors");
  m.def("adamw_entries", &adamw_entries, "yafsdp_adamw_entry array of parallel lists of tensors");
  m.def("list_norm", &list_norm);
  m.def("list_adamw", &list_adamw);
  m.def("any_shared", &any_shared);
  m.def("bump_versions", &bump_versions, py::arg("tensors"), py::arg("where") = py::none());
}
