// Host-side helper of the Python binding: one pass over a Python list of tensors
// that validates it against a tensor table and writes the per-call pointer and
// mode arrays the C ABI takes (yafsdp_gather_in / yafsdp_scatter_out).
//
// The same checks written in Python cost about 0.6 us per tensor (five
// interpreter-level passes); a parameter group with 1,400 tensors then spends
// longer on the host than its kernel runs.  This pass takes about 10 ns per
// tensor.  It moves no tensor data and launches nothing; the kernels and the
// C ABI stay free of torch types.  Any list it does not accept is handed back to
// the Python checks, which raise the descriptive error.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <cstdint>
#include <string>

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

// (entries, count, device index) of a list of tensors, None entries left out; None if the list is not accepted as it
// stands.  Elementwise and order-free passes: any dense layout will do, whatever its dimension order.
py::object list_entries(py::handle tensors, bool want_cuda) {
  PyObject* seq = tensors.ptr();
  if (!PyList_Check(seq) && !PyTuple_Check(seq)) return py::none();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  PyObject** items = PySequence_Fast_ITEMS(seq);
  std::string buf(size_t(n) * sizeof(yafsdp_list_entry), '\0');
  auto* out = reinterpret_cast<yafsdp_list_entry*>(&buf[0]);
  int64_t device_index = -2, count = 0;
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (items[i] == Py_None) continue;
    const at::Tensor* t = plain_tensor(items[i], want_cuda, device_index);
    if (t == nullptr) return py::none();
    const int code = dtype_code(t->scalar_type());
    if (code < 0 || !t->is_non_overlapping_and_dense()) return py::none();
    out[count++] = yafsdp_list_entry{t->numel() ? t->data_ptr() : nullptr, t->numel(), code, 0};
  }
  if (count == 0) return py::none();
  return py::make_tuple(py::bytes(buf.data(), size_t(count) * sizeof(yafsdp_list_entry)), count, device_index);
}

// (entries, count, device index, gradient dtype code, 16-bit copy's dtype code or 0) of five parallel lists; positions
// without a gradient are left out.  `outs`: None for "no 16-bit copies".  None if not accepted as they stand.
py::object adamw_entries(py::handle params, py::handle grads, py::handle exp_avgs, py::handle exp_avg_sqs,
                         py::handle outs, bool want_cuda) {
  const bool has_out = !outs.is_none();
  PyObject* seqs[5] = {params.ptr(), grads.ptr(), exp_avgs.ptr(), exp_avg_sqs.ptr(), outs.ptr()};
  const int lists = has_out ? 5 : 4;
  PyObject** items[5] = {};
  Py_ssize_t n = -1;
  for (int k = 0; k < lists; ++k) {
    if (!PyList_Check(seqs[k]) && !PyTuple_Check(seqs[k])) return py::none();
    if (n >= 0 && PySequence_Fast_GET_SIZE(seqs[k]) != n) return py::none();
    n = PySequence_Fast_GET_SIZE(seqs[k]);
    items[k] = PySequence_Fast_ITEMS(seqs[k]);
  }
  std::string buf(size_t(n) * sizeof(yafsdp_adamw_entry), '\0');
  auto* out = reinterpret_cast<yafsdp_adamw_entry*>(&buf[0]);
  int64_t device_index = -2, count = 0;
  int grad_code = -1, out_code = 0;
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (items[1][i] == Py_None) continue;
    const at::Tensor* t[5] = {};
    for (int k = 0; k < lists; ++k) {
      t[k] = plain_tensor(items[k][i], want_cuda, device_index);
      if (t[k] == nullptr || t[k]->numel() != t[0]->numel() || !t[k]->is_contiguous()) return py::none();
    }
    for (int k : {0, 2, 3})
      if (t[k]->scalar_type() != at::kFloat) return py::none();
    const int g = dtype_code(t[1]->scalar_type());
    if (g < 0 || (grad_code >= 0 && g != grad_code)) return py::none();
    grad_code = g;
    if (has_out) {
      const int o = dtype_code(t[4]->scalar_type());
      if (o <= 0 || (out_code > 0 && o != out_code)) return py::none();
      out_code = o;
    }
    const int64_t numel = t[0]->numel();
    if (numel == 0) continue;
    out[count++] = yafsdp_adamw_entry{static_cast<float*>(t[0]->data_ptr()), t[1]->data_ptr(),
                                      static_cast<float*>(t[2]->data_ptr()), static_cast<float*>(t[3]->data_ptr()),
                                      has_out ? t[4]->data_ptr() : nullptr, numel};
  }
  if (grad_code < 0) return py::none();
  return py::make_tuple(py::bytes(buf.data(), size_t(count) * sizeof(yafsdp_adamw_entry)), count, device_index,
                        grad_code, out_code);
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

}  // namespace

PYBIND11_MODULE(_tensorlist, m) {
  m.attr("REJECTED") = kRejected;
  m.def("fill", &fill, "validate a tensor list against a table and write its pointer / mode arrays");
  m.def("all_contiguous", &all_contiguous);
  m.def("list_entries", &list_entries, "yafsdp_list_entry array of a list of tensors");
  m.def("adamw_entries", &adamw_entries, "yafsdp_adamw_entry array of parallel lists of tensors");
  m.def("bump_versions", &bump_versions, py::arg("tensors"), py::arg("where") = py::none());
}
