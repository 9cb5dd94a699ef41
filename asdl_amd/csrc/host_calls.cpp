// The usual calls of the operators with many small ones (layer norm, filtered draws, norms of all gradients) from Python's tensors to
// the C interface: arguments looked at, results allocated and the entry point called in one step.  Written in Python that takes
// longer than the kernels: 12.4 us a layer norm, 0.4 us a gradient, against 5.2 us and 0.07 us here.
//
// Every function returns None for anything out of the ordinary, a wrong argument included: asdl_amd/kernels.py then goes its own way,
// which copies, refuses and explains.  A return code of an entry point comes back as an int.  Streams are handles, devices the
// current one: the callers see to both.
#include <algorithm>
#include <cmath>
#include <vector>

#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/asdl_amd.h"

namespace {

struct Entries {
  decltype(&ak_layer_norm) layer_norm;
  decltype(&ak_layer_norm_backward) layer_norm_backward;
  decltype(&ak_layer_norm_backward_ws_bytes) layer_norm_backward_ws_bytes;
  decltype(&ak_sample_filtered) sample_filtered;
  decltype(&ak_grad_norm) grad_norm;
  decltype(&ak_clip_grad_norm) clip_grad_norm;
  decltype(&ak_grad_norm_ws_bytes) grad_norm_ws_bytes;
} entries;

// The code of an element type; -1: none of the three.
int code_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return AK_F32;
    case at::kBFloat16: return AK_BF16;
    case at::kHalf: return AK_F16;
    default: return -1;
  }
}

bool plain(const at::Tensor& t) { return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous(); }

// A tensor or None; false for another object.
bool optional(PyObject* o, at::Tensor& t) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  t = THPVariable_Unpack(o);
  return true;
}

void* address(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

at::Tensor made(at::IntArrayRef sizes, const at::Tensor& like, at::ScalarType type) { return at::empty(sizes, like.options().dtype(type).requires_grad(false)); }

PyObject* none() { Py_RETURN_NONE; }

PyObject* wrapped(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

// bind(seven addresses, in the order of Entries)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != 7) {
    PyErr_SetString(PyExc_TypeError, "bind() takes seven addresses");
    return nullptr;
  }
  void* a[7];
  for (int i = 0; i < 7; ++i) {
    a[i] = PyLong_AsVoidPtr(args[i]);
    if (a[i] == nullptr) return PyErr_Occurred() != nullptr ? nullptr : (PyErr_SetString(PyExc_ValueError, "an entry point is missing"), nullptr);
  }
  entries.layer_norm = reinterpret_cast<decltype(entries.layer_norm)>(a[0]);
  entries.layer_norm_backward = reinterpret_cast<decltype(entries.layer_norm_backward)>(a[1]);
  entries.layer_norm_backward_ws_bytes = reinterpret_cast<decltype(entries.layer_norm_backward_ws_bytes)>(a[2]);
  entries.sample_filtered = reinterpret_cast<decltype(entries.sample_filtered)>(a[3]);
  entries.grad_norm = reinterpret_cast<decltype(entries.grad_norm)>(a[4]);
  entries.clip_grad_norm = reinterpret_cast<decltype(entries.clip_grad_norm)>(a[5]);
  entries.grad_norm_ws_bytes = reinterpret_cast<decltype(entries.grad_norm_ws_bytes)>(a[6]);
  Py_RETURN_NONE;
}

// layer_norm(x, weight, bias, eps, float32 result, stream) -> (y, mean, rstd)
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  at::Tensor w, b;
  if (count != 6 || !THPVariable_Check(args[0]) || !optional(args[1], w) || !optional(args[2], b) || !PyFloat_Check(args[3])) return none();
  const at::Tensor& x = THPVariable_Unpack(args[0]);
  const int xt = plain(x) ? code_of(x) : -1;
  if (xt < 0 || x.dim() == 0 || x.size(-1) == 0) return none();
  const int64_t F = x.size(-1), rows = x.numel() / F;
  int wt = AK_F32;
  for (const at::Tensor* v : {&w, &b}) {
    if (!v->defined()) continue;
    wt = plain(*v) ? code_of(*v) : -1;
    if ((wt != AK_F32 && wt != xt) || v->numel() != F || v->device() != x.device()) return none();
  }
  if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type()) return none();
  const double eps = PyFloat_AS_DOUBLE(args[3]);
  const bool as_float = args[4] == Py_True;
  void* stream = PyLong_AsVoidPtr(args[5]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  if (!(eps >= 0)) return none();
  at::Tensor y, mean, rstd;
  int rc;
  {
    pybind11::gil_scoped_release release;
    y = made(x.sizes(), x, as_float ? at::kFloat : x.scalar_type());
    mean = made(x.sizes().slice(0, x.dim() - 1), x, at::kFloat);
    rstd = made(x.sizes().slice(0, x.dim() - 1), x, at::kFloat);
    rc = entries.layer_norm(x.data_ptr(), xt, F, address(w), address(b), wt, rows, F, static_cast<float>(eps), y.data_ptr(), as_float ? AK_F32 : xt, F,
                            mean.data_ptr<float>(), rstd.data_ptr<float>(), stream);
  }
  if (rc != AK_OK) return PyLong_FromLong(rc);
  return Py_BuildValue("(NNN)", wrapped(y), wrapped(mean), wrapped(rstd));
  END_HANDLE_TH_ERRORS
}

// layer_norm_backward(g, x, mean, rstd, weight, blocks, alpha, beta, bits of dx 1, dw 2, db 4, stream) -> (dx, dw, db)
PyObject* layer_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  at::Tensor w, blocks;
  if (count != 10 || !optional(args[4], w) || !optional(args[5], blocks) || !PyFloat_Check(args[6]) || !PyFloat_Check(args[7])) return none();
  for (int i = 0; i < 4; ++i)
    if (!THPVariable_Check(args[i])) return none();
  const at::Tensor &g = THPVariable_Unpack(args[0]), &x = THPVariable_Unpack(args[1]), &mean = THPVariable_Unpack(args[2]), &rstd = THPVariable_Unpack(args[3]);
  if (!plain(g) || !plain(x) || !plain(mean) || !plain(rstd)) return none();
  const int xt = code_of(x), gt = code_of(g);
  if (xt < 0 || (gt != xt && gt != AK_F32) || x.dim() == 0 || x.size(-1) == 0 || g.sizes() != x.sizes()) return none();
  const int64_t F = x.size(-1), rows = x.numel() / F;
  for (const at::Tensor* v : {&mean, &rstd})
    if (v->scalar_type() != at::kFloat || v->numel() != rows || v->device() != x.device()) return none();
  if (g.device() != x.device()) return none();
  int wt = AK_F32;
  if (w.defined()) {
    wt = plain(w) ? code_of(w) : -1;
    if ((wt != AK_F32 && wt != xt) || w.numel() != F || w.device() != x.device()) return none();
  }
  if (blocks.defined() && (!plain(blocks) || blocks.scalar_type() != at::kFloat || blocks.dim() != 3 || blocks.size(0) != F || blocks.size(1) != 2 ||
                           blocks.size(2) != 2 || blocks.device() != x.device()))
    return none();
  const long need = PyLong_AsLong(args[8]);
  void* stream = PyLong_AsVoidPtr(args[9]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  at::Tensor dx, dw, db, ws;
  size_t bytes = 0;
  int rc;
  {
    pybind11::gil_scoped_release release;
    const at::ScalarType weight_type = w.defined() ? w.scalar_type() : at::kFloat;
    if (need & 1) dx = made(x.sizes(), x, x.scalar_type());
    if (need & 2) dw = made({F}, x, weight_type);
    if (need & 4) db = made({F}, x, weight_type);
    if ((need & 6) != 0 || blocks.defined()) {
      bytes = entries.layer_norm_backward_ws_bytes(rows, F, blocks.defined() ? 1 : 0);
      ws = made({static_cast<int64_t>(bytes)}, x, at::kByte);      // (a graph that is captured has its own)
    }
    rc = entries.layer_norm_backward(g.data_ptr(), gt, F, x.data_ptr(), xt, F, mean.data_ptr<float>(), rstd.data_ptr<float>(), address(w), wt, rows, F,
                                     address(dx), F, address(dw), address(db), static_cast<float*>(address(blocks)),
                                     static_cast<float>(PyFloat_AS_DOUBLE(args[6])), static_cast<float>(PyFloat_AS_DOUBLE(args[7])), address(ws), bytes, stream);
  }
  if (rc != AK_OK) return PyLong_FromLong(rc);
  return Py_BuildValue("(NNN)", wrapped(dx), wrapped(dw), wrapped(db));
  END_HANDLE_TH_ERRORS
}

// A filter: None (off), a number, or a tensor of `type` with one element per row.
bool filter(PyObject* o, double off, at::ScalarType type, int64_t rows, const at::Tensor& like, double& number, at::Tensor& each) {
  number = off;
  if (o == Py_None) return true;
  if (PyFloat_Check(o)) {
    number = PyFloat_AS_DOUBLE(o);
    return number == number;
  }
  if (PyLong_Check(o)) {
    number = PyLong_AsDouble(o);
    if (PyErr_Occurred() != nullptr) PyErr_Clear(), number = NAN;
    return number == number;
  }
  if (!THPVariable_Check(o)) return false;
  each = THPVariable_Unpack(o);
  return plain(each) && each.scalar_type() == type && each.numel() == rows && each.device() == like.device();
}

// sample_filtered(logits, u, temperature, top_k, top_p, min_p, stream) -> classes
PyObject* sample_filtered(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 7 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) return none();
  const at::Tensor &x = THPVariable_Unpack(args[0]), &u = THPVariable_Unpack(args[1]);
  if (!x.defined() || !x.is_cuda() || x.layout() != at::kStrided || x.dim() == 0 || x.size(-1) == 0 || !plain(u) || u.device() != x.device()) return none();
  const int code = code_of(x);
  const int64_t n = x.size(-1), rows = x.numel() / n;
  const bool in_rows = x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= n;
  if (code < 0 || rows == 0 || !(x.is_contiguous() || in_rows) || u.numel() != rows || (u.scalar_type() != at::kFloat && u.scalar_type() != at::kDouble))
    return none();
  double t, k, p, m;
  at::Tensor ts, ks, ps, ms;
  if (!filter(args[2], 1., at::kFloat, rows, x, t, ts) || !filter(args[3], 0., at::kLong, rows, x, k, ks) || !filter(args[4], 1., at::kFloat, rows, x, p, ps) ||
      !filter(args[5], 0., at::kFloat, rows, x, m, ms) || !(t >= 0.))
    return none();
  void* stream = PyLong_AsVoidPtr(args[6]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  at::Tensor targets;
  int rc;
  {
    pybind11::gil_scoped_release release;
    targets = made(x.sizes().slice(0, x.dim() - 1), x, at::kLong);
    const int64_t top_k = k <= 0. ? 0 : k >= static_cast<double>(n) ? n : static_cast<int64_t>(k);
    rc = entries.sample_filtered(x.data_ptr(), code, rows, n, x.is_contiguous() ? n : x.stride(0), u.data_ptr(), u.scalar_type() == at::kDouble, t,
                                 static_cast<float*>(address(ts)), top_k, static_cast<int64_t*>(address(ks)), p, static_cast<float*>(address(ps)), m,
                                 static_cast<float*>(address(ms)), targets.data_ptr<int64_t>(), nullptr, stream);
  }
  if (rc != AK_OK) return PyLong_FromLong(rc);
  return wrapped(targets);
  END_HANDLE_TH_ERRORS
}

// gradient_norm(list of gradients, list of results or None, kind, max_norm, stream) -> norm; without results the norm alone
PyObject* gradient_norm(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 5 || !PyList_Check(args[0]) || !(args[1] == Py_None || PyList_Check(args[1])) || !PyFloat_Check(args[3])) return none();
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  const bool clip = args[1] != Py_None, in_place = args[1] == args[0];
  if (n == 0 || (clip && PyList_GET_SIZE(args[1]) != n)) return none();
  std::vector<int64_t> table(static_cast<size_t>(n) * 5), seen(static_cast<size_t>(n));
  at::Tensor first;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* item = PyList_GET_ITEM(args[0], i);
    if (!THPVariable_Check(item)) return none();
    const at::Tensor& g = THPVariable_Unpack(item);
    if (!g.defined() || !g.is_cuda() || g.layout() != at::kStrided) return none();
    if (i == 0) first = g;
    const int code = code_of(g);
    if (code < 0 || g.numel() == 0 || g.device() != first.device() || !g.is_non_overlapping_and_dense()) return none();
    int64_t* row = table.data() + 5 * i;
    row[0] = row[1] = reinterpret_cast<int64_t>(g.data_ptr());
    row[2] = g.numel();
    row[3] = row[4] = code;
    seen[static_cast<size_t>(i)] = row[0];
    if (!clip || in_place) continue;
    PyObject* to = PyList_GET_ITEM(args[1], i);
    if (!THPVariable_Check(to)) return none();
    const at::Tensor& out = THPVariable_Unpack(to);
    if (!out.defined() || !out.is_cuda() || out.layout() != at::kStrided || out.device() != first.device() || out.numel() != g.numel()) return none();
    const int out_code = code_of(out);
    if ((out_code != code && out_code != AK_F32) || !((g.is_contiguous() && out.is_contiguous()) || (out.sizes() == g.sizes() && out.strides() == g.strides())))
      return none();
    row[1] = reinterpret_cast<int64_t>(out.data_ptr());
    row[4] = out_code;
  }
  std::sort(seen.begin(), seen.end());
  if (std::adjacent_find(seen.begin(), seen.end()) != seen.end()) return none();          // listed twice
  const long kind = PyLong_AsLong(args[2]);
  const double max_norm = PyFloat_AS_DOUBLE(args[3]);
  void* stream = PyLong_AsVoidPtr(args[4]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  at::Tensor norm, ws;
  int rc;
  {
    pybind11::gil_scoped_release release;
    const size_t bytes = entries.grad_norm_ws_bytes(static_cast<int>(n));
    norm = made({}, first, at::kFloat);
    ws = made({static_cast<int64_t>(bytes)}, first, at::kByte);
    rc = clip ? entries.clip_grad_norm(table.data(), static_cast<int>(n), static_cast<int>(kind), max_norm, norm.data_ptr<float>(), ws.data_ptr(), bytes, stream)
              : entries.grad_norm(table.data(), static_cast<int>(n), static_cast<int>(kind), norm.data_ptr<float>(), ws.data_ptr(), bytes, stream);
  }
  if (rc != AK_OK) return PyLong_FromLong(rc);
  for (Py_ssize_t i = 0; clip && i < n; ++i) {
    const at::Tensor& changed = THPVariable_Unpack(PyList_GET_ITEM(args[1], i));
    if (!changed.is_inference()) changed.unsafeGetTensorImpl()->bump_version();       // (autograd notices what it keeps)
  }
  return wrapped(norm);
  END_HANDLE_TH_ERRORS
}

#define AK_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {AK_METHOD(bind), AK_METHOD(layer_norm), AK_METHOD(layer_norm_backward), AK_METHOD(sample_filtered), AK_METHOD(gradient_norm), {}};
PyModuleDef definition = {PyModuleDef_HEAD_INIT, "asdl_amd_host_calls", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_asdl_amd_host_calls() { return PyModule_Create(&definition); }
