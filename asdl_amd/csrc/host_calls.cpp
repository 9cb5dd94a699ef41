// The usual calls of the operators with many small ones (layer norm, filtered draws, norms of all gradients, cross entropy of a linear
// layer, embeddings, activations in 8 bits) from Python's tensors to the C interface: arguments looked at, results allocated and the
// entry point called in one step.  Written in Python that takes longer than the kernels: 12.4 us a layer norm, 0.4 us a gradient, 8.5 us
// an embedding, against 5.2 us, 0.07 us and 5.0 us here.
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
  decltype(&ak_linear_cross_entropy) linear_cross_entropy;
  decltype(&ak_linear_cross_entropy_backward) linear_cross_entropy_backward;
  decltype(&ak_linear_cross_entropy_ws_bytes_of) linear_cross_entropy_ws_bytes_of;
  decltype(&ak_embedding) embedding;
  decltype(&ak_embedding_backward) embedding_backward;
  decltype(&ak_embedding_backward_ws_bytes) embedding_backward_ws_bytes;
  decltype(&ak_quantize_8bit) quantize_8bit;
  decltype(&ak_dequantize_8bit) dequantize_8bit;
  decltype(&ak_weight_grad_8bit) weight_grad_8bit;
  decltype(&ak_weight_grad_8bit_ws_bytes_of) weight_grad_8bit_ws_bytes_of;
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

// `count` addresses of entry points, to `entries` in order.
template <typename... Entry>
PyObject* bind_to(PyObject* const* args, Py_ssize_t count, Entry&... entry) {
  if (count != static_cast<Py_ssize_t>(sizeof...(Entry))) {
    PyErr_SetString(PyExc_TypeError, "the address of every entry point is asked for");
    return nullptr;
  }
  void* a[sizeof...(Entry)];
  for (Py_ssize_t i = 0; i < count; ++i) {
    a[i] = PyLong_AsVoidPtr(args[i]);
    if (a[i] == nullptr) return PyErr_Occurred() != nullptr ? nullptr : (PyErr_SetString(PyExc_ValueError, "an entry point is missing"), nullptr);
  }
  int i = 0;
  ((entry = reinterpret_cast<Entry>(a[i++])), ...);
  Py_RETURN_NONE;
}

// bind(seven addresses, in the order of Entries)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return bind_to(args, count, entries.layer_norm, entries.layer_norm_backward, entries.layer_norm_backward_ws_bytes, entries.sample_filtered, entries.grad_norm,
                 entries.clip_grad_norm, entries.grad_norm_ws_bytes);
}

// bind_step(the addresses behind those)
PyObject* bind_step(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return bind_to(args, count, entries.linear_cross_entropy, entries.linear_cross_entropy_backward, entries.linear_cross_entropy_ws_bytes_of, entries.embedding,
                 entries.embedding_backward, entries.embedding_backward_ws_bytes, entries.quantize_8bit, entries.dequantize_8bit, entries.weight_grad_8bit,
                 entries.weight_grad_8bit_ws_bytes_of);
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

// The operands that both passes of a linear cross entropy look at.
struct Loss {
  at::Tensor bias;
  int code, bias_code;
  int64_t rows, classes, width;
};

bool loss_operands(PyObject* const* args, Loss& l, const at::Tensor*& h, const at::Tensor*& w, const at::Tensor*& t) {
  if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !THPVariable_Check(args[2]) || !optional(args[3], l.bias)) return false;
  h = &THPVariable_Unpack(args[0]);
  w = &THPVariable_Unpack(args[1]);
  t = &THPVariable_Unpack(args[2]);
  if (!plain(*h) || !plain(*w) || !plain(*t)) return false;
  l.code = code_of(*h);
  if (l.code < 0 || w->scalar_type() != h->scalar_type() || t->scalar_type() != at::kLong || h->dim() == 0 || w->dim() != 2) return false;
  l.width = h->size(-1);
  l.classes = w->size(0);
  l.rows = t->numel();
  if (l.width == 0 || l.classes == 0 || l.rows == 0 || w->size(1) != l.width || t->sizes() != h->sizes().slice(0, h->dim() - 1)) return false;
  if (w->device() != h->device() || t->device() != h->device()) return false;
  l.bias_code = l.code;
  if (l.bias.defined()) {
    l.bias_code = plain(l.bias) ? code_of(l.bias) : -1;
    if ((l.bias_code != AK_F32 && l.bias_code != l.code) || l.bias.dim() != 1 || l.bias.size(0) != l.classes || l.bias.device() != h->device()) return false;
  }
  return true;
}

// linear_cross_entropy(h, weight, targets, bias, ignored target, code of the reduction, stream) -> (loss, lse)
PyObject* linear_cross_entropy(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  Loss l;
  const at::Tensor *h, *w, *t;
  if (count != 7 || !loss_operands(args, l, h, w, t) || !PyLong_Check(args[4])) return none();
  int overflow = 0;
  const int64_t ignore = PyLong_AsLongLongAndOverflow(args[4], &overflow);
  const long kind = PyLong_AsLong(args[5]);
  void* stream = PyLong_AsVoidPtr(args[6]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  if (overflow != 0) return none();
  at::Tensor loss, lse;
  int rc;
  {
    pybind11::gil_scoped_release release;
    loss = kind == 0 ? made(t->sizes(), *h, at::kFloat) : made({}, *h, at::kFloat);
    lse = made(t->sizes(), *h, at::kFloat);
    const size_t bytes = entries.linear_cross_entropy_ws_bytes_of(h->data_ptr(), l.code, l.width, w->data_ptr(), l.width, l.bias.defined() ? l.bias_code : -1, l.rows,
                                                                  l.classes, l.width, 0);
    at::Tensor ws = made({static_cast<int64_t>(bytes)}, *h, at::kByte);
    rc = entries.linear_cross_entropy(h->data_ptr(), l.code, l.width, w->data_ptr(), l.width, address(l.bias), l.bias_code, t->data_ptr<int64_t>(), l.rows,
                                      l.classes, l.width, ignore, static_cast<int>(kind), loss.data_ptr<float>(), lse.data_ptr<float>(), ws.data_ptr(), bytes,
                                      stream);
  }
  if (rc != AK_OK) return PyLong_FromLong(rc);
  return Py_BuildValue("(NN)", wrapped(loss), wrapped(lse));
  END_HANDLE_TH_ERRORS
}

// linear_cross_entropy_backward(h, weight, targets, bias, ignored target, code of the reduction, g, lse, bits of dh 1, dw 2, db 4, stream)
//   -> (dh, dw, db)
PyObject* linear_cross_entropy_backward(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  Loss l;
  const at::Tensor *h, *w, *t;
  if (count != 10 || !loss_operands(args, l, h, w, t) || !PyLong_Check(args[4]) || !THPVariable_Check(args[6]) || !THPVariable_Check(args[7])) return none();
  const at::Tensor &g = THPVariable_Unpack(args[6]), &lse = THPVariable_Unpack(args[7]);
  int overflow = 0;
  const int64_t ignore = PyLong_AsLongLongAndOverflow(args[4], &overflow);
  const long kind = PyLong_AsLong(args[5]), need = PyLong_AsLong(args[8]);
  void* stream = PyLong_AsVoidPtr(args[9]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  if (overflow != 0 || !plain(g) || !plain(lse) || g.scalar_type() != at::kFloat || lse.scalar_type() != at::kFloat || lse.sizes() != t->sizes() ||
      (kind == 0 ? g.sizes() != t->sizes() : g.dim() != 0) || g.device() != h->device() || lse.device() != h->device())
    return none();
  at::Tensor dh, dw, db;
  int rc = AK_OK;
  {
    pybind11::gil_scoped_release release;
    if (need & 1) dh = made(h->sizes(), *h, h->scalar_type());
    if (need & 2) dw = made(w->sizes(), *h, h->scalar_type());
    if ((need & 4) && l.bias.defined()) db = made(l.bias.sizes(), *h, l.bias.scalar_type());
    if (dh.defined() || dw.defined() || db.defined()) {
      const size_t bytes = entries.linear_cross_entropy_ws_bytes_of(h->data_ptr(), l.code, l.width, w->data_ptr(), l.width, l.bias.defined() ? l.bias_code : -1,
                                                                    l.rows, l.classes, l.width, (dh.defined() ? 1 : 0) | (dw.defined() ? 2 : 0) | (db.defined() ? 4 : 0));
      at::Tensor ws = made({static_cast<int64_t>(bytes)}, *h, at::kByte);
      rc = entries.linear_cross_entropy_backward(g.data_ptr<float>(), h->data_ptr(), l.code, l.width, w->data_ptr(), l.width, address(l.bias), l.bias_code,
                                                 t->data_ptr<int64_t>(), lse.data_ptr<float>(), l.rows, l.classes, l.width, ignore, static_cast<int>(kind),
                                                 address(dh), address(dw), address(db), ws.data_ptr(), bytes, stream);
    }
  }
  if (rc != AK_OK) return PyLong_FromLong(rc);
  return Py_BuildValue("(NNN)", wrapped(dh), wrapped(dw), wrapped(db));
  END_HANDLE_TH_ERRORS
}

int token_code(const at::Tensor& t) {
  return t.scalar_type() == at::kLong ? AK_I64 : t.scalar_type() == at::kInt ? AK_I32 : -1;
}

// embedding(tokens, weight, scale, float32 result, stream) -> rows
PyObject* embedding(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 5 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !PyFloat_Check(args[2])) return none();
  const at::Tensor &t = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]);
  if (!plain(t) || !plain(w) || w.dim() != 2 || w.size(1) == 0 || t.device() != w.device()) return none();
  const int code = code_of(w), tokens = token_code(t);
  if (code < 0 || tokens < 0) return none();
  const bool as_float = args[3] == Py_True;
  void* stream = PyLong_AsVoidPtr(args[4]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  at::Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release release;
    std::vector<int64_t> sizes(t.sizes().begin(), t.sizes().end());
    sizes.push_back(w.size(1));
    out = made(sizes, w, as_float ? at::kFloat : w.scalar_type());
    rc = entries.embedding(t.data_ptr(), tokens, t.numel(), w.data_ptr(), code, w.size(1), w.size(0), w.size(1), static_cast<float>(PyFloat_AS_DOUBLE(args[2])),
                           out.data_ptr(), as_float ? AK_F32 : code, stream);
  }
  if (rc != AK_OK) return PyLong_FromLong(rc);
  return wrapped(out);
  END_HANDLE_TH_ERRORS
}

// embedding_backward(g, tokens, rows of the table, scale, padding or -1, stream) -> gradient of the type of g
PyObject* embedding_backward(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 6 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !PyLong_Check(args[2]) || !PyFloat_Check(args[3]) || !PyLong_Check(args[4]))
    return none();
  const at::Tensor &g = THPVariable_Unpack(args[0]), &t = THPVariable_Unpack(args[1]);
  if (!plain(g) || !plain(t) || g.dim() == 0 || g.size(-1) == 0 || t.device() != g.device() || g.sizes().slice(0, g.dim() - 1) != t.sizes()) return none();
  const int code = code_of(g), tokens = token_code(t);
  const int64_t rows = PyLong_AsLongLong(args[2]), padding = PyLong_AsLongLong(args[4]), D = g.size(-1);
  void* stream = PyLong_AsVoidPtr(args[5]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  if (code < 0 || tokens < 0 || rows <= 0) return none();
  at::Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release release;
    out = made({rows, D}, g, g.scalar_type());
    const size_t bytes = entries.embedding_backward_ws_bytes(t.numel(), rows, D);
    at::Tensor ws = made({static_cast<int64_t>(bytes)}, g, at::kByte);
    rc = entries.embedding_backward(g.data_ptr(), code, D, t.data_ptr(), tokens, t.numel(), rows, D, static_cast<float>(PyFloat_AS_DOUBLE(args[3])), padding,
                                    0.f, out.data_ptr(), code, D, ws.data_ptr(), bytes, stream);
  }
  if (rc != AK_OK) return PyLong_FromLong(rc);
  return wrapped(out);
  END_HANDLE_TH_ERRORS
}

constexpr int64_t kKeepBlock = 128;        // features that share an exponent

// quantize_8bit(x, code of the GELU or -1, stream) -> (y or None, codes, exponents)
PyObject* quantize_8bit(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 3 || !THPVariable_Check(args[0])) return none();
  const at::Tensor& x = THPVariable_Unpack(args[0]);
  const int code = plain(x) ? code_of(x) : -1;
  const long gelu = PyLong_AsLong(args[1]);
  void* stream = PyLong_AsVoidPtr(args[2]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  if (code < 0 || x.dim() == 0 || x.size(-1) == 0) return none();
  at::Tensor y, codes, exponents;
  int rc;
  {
    pybind11::gil_scoped_release release;
    const int64_t F = x.size(-1);
    std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = (F + kKeepBlock - 1) / kKeepBlock;
    codes = made(x.sizes(), x, at::kFloat8_e4m3fn);
    exponents = made(sizes, x, at::kChar);
    if (gelu >= 0) y = made(x.sizes(), x, x.scalar_type());
    rc = entries.quantize_8bit(x.data_ptr(), code, F, x.numel() / F, F, static_cast<int>(gelu), address(y), static_cast<uint8_t*>(codes.data_ptr()),
                               static_cast<int8_t*>(exponents.data_ptr()), stream);
  }
  if (rc != AK_OK) return PyLong_FromLong(rc);
  return Py_BuildValue("(NNN)", wrapped(y), wrapped(codes), wrapped(exponents));
  END_HANDLE_TH_ERRORS
}

// Codes and exponents as quantize_8bit() makes them.
bool kept(PyObject* const* args, const at::Tensor*& codes, const at::Tensor*& exponents) {
  if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) return false;
  codes = &THPVariable_Unpack(args[0]);
  exponents = &THPVariable_Unpack(args[1]);
  if (!plain(*codes) || !plain(*exponents) || codes->scalar_type() != at::kFloat8_e4m3fn || exponents->scalar_type() != at::kChar || codes->dim() == 0 ||
      exponents->dim() != codes->dim() || codes->size(-1) == 0 || exponents->size(-1) != (codes->size(-1) + kKeepBlock - 1) / kKeepBlock)
    return false;
  return codes->sizes().slice(0, codes->dim() - 1) == exponents->sizes().slice(0, codes->dim() - 1) && codes->device() == exponents->device();
}

constexpr at::ScalarType kTypes[5] = {at::kFloat, at::kBFloat16, at::kFloat, at::kFloat, at::kHalf};      // by code

// dequantize_8bit(codes, exponents, code of the GELU or -1, g or None, code of the type, stream) -> values, or the GELU's gradient
PyObject* dequantize_8bit(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  const at::Tensor *codes, *exponents;
  at::Tensor g;
  if (count != 6 || !kept(args, codes, exponents) || !optional(args[3], g)) return none();
  const long gelu = PyLong_AsLong(args[2]), type = PyLong_AsLong(args[4]);
  void* stream = PyLong_AsVoidPtr(args[5]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  if ((type != AK_F32 && type != AK_BF16 && type != AK_F16) || g.defined() != (gelu >= 0)) return none();
  if (g.defined() && (!plain(g) || code_of(g) != type || g.sizes() != codes->sizes() || g.device() != codes->device())) return none();
  at::Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release release;
    const int64_t F = codes->size(-1);
    out = made(codes->sizes(), *codes, kTypes[type]);
    rc = entries.dequantize_8bit(static_cast<const uint8_t*>(codes->data_ptr()), static_cast<const int8_t*>(exponents->data_ptr()), codes->numel() / F, F,
                                 static_cast<int>(gelu), address(g), F, out.data_ptr(), static_cast<int>(type), stream);
  }
  if (rc != AK_OK) return PyLong_FromLong(rc);
  return wrapped(out);
  END_HANDLE_TH_ERRORS
}

// weight_grad_8bit(codes, exponents, g, bits of dw 1, db 2, code of their type, stream) -> (dw, db)
PyObject* weight_grad_8bit(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  const at::Tensor *codes, *exponents;
  if (count != 6 || !kept(args, codes, exponents) || !THPVariable_Check(args[2])) return none();
  const at::Tensor& g = THPVariable_Unpack(args[2]);
  const long need = PyLong_AsLong(args[3]), type = PyLong_AsLong(args[4]);
  void* stream = PyLong_AsVoidPtr(args[5]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  const int code = plain(g) ? code_of(g) : -1;
  if (code < 0 || (type != AK_F32 && type != AK_BF16 && type != AK_F16) || g.dim() == 0 || g.numel() == 0 || need == 0 ||
      g.sizes().slice(0, g.dim() - 1) != codes->sizes().slice(0, codes->dim() - 1) || g.device() != codes->device())
    return none();
  at::Tensor dw, db;
  int rc;
  {
    pybind11::gil_scoped_release release;
    const int64_t F = codes->size(-1), out = g.size(-1), rows = g.numel() / out;
    if (need & 1) dw = made({out, F}, g, kTypes[type]);
    if (need & 2) db = made({out}, g, kTypes[type]);
    const size_t bytes = entries.weight_grad_8bit_ws_bytes_of(g.data_ptr(), code, out, rows, F, out, static_cast<int>(need));
    at::Tensor ws = made({static_cast<int64_t>(bytes)}, g, at::kByte);
    rc = entries.weight_grad_8bit(g.data_ptr(), code, out, static_cast<const uint8_t*>(codes->data_ptr()), static_cast<const int8_t*>(exponents->data_ptr()), rows,
                                  F, out, address(dw), address(db), static_cast<int>(type), ws.data_ptr(), bytes, stream);
  }
  if (rc != AK_OK) return PyLong_FromLong(rc);
  return Py_BuildValue("(NN)", wrapped(dw), wrapped(db));
  END_HANDLE_TH_ERRORS
}

#define AK_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {AK_METHOD(bind), AK_METHOD(bind_step), AK_METHOD(layer_norm), AK_METHOD(layer_norm_backward), AK_METHOD(sample_filtered), AK_METHOD(gradient_norm),
                         AK_METHOD(linear_cross_entropy), AK_METHOD(linear_cross_entropy_backward), AK_METHOD(embedding), AK_METHOD(embedding_backward),
                         AK_METHOD(quantize_8bit), AK_METHOD(dequantize_8bit), AK_METHOD(weight_grad_8bit), {}};
PyModuleDef definition = {PyModuleDef_HEAD_INIT, "asdl_amd_host_calls", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_asdl_amd_host_calls() { return PyModule_Create(&definition); }
