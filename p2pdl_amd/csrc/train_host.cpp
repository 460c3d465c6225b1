// Host side of the trainer's operators (p2pdl_amd/training.py): the call that
// a step makes -- dense tensors of one type on the current device, shapes
// that match -- checked, its results and workspace allocated and the C ABI
// called, without Python between.  At a small model's sizes the kernels of an
// operator take less time than its Python wrapper (layer norm of 32 x 512,
// forward and backward: 12 us on the device, 31 us a pass through Python).
//
// Every function returns None, having done nothing, where anything is not as
// above; training.py then takes its own path, which copies what has to be
// copied and says what is wrong.  The kernels and their results are the same.
// A non-zero status of the C ABI goes to the callable given to bind().
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <exception>
#include <utility>

#include "../../include/p2pdl.h"

namespace {

struct Abi {
  decltype(&p2p_layernorm_fwd) layernorm_fwd;
  decltype(&p2p_layernorm_bwd_workspace) layernorm_bwd_workspace;
  decltype(&p2p_layernorm_bwd) layernorm_bwd;
  decltype(&p2p_dropout) dropout;
  decltype(&p2p_gated_linear_workspace) gated_workspace;
  decltype(&p2p_gated_linear_fwd) gated_fwd;
  decltype(&p2p_gated_linear_bwd) gated_bwd;
  decltype(&p2p_linear_ce_workspace) ce_workspace;
  decltype(&p2p_linear_ce_fwd) ce_fwd;
  decltype(&p2p_linear_ce_bwd) ce_bwd;
} g_abi;
constexpr int kAbiFunctions = sizeof(Abi) / sizeof(void*);
bool g_bound = false;
PyObject *g_check, *g_get_device, *g_get_stream;  // N.check, torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream

// The caller's path: None, no error set.
struct OtherPath {};
// A Python error is set.
struct Raised {};

const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) throw OtherPath{};
  return THPVariable_Unpack(o);
}
const at::Tensor* tensor_or_none(PyObject* o) { return o == Py_None ? nullptr : &tensor(o); }

int32_t dtype_of(const at::Tensor& x) {
  switch (x.scalar_type()) {
    case at::kFloat: return P2P_DTYPE_F32;
    case at::kHalf: return P2P_DTYPE_F16;
    case at::kBFloat16: return P2P_DTYPE_BF16;
    default: throw OtherPath{};
  }
}

// The first operand of a call: dense, not empty, on the current device.
struct Call {
  const at::Tensor& x;
  int32_t dtype;
  int64_t cols, rows;
  explicit Call(PyObject* o) : x(tensor(o)), dtype(0) {
    if (!g_bound || x.layout() != at::kStrided || !x.is_cuda() || x.dim() < 1 || x.numel() == 0 || !x.is_contiguous())
      throw OtherPath{};
    dtype = dtype_of(x);
    cols = x.size(-1);
    rows = x.numel() / cols;
    PyObject* d = PyObject_CallNoArgs(g_get_device);
    if (!d) throw Raised{};
    const long now = PyLong_AsLong(d);
    Py_DECREF(d);
    if (now != x.get_device()) throw OtherPath{};
  }
  // dense, on x's device
  void with(const at::Tensor& t, at::ScalarType type) const {
    if (t.layout() != at::kStrided || t.scalar_type() != type || !t.is_cuda() || t.get_device() != x.get_device() || !t.is_contiguous())
      throw OtherPath{};
  }
  void with(const at::Tensor& t, at::ScalarType type, at::IntArrayRef shape) const {
    if (t.sizes() != shape) throw OtherPath{};
    with(t, type);
  }
  void same(const at::Tensor& t) const { with(t, x.scalar_type(), x.sizes()); }
  at::IntArrayRef lead() const { return x.sizes().slice(0, x.dim() - 1); }
  at::TensorOptions options(at::ScalarType t) const { return x.options().dtype(t); }
  p2p_stream_t stream() const {
    PyObject* i = PyLong_FromLong(x.get_device());
    PyObject* s = i ? PyObject_CallOneArg(g_get_stream, i) : nullptr;
    Py_XDECREF(i);
    if (!s) throw Raised{};
    void* p = PyLong_AsVoidPtr(s);
    Py_DECREF(s);
    if (PyErr_Occurred()) throw Raised{};
    return p;
  }
  at::Tensor workspace(int64_t bytes, const char* what) const;
};

void check(int64_t rc, const char* what) {
  if (rc == 0) return;
  PyObject* r = PyObject_CallFunction(g_check, "Ls", static_cast<long long>(rc), what);
  Py_XDECREF(r);
  throw Raised{};
}
at::Tensor Call::workspace(int64_t bytes, const char* what) const {
  if (bytes < 0) check(bytes, what);
  return bytes ? at::empty({bytes}, options(at::kByte)) : at::Tensor();
}
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// A leading shape with one more dimension in front or behind, without an allocation.
struct Shape {
  int64_t d[9];
  int n = 0;
  Shape(at::IntArrayRef lead, int64_t front, int64_t back) {
    if (lead.size() > 7) throw OtherPath{};
    if (front) d[n++] = front;
    for (const int64_t v : lead) d[n++] = v;
    if (back) d[n++] = back;
  }
  operator at::IntArrayRef() const { return {d, static_cast<size_t>(n)}; }
};

PyObject* wrap(at::Tensor t) {
  if (!t.defined()) Py_RETURN_NONE;
  PyObject* o = THPVariable_Wrap(std::move(t));
  if (!o) throw Raised{};
  return o;
}
template <typename... T>
PyObject* tuple(T... t) {
  PyObject* r = PyTuple_New(sizeof...(T));
  if (!r) throw Raised{};
  Py_ssize_t i = 0;
  try {
    (PyTuple_SET_ITEM(r, i++, wrap(std::move(t))), ...);
  } catch (...) {
    Py_DECREF(r);
    throw;
  }
  return r;
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw OtherPath{};
  }
  return v;
}
uint64_t word(PyObject* o) {
  if (!PyLong_Check(o)) throw OtherPath{};
  const unsigned long long v = PyLong_AsUnsignedLongLong(o);
  if (v == static_cast<unsigned long long>(-1) && PyErr_Occurred()) {
    PyErr_Clear();
    throw OtherPath{};
  }
  return v;
}
int64_t integer(PyObject* o) {
  if (!PyLong_Check(o)) throw OtherPath{};
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw OtherPath{};
  }
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v;
}

// layer_norm_forward(x, weight, bias, eps) -> (y, mean, rstd)
PyObject* layer_norm_forward(PyObject* const* a) {
  const Call c(a[0]);
  const at::Tensor *w = tensor_or_none(a[1]), *b = tensor_or_none(a[2]);
  const double eps = real(a[3]);
  if (b && !w) throw OtherPath{};
  if (w) c.with(*w, c.x.scalar_type(), {c.cols});
  if (b) c.with(*b, c.x.scalar_type(), {c.cols});
  if (c.cols > 16384) throw OtherPath{};
  at::Tensor y = at::empty_like(c.x), mean = at::empty(c.lead(), c.options(at::kFloat)), rstd = at::empty(c.lead(), c.options(at::kFloat));
  check(g_abi.layernorm_fwd(c.x.data_ptr(), c.cols, w ? w->data_ptr() : nullptr, b ? b->data_ptr() : nullptr, c.rows, c.cols,
                            static_cast<float>(eps), y.data_ptr(), mean.data_ptr<float>(), rstd.data_ptr<float>(), c.dtype,
                            c.stream()),
        "p2p_layernorm_fwd");
  return tuple(std::move(y), std::move(mean), std::move(rstd));
}

// layer_norm_backward(dy, x, mean, rstd, weight) -> (dx, dweight, dbias)
PyObject* layer_norm_backward(PyObject* const* a) {
  const Call c(a[1]);
  const at::Tensor &dy = tensor(a[0]), &mean = tensor(a[2]), &rstd = tensor(a[3]);
  const at::Tensor* w = tensor_or_none(a[4]);
  c.same(dy);
  c.with(mean, at::kFloat, c.lead());
  c.with(rstd, at::kFloat, c.lead());
  if (w) c.with(*w, c.x.scalar_type(), {c.cols});
  if (c.cols > 16384) throw OtherPath{};
  at::Tensor dx = at::empty_like(c.x), dw, db, ws;
  int64_t bytes = 0;
  if (w) {
    dw = at::empty({c.cols}, c.x.options());
    db = at::empty({c.cols}, c.x.options());
    bytes = g_abi.layernorm_bwd_workspace(c.rows, c.cols, c.dtype);
    ws = c.workspace(bytes, "p2p_layernorm_bwd_workspace");
  }
  check(g_abi.layernorm_bwd(dy.data_ptr(), c.cols, c.x.data_ptr(), c.cols, w ? w->data_ptr() : nullptr, mean.data_ptr<float>(),
                            rstd.data_ptr<float>(), c.rows, c.cols, dx.data_ptr(), ptr(dw), ptr(db), ptr(ws), bytes, c.dtype,
                            c.stream()),
        "p2p_layernorm_bwd");
  return tuple(std::move(dx), std::move(dw), std::move(db));
}

// dropout(x, p, seed, offset, residual) -> y
PyObject* dropout(PyObject* const* a) {
  const Call c(a[0]);
  const double p = real(a[1]);
  if (!(p >= 0.0 && p <= 1.0)) throw OtherPath{};
  const uint64_t seed = word(a[2]);
  uint64_t offset = 0;
  const at::Tensor* counter = nullptr;
  if (PyLong_Check(a[3])) {
    offset = word(a[3]);
  } else {
    counter = &tensor(a[3]);
    c.with(*counter, at::kLong);
    if (counter->numel() != 1) throw OtherPath{};
  }
  const at::Tensor* r = tensor_or_none(a[4]);
  if (r) c.same(*r);
  at::Tensor y = at::empty_like(c.x);
  check(g_abi.dropout(c.x.data_ptr(), r ? r->data_ptr() : nullptr, c.x.numel(), p, seed, offset,
                      counter ? static_cast<const uint64_t*>(counter->data_ptr()) : nullptr, y.data_ptr(), c.dtype, c.stream()),
        "p2p_dropout");
  return wrap(std::move(y));
}

struct Gated : Call {
  const at::Tensor &wg, &wu;
  p2p_gated_linear_t args{};
  Gated(PyObject* xo, PyObject* wgo, PyObject* wuo, PyObject* act) : Call(xo), wg(tensor(wgo)), wu(tensor(wuo)) {
    if (wg.dim() != 2 || wg.size(0) < 1 || wg.size(1) != cols) throw OtherPath{};
    with(wg, x.scalar_type());
    with(wu, x.scalar_type(), wg.sizes());
    args.x = x.data_ptr(), args.w_gate = wg.data_ptr(), args.w_up = wu.data_ptr();
    args.ldx = args.ldg = args.ldu = cols;
    args.tokens = rows, args.hidden = cols, args.units = wg.size(0);
    args.activation = static_cast<int32_t>(integer(act)), args.dtype = dtype;
    if (cols > (1 << 22) - 8 || args.units > (1 << 21) - 8) throw OtherPath{};
  }
};

// gated_linear_forward(x, w_gate, w_up, activation, save) -> (h, gate, up)
PyObject* gated_linear_forward(PyObject* const* a) {
  Gated c(a[0], a[1], a[2], a[3]);
  const bool save = truth(a[4]);
  const Shape shape(c.lead(), 0, c.args.units);
  at::Tensor h = at::empty(shape, c.x.options()), gate, up;
  if (save) {
    gate = at::empty(shape, c.options(at::kFloat));
    up = at::empty(shape, c.options(at::kFloat));
  }
  c.args.h = h.data_ptr(), c.args.gate = static_cast<float*>(ptr(gate)), c.args.up = static_cast<float*>(ptr(up));
  const int64_t bytes = g_abi.gated_workspace(&c.args, 0);
  const at::Tensor ws = c.workspace(bytes, "p2p_gated_linear_workspace");
  check(g_abi.gated_fwd(&c.args, ptr(ws), bytes, c.stream()), "p2p_gated_linear_fwd");
  return tuple(std::move(h), std::move(gate), std::move(up));
}

// gated_linear_backward(dh, x, w_gate, w_up, gate, up, activation) -> (dx, dw_gate, dw_up)
PyObject* gated_linear_backward(PyObject* const* a) {
  Gated c(a[1], a[2], a[3], a[6]);
  const at::Tensor &dh = tensor(a[0]), &gate = tensor(a[4]), &up = tensor(a[5]);
  const Shape shape(c.lead(), 0, c.args.units);
  c.with(dh, c.x.scalar_type(), shape);
  c.with(gate, at::kFloat, shape);
  c.with(up, at::kFloat, shape);
  at::Tensor dx = at::empty_like(c.x), dwg = at::empty_like(c.wg), dwu = at::empty_like(c.wu);
  c.args.gate = gate.data_ptr<float>(), c.args.up = up.data_ptr<float>();
  c.args.dh = dh.data_ptr(), c.args.lddh = c.args.units;
  c.args.dx = dx.data_ptr(), c.args.dw_gate = dwg.data_ptr(), c.args.dw_up = dwu.data_ptr();
  const int64_t bytes = g_abi.gated_workspace(&c.args, 1);
  const at::Tensor ws = c.workspace(bytes, "p2p_gated_linear_workspace");
  check(g_abi.gated_bwd(&c.args, ptr(ws), bytes, c.stream()), "p2p_gated_linear_bwd");
  return tuple(std::move(dx), std::move(dwg), std::move(dwu));
}

struct Ce : Call {
  const at::Tensor &w, &target;
  p2p_linear_ce_t args{};
  Ce(PyObject* xo, PyObject* wo, PyObject* to, PyObject* ignore) : Call(xo), w(tensor(wo)), target(tensor(to)) {
    if (w.dim() != 2 || w.size(0) < 1 || w.size(1) != cols || cols > (1 << 22) - 8) throw OtherPath{};
    with(w, x.scalar_type());
    with(target, at::kLong, lead());
    args.x = x.data_ptr(), args.w = w.data_ptr(), args.target = target.data_ptr<int64_t>();
    args.ldx = args.ldw = cols;
    args.tokens = rows, args.hidden = cols, args.vocab = w.size(0);
    args.ignore_index = integer(ignore), args.dtype = dtype;
  }
};

// linear_cross_entropy_forward(x, weight, target, ignore_index, mean) -> (loss, lse, norm)
PyObject* linear_cross_entropy_forward(PyObject* const* a) {
  Ce c(a[0], a[1], a[2], a[3]);
  c.args.mean = truth(a[4]);
  at::Tensor loss = at::empty({}, c.options(at::kFloat)), norm = at::empty({}, c.options(at::kFloat));
  at::Tensor lse = at::empty(c.lead(), c.options(at::kFloat));
  c.args.loss = loss.data_ptr<float>(), c.args.norm = norm.data_ptr<float>(), c.args.lse = lse.data_ptr<float>();
  const int64_t bytes = g_abi.ce_workspace(&c.args, 0);
  const at::Tensor ws = c.workspace(bytes, "p2p_linear_ce_workspace");
  check(g_abi.ce_fwd(&c.args, ptr(ws), bytes, c.stream()), "p2p_linear_ce_fwd");
  return tuple(std::move(loss), std::move(lse), std::move(norm));
}

// linear_cross_entropy_backward(x, weight, target, lse, norm, dloss, ignore_index) -> (dx, dweight)
PyObject* linear_cross_entropy_backward(PyObject* const* a) {
  Ce c(a[0], a[1], a[2], a[6]);
  const at::Tensor &lse = tensor(a[3]), &norm = tensor(a[4]);
  const at::Tensor* dloss = tensor_or_none(a[5]);
  c.with(lse, at::kFloat, c.lead());
  c.with(norm, at::kFloat, at::IntArrayRef());
  if (dloss) {
    c.with(*dloss, at::kFloat);
    if (dloss->numel() != 1) throw OtherPath{};
  }
  at::Tensor dx = at::empty_like(c.x), dw = at::empty_like(c.w);
  c.args.lse = lse.data_ptr<float>(), c.args.norm = norm.data_ptr<float>();
  c.args.dloss = dloss ? dloss->data_ptr<float>() : nullptr;
  c.args.dx = dx.data_ptr(), c.args.dw = dw.data_ptr();
  const int64_t bytes = g_abi.ce_workspace(&c.args, 1);
  const at::Tensor ws = c.workspace(bytes, "p2p_linear_ce_workspace");
  check(g_abi.ce_bwd(&c.args, ptr(ws), bytes, c.stream()), "p2p_linear_ce_bwd");
  return tuple(std::move(dx), std::move(dw));
}

// No C++ exception leaves a call.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "_train_host: %d arguments expected, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const OtherPath&) {
    Py_RETURN_NONE;
  } catch (const Raised&) {
    return nullptr;
  } catch (const c10::OutOfMemoryError&) {
    Py_RETURN_NONE;  // torch's own allocation in the caller's path raises it as torch does
  } catch (const std::exception& e) {
    PyErr_Format(PyExc_RuntimeError, "_train_host: %s", e.what());
    return nullptr;
  }
}

// bind(addresses, check, get_device, get_stream): the C ABI's functions in the order of Abi.
PyObject* bind(PyObject*, PyObject* args) {
  PyObject *list, *chk, *dev, *stream;
  if (!PyArg_ParseTuple(args, "O!OOO", &PyTuple_Type, &list, &chk, &dev, &stream)) return nullptr;
  if (PyTuple_GET_SIZE(list) != kAbiFunctions) {
    PyErr_SetString(PyExc_ValueError, "_train_host.bind: another number of functions");
    return nullptr;
  }
  void* f[kAbiFunctions];
  for (int i = 0; i < kAbiFunctions; ++i) {
    f[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(list, i));
    if (!f[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "_train_host.bind: a null function");
      return nullptr;
    }
  }
  static_assert(sizeof(f) == sizeof(g_abi), "pointers only");
  __builtin_memcpy(&g_abi, f, sizeof(f));
  for (PyObject* o : {chk, dev, stream}) Py_INCREF(o);
  g_check = chk, g_get_device = dev, g_get_stream = stream;
  g_bound = true;
  Py_RETURN_NONE;
}

#define P2P_ENTRY(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                         P2P_ENTRY(layer_norm_forward, 4),
                         P2P_ENTRY(layer_norm_backward, 5),
                         P2P_ENTRY(dropout, 5),
                         P2P_ENTRY(gated_linear_forward, 5),
                         P2P_ENTRY(gated_linear_backward, 7),
                         P2P_ENTRY(linear_cross_entropy_forward, 5),
                         P2P_ENTRY(linear_cross_entropy_backward, 7),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_train_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__train_host(void) { return PyModule_Create(&module); }
