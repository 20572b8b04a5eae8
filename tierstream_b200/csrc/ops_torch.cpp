// tierstream_b200._torch_ops: the operators of tsb.h on torch tensors, for ops.py. One C++ call checks the tensors, takes
// outputs and scratch from torch's allocator and enqueues on torch's current stream of the tensors' device; a small
// operator's call costs about 4 us this way, 10 through ctypes. Refused tensors raise ValueError, refusals of the library
// abi.TsError.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <string>

#include "tierstream/tsb.h"

namespace {

PyObject* g_error = nullptr;  // abi.TsError

// Messages are put together from strings: a stream's number formatting lives in the C++ library's locale, and the process
// (python, torch) may hold another version of it than this file was compiled against.
std::string text(const std::string& v) { return v; }
std::string text(const char* v) { return v; }
std::string text(int64_t v) { return std::to_string(v); }
template <class... A>
[[noreturn]] void refuse(const A&... a) {
  throw c10::ValueError({__func__, __FILE__, uint32_t(__LINE__)}, (text(a) + ...));
}
std::string place_of(const at::Tensor& t) { return t.is_cuda() ? "cuda:" + std::to_string(t.get_device()) : "the CPU"; }
std::string shape_of(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}
void check(ss_status st) {
  if (st == SS_OK) return;
  PyObject* args = Py_BuildValue("(is)", int(st), ss_last_error());
  if (args && g_error) {
    PyObject* e = PyObject_CallObject(g_error, args);
    if (e) {
      PyErr_SetObject(g_error, e);
      Py_DECREF(e);
    }
  }
  Py_XDECREF(args);
  throw python_error();
}

const at::Tensor& tensor(const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) refuse(name, ": a tensor is wanted, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
uint32_t type_code(const char* name, const at::Tensor& t, bool any) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return TSB_BF16;
    case at::kHalf: return TSB_F16;
    case at::kFloat:
      if (any) return TSB_F32;
      [[fallthrough]];
    default: refuse(name, ": ", c10::toString(t.scalar_type()), " is not served (bfloat16, float16", any ? ", float32)" : ")");
  }
}
void first(const char* name, const at::Tensor& t) {
  if (t.dim() != 2) refuse(name, ": two dimensions are wanted, got ", shape_of(t.sizes()));
}

struct Mat {
  void* p = nullptr;
  uint64_t ld = 0;
};
// a [rows][cols] matrix of like's type on like's device, rows at any distance
Mat mat(const char* name, const at::Tensor& t, int64_t rows, int64_t cols, const at::Tensor& like) {
  if (t.scalar_type() != like.scalar_type() || t.device() != like.device())
    refuse(name, ": ", c10::toString(like.scalar_type()), " on ", place_of(like), " is wanted, got ",
           c10::toString(t.scalar_type()), " on ", place_of(t));
  if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols)
    refuse(name, ": shape [", rows, ", ", cols, "] is wanted, got ", shape_of(t.sizes()));
  if (cols > 1 && t.stride(1) != 1) refuse(name, ": the elements of a row must be adjacent");
  if (rows > 1 && t.stride(0) < cols) refuse(name, ": rows overlap");
  return {t.data_ptr(), uint64_t(rows > 1 ? t.stride(0) : cols)};
}
void* flat(const char* name, const at::Tensor& t, at::IntArrayRef shape, at::ScalarType type, const at::Tensor& like) {
  if (t.scalar_type() != type || t.device() != like.device() || t.sizes() != shape || !t.is_contiguous())
    refuse(name, ": a contiguous ", c10::toString(type), " of shape ", shape_of(shape), " on ", place_of(like), " is wanted, got ",
           c10::toString(t.scalar_type()), " ", shape_of(t.sizes()), " on ", place_of(t));
  return t.data_ptr();
}
// whether two matrices are other columns of one buffer's rows
bool beside(const at::Tensor& a, const at::Tensor& b) {
  if (a.dim() != 2 || b.dim() != 2 || a.scalar_type() != b.scalar_type() || a.stride(0) != b.stride(0)) return false;
  const int64_t ld = a.stride(0), size = a.element_size();
  const int64_t bytes = static_cast<char*>(a.data_ptr()) - static_cast<char*>(b.data_ptr());
  if (ld <= 0 || a.stride(1) != 1 || b.stride(1) != 1 || bytes % size) return false;
  const int64_t first = (bytes / size % ld + ld) % ld;  // a's first column, b's being 0
  return first >= b.size(1) && first + a.size(1) <= ld;
}
// refuses an output that shares memory with an input
void apart(const char* name, const at::Tensor& out, const at::Tensor& in) {
  auto end = [](const at::Tensor& t) {
    int64_t n = t.numel() ? 1 : 0;
    for (int64_t d = 0; d < t.dim() && n; ++d) n += (t.size(d) - 1) * t.stride(d);
    return static_cast<char*>(t.data_ptr()) + n * t.element_size();
  };
  if (static_cast<char*>(out.data_ptr()) < end(in) && static_cast<char*>(in.data_ptr()) < end(out) && !beside(out, in))
    refuse(name, ": overlaps an input");
}
// refuses an output that lies on its residual in any other way than element on element
void on_residual(const at::Tensor& out, const at::Tensor& residual) {
  if (out.data_ptr() != residual.data_ptr() || out.strides() != residual.strides()) apart("out", out, residual);
}
at::Tensor fresh(const at::Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options().requires_grad(false)); }

c10::Device cuda_of(const at::Tensor& t) {
  if (!t.is_cuda()) refuse("CUDA tensors are wanted");
  return t.device();
}
// the device of `like` current, and its stream
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const at::Tensor& like)
      : guard(cuda_of(like)), stream(c10::cuda::getCurrentCUDAStream(like.device().index()).stream()) {}
};
// runs an entry point with scratch of the size it asks for
template <class A>
void run(A& a, const On& on, const at::Tensor& like, uint64_t (*size)(const A*), ss_status (*fn)(const A*)) {
  a.struct_size = sizeof a;
  a.stream = on.stream;
  at::Tensor scratch;
  if (const uint64_t n = size(&a)) {
    scratch = at::empty({int64_t(n + 256)}, like.options().dtype(at::kByte).requires_grad(false));
    a.workspace = reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(scratch.data_ptr()) + 255) & ~uintptr_t(255));
    a.workspace_bytes = n;
  }
  check(fn(&a));
}
bool there(PyObject* o) { return o != Py_None; }
long integer(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
void argc(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) refuse(int64_t(want), " arguments are wanted, got ", int64_t(n));
}

// linear(x, w, bias, residual, act, pre, out)
PyObject* linear(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  argc(n, 7);
  const at::Tensor &x = tensor("x", v[0]), &w = tensor("w", v[1]);
  tsb_linear_args a{};
  a.dtype = type_code("x", x, false);
  first("x", x);
  if (w.dim() != 2) refuse("w: two dimensions are wanted, got ", shape_of(w.sizes()));
  const int64_t rows = x.size(0), k = x.size(1), cols = w.size(0);
  a.act = uint32_t(integer(v[4]));
  a.rows = uint64_t(rows), a.n = uint64_t(cols), a.k = uint64_t(k);
  Mat m = mat("x", x, rows, k, x);
  a.x = m.p, a.ldx = m.ld;
  m = mat("w", w, cols, k, x);
  a.w = m.p, a.ldw = m.ld;
  if (there(v[2])) a.bias = flat("bias", tensor("bias", v[2]), {cols}, x.scalar_type(), x);
  if (there(v[3])) {
    m = mat("residual", tensor("residual", v[3]), rows, cols, x);
    a.residual = m.p, a.ldr = m.ld;
  }
  if (there(v[5])) {
    const at::Tensor& pre = tensor("pre", v[5]);
    m = mat("pre", pre, rows, cols, x);
    for (int i : {0, 1, 2, 3})
      if (there(v[i])) apart("pre", pre, tensor("pre", v[i]));
    a.pre = m.p, a.ldp = m.ld;
  }
  const On on(x);
  at::Tensor out;
  if (there(v[6])) {
    out = tensor("out", v[6]);
    m = mat("out", out, rows, cols, x);
    for (int i : {0, 1, 2, 5})
      if (there(v[i])) apart("out", out, tensor("out", v[i]));
    if (there(v[3])) on_residual(out, tensor("residual", v[3]));
  } else {
    out = fresh(x, {rows, cols});
    m = {out.data_ptr(), uint64_t(cols)};
  }
  a.y = m.p, a.ldy = m.ld;
  run(a, on, x, tsb_linear_workspace, tsb_linear);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// linear_backward(dy, x, w, act, pre, need x, need w, need bias) -> (dx, dw, db)
PyObject* linear_backward(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  argc(n, 8);
  const at::Tensor &dy = tensor("dy", v[0]), &x = tensor("x", v[1]), &w = tensor("w", v[2]);
  tsb_linear_grad_args a{};
  a.dtype = type_code("dy", dy, false);
  first("dy", dy);
  if (x.dim() != 2) refuse("x: two dimensions are wanted, got ", shape_of(x.sizes()));
  const int64_t rows = dy.size(0), cols = dy.size(1), k = x.size(1);
  a.act = uint32_t(integer(v[3]));
  a.rows = uint64_t(rows), a.n = uint64_t(cols), a.k = uint64_t(k);
  Mat m = mat("dy", dy, rows, cols, dy);
  a.dy = m.p, a.lddy = m.ld;
  m = mat("x", x, rows, k, dy);
  a.x = m.p, a.ldx = m.ld;
  m = mat("w", w, cols, k, dy);
  a.w = m.p, a.ldw = m.ld;
  if (a.act != TSB_ACT_NONE) {
    if (!there(v[4])) refuse("pre: an activation's slope needs it");
    m = mat("pre", tensor("pre", v[4]), rows, cols, dy);
    a.pre = m.p, a.ldp = m.ld;
  }
  const On on(dy);
  at::Tensor dx, dw, db;
  if (PyObject_IsTrue(v[5])) {
    dx = fresh(dy, {rows, k});
    a.dx = dx.data_ptr(), a.lddx = uint64_t(k);
  }
  if (PyObject_IsTrue(v[6])) {
    dw = fresh(dy, {cols, k});
    a.dw = dw.data_ptr(), a.lddw = uint64_t(k);
  }
  if (PyObject_IsTrue(v[7])) {
    db = fresh(dy, {cols});
    a.db = db.data_ptr();
  }
  run(a, on, dy, tsb_linear_backward_workspace, tsb_linear_backward);
  PyObject* r = PyTuple_New(3);
  const at::Tensor* g[3] = {&dx, &dw, &db};
  for (int i = 0; r && i < 3; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(*g[i]));  // (an undefined tensor is None)
  return r;
  END_HANDLE_TH_ERRORS
}

// route(logits, top, norm) -> (ids, weights)
PyObject* route(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  argc(n, 3);
  const at::Tensor& z = tensor("logits", v[0]);
  const uint32_t type = type_code("logits", z, true);
  first("logits", z);
  const int64_t rows = z.size(0), experts = z.size(1), top = integer(v[1]);
  const Mat m = mat("logits", z, rows, experts, z);
  if (top < 1 || top > 32 || top > experts) refuse("top: must be in [1, 32] and at most the experts, got ", top);
  const On on(z);
  at::Tensor ids = at::empty({rows, top}, z.options().dtype(at::kInt).requires_grad(false));
  at::Tensor w = at::empty({rows, top}, z.options().dtype(at::kFloat).requires_grad(false));
  check(tsb_route(type, m.p, m.ld, uint64_t(rows), uint32_t(experts), uint32_t(top), PyObject_IsTrue(v[2]),
                  static_cast<int32_t*>(ids.data_ptr()), static_cast<float*>(w.data_ptr()), on.stream));
  PyObject* r = PyTuple_New(2);
  if (r) {
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(ids));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(w));
  }
  return r;
  END_HANDLE_TH_ERRORS
}

// route_backward(dweights, logits, ids, weights, norm) -> dlogits
PyObject* route_backward(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  argc(n, 5);
  const at::Tensor &d = tensor("dweights", v[0]), &z = tensor("logits", v[1]), &i = tensor("ids", v[2]),
                   &w = tensor("weights", v[3]);
  const uint32_t type = type_code("logits", z, true), dtype = type_code("dweights", d, true);
  first("logits", z);
  first("dweights", d);
  const int64_t rows = z.size(0), experts = z.size(1);
  const Mat m = mat("logits", z, rows, experts, z);
  if (d.size(0) != rows) refuse("dweights: ", rows, " rows are wanted, got ", d.size(0));
  const void* pd = flat("dweights", d, d.sizes(), d.scalar_type(), z);
  const void* pi = flat("ids", i, d.sizes(), at::kInt, z);
  const void* pw = flat("weights", w, d.sizes(), at::kFloat, z);
  const On on(z);
  at::Tensor out = fresh(z, {rows, experts});
  check(tsb_route_backward(type, dtype, pd, m.p, m.ld, static_cast<const int32_t*>(pi), static_cast<const float*>(pw),
                           uint64_t(rows), uint32_t(experts), uint32_t(d.size(1)), PyObject_IsTrue(v[4]), out.data_ptr(),
                           uint64_t(experts), on.stream));
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// units(address of a tsb_units, gate, up, down, slot_of) -> (units, ffn, hidden), the struct filled
PyObject* units(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  argc(n, 5);
  tsb_units* u = static_cast<tsb_units*>(PyLong_AsVoidPtr(v[0]));
  if (!u) throw python_error();
  const at::Tensor& gate = tensor("gate", v[1]);
  (void)type_code("gate", gate, false);
  if (gate.dim() != 3) refuse("gate: [slots][ffn][hidden] is wanted, got ", shape_of(gate.sizes()));
  const int64_t slots = gate.size(0), ffn = gate.size(1), hidden = gate.size(2);
  *u = tsb_units{};
  u->struct_size = sizeof *u;
  u->n_slots = uint32_t(slots);
  const char* names[3] = {"gate", "up", "down"};
  for (int i = 0; i < 3; ++i) {
    const at::Tensor& t = tensor(names[i], v[1 + i]);
    const int64_t r = i == 2 ? hidden : ffn, c = i == 2 ? ffn : hidden;
    if (t.scalar_type() != gate.scalar_type() || t.device() != gate.device() || t.dim() != 3 || t.size(0) != slots ||
        t.size(1) != r || t.size(2) != c)
      refuse(names[i], ": ", c10::toString(gate.scalar_type()), " of shape [", slots, ", ", r, ", ", c, "] on ", place_of(gate),
             " is wanted, got ", c10::toString(t.scalar_type()), " ", shape_of(t.sizes()), " on ", place_of(t));
    if (!t.is_contiguous() &&
        ((r > 1 && t.stride(1) != c) || (c > 1 && t.stride(2) != 1) || (slots > 1 && t.stride(0) < r * c)))
      refuse(names[i], ": a slot's matrix must be contiguous, and slots apart");
    u->part[i] = t.data_ptr();
    u->stride[i] = uint64_t(t.stride(0)) * 2;
  }
  u->n_units = uint32_t(slots);
  if (there(v[4])) {
    const at::Tensor& s = tensor("slot_of", v[4]);
    u->n_units = uint32_t(s.numel());
    u->slot_of = static_cast<const int32_t*>(flat("slot_of", s, {s.numel()}, at::kInt, gate));
  }
  (void)cuda_of(gate);
  return Py_BuildValue("(ILL)", u->n_units, (long long)ffn, (long long)hidden);
  END_HANDLE_TH_ERRORS
}

// What the block's two calls share; the units' type and device are checked by ops.py.
template <class A>
void ffn_args(A& a, const at::Tensor& x, PyObject* ids, PyObject* weights, PyObject* units, PyObject* ffn, PyObject* act) {
  a.dtype = type_code("x", x, false);
  first("x", x);
  const at::Tensor& i = tensor("ids", ids);
  if (i.dim() != 2) refuse("ids: two dimensions are wanted, got ", shape_of(i.sizes()));
  const int64_t shape[2] = {x.size(0), i.size(1)};
  const Mat m = mat("x", x, x.size(0), x.size(1), x);
  a.x = m.p, a.ldx = m.ld;
  a.act = uint32_t(integer(act));
  a.top = uint32_t(shape[1]);
  a.rows = uint64_t(x.size(0)), a.hidden = uint64_t(x.size(1)), a.ffn = uint64_t(integer(ffn));
  a.ids = static_cast<const int32_t*>(flat("ids", i, shape, at::kInt, x));
  a.weights = static_cast<const float*>(flat("weights", tensor("weights", weights), shape, at::kFloat, x));
  a.units = static_cast<const tsb_units*>(PyLong_AsVoidPtr(units));
}

// ffn(x, ids, weights, address of the units, ffn, act, residual, out)
PyObject* ffn(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  argc(n, 8);
  const at::Tensor& x = tensor("x", v[0]);
  tsb_ffn_args a{};
  ffn_args(a, x, v[1], v[2], v[3], v[4], v[5]);
  const int64_t rows = x.size(0), hidden = x.size(1);
  const bool on_x = there(v[6]) && there(v[7]) && tensor("residual", v[6]).data_ptr() == x.data_ptr() &&
                    tensor("out", v[7]).data_ptr() == x.data_ptr();
  if (there(v[6])) {
    const Mat m = mat("residual", tensor("residual", v[6]), rows, hidden, x);
    a.residual = m.p, a.ldr = m.ld;
  }
  const On on(x);
  at::Tensor out;
  if (there(v[7])) {
    out = tensor("out", v[7]);
    const Mat m = mat("out", out, rows, hidden, x);
    if (!on_x) apart("out", out, x);  // (in place on x as its own residual: x is read first)
    apart("out", out, tensor("ids", v[1]));
    apart("out", out, tensor("weights", v[2]));
    if (there(v[6])) on_residual(out, tensor("residual", v[6]));
    a.y = m.p, a.ldy = m.ld;
  } else {
    out = fresh(x, {rows, hidden});
    a.y = out.data_ptr(), a.ldy = uint64_t(hidden);
  }
  run(a, on, x, tsb_ffn_workspace, tsb_ffn);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ffn_backward(dy, x, ids, weights, address of the units, units, ffn, act, need x, need weights, need units)
// -> (dx, dweights, dgate, dup, ddown)
PyObject* ffn_backward(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  argc(n, 11);
  const at::Tensor &dy = tensor("dy", v[0]), &x = tensor("x", v[1]);
  tsb_ffn_grad_args a{};
  ffn_args(a, x, v[2], v[3], v[4], v[6], v[7]);
  const int64_t rows = x.size(0), hidden = x.size(1), units = integer(v[5]), ffn = int64_t(a.ffn);
  const Mat m = mat("dy", dy, rows, hidden, x);
  a.dy = m.p, a.lddy = m.ld;
  const On on(x);
  at::Tensor g[5];
  if (PyObject_IsTrue(v[8])) {
    g[0] = fresh(x, {rows, hidden});
    a.dx = g[0].data_ptr(), a.lddx = uint64_t(hidden);
  }
  if (PyObject_IsTrue(v[9])) {
    g[1] = fresh(x, {rows, int64_t(a.top)});
    a.dweights = g[1].data_ptr();
  }
  if (PyObject_IsTrue(v[10])) {
    g[2] = fresh(x, {units, ffn, hidden});
    g[3] = fresh(x, {units, ffn, hidden});
    g[4] = fresh(x, {units, hidden, ffn});
    a.dgate = g[2].data_ptr(), a.dup = g[3].data_ptr(), a.ddown = g[4].data_ptr();
  }
  run(a, on, x, tsb_ffn_backward_workspace, tsb_ffn_backward);
  PyObject* r = PyTuple_New(5);
  for (int i = 0; r && i < 5; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(g[i]));
  return r;
  END_HANDLE_TH_ERRORS
}

PyObject* set_error(PyObject*, PyObject* e) {
  Py_INCREF(e);
  Py_XDECREF(g_error);
  g_error = e;
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef fast(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef g_methods[] = {fast<linear>("linear"),
                           fast<linear_backward>("linear_backward"),
                           fast<route>("route"),
                           fast<route_backward>("route_backward"),
                           fast<units>("units"),
                           fast<ffn>("ffn"),
                           fast<ffn_backward>("ffn_backward"),
                           {"set_error", set_error, METH_O, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_ops", "The operators of tsb.h on torch tensors (ops.py).", -1,
                        g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops(void) { return PyModule_Create(&g_module); }
