// The Python binding of the operators that run once or more a layer of every step (rope.py, kv_attn.py): argument checks,
// outputs and the call into the library in one trip out of Python.  At the sizes of a decode step the ctypes route took
// longer on the host than the kernels on the GPU (16 sequences: rotation 13 us of the host for 4 us, append 18 for 12,
// attention 20 for 11).  The library itself is loaded by _lib.py, which hands over the entry points' addresses.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <optional>
#include <string>

#include "../../include/sdcguard_hip.h"

namespace {

using at::Tensor;
typedef std::optional<Tensor> Maybe;

struct Entry {
  decltype(&sdc_rope) rope;
  decltype(&sdc_kv_append) append;
  decltype(&sdc_kv_attend_workspace) workspace;
  decltype(&sdc_kv_attend) attend;
};
Entry g_entry;
PyObject* g_check = nullptr;                   // _lib.check: raises for a status
PyObject* g_error = nullptr;                   // _lib.HipLibraryError

// Python's own exceptions, thrown through C++ (the error is already set)
struct Raised {};
[[noreturn]] void refuse(PyObject* kind, const std::string& what) {
  PyErr_SetString(kind, what.c_str());
  throw Raised{};
}
[[noreturn]] void value_error(const std::string& what) { refuse(PyExc_ValueError, what); }

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(name) + " must be a tensor");
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda())
    refuse(g_error, std::string("sdcguard_amd runs on the GPU only (") + name + " is on " + t.device().str() +
                        "); there is no CPU implementation in the product");
  return t;
}
Maybe maybe(PyObject* o, const char* name) { return o == Py_None ? Maybe() : Maybe(tensor(o, name)); }
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return v;
}
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v != 0;
}

// The cache's operators, and a rotation's frequencies, have no gradient: rather than drop one the call is refused.
void no_tangent(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t && t->_fw_grad(/*level=*/0).defined()) value_error(std::string(what) + ": no forward-mode gradient");
}
void no_gradient(const char* what, std::initializer_list<const Tensor*> ts) {
  no_tangent(what, ts);
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : ts)
    if (t && t->requires_grad())
      value_error(std::string(what) + " takes no gradient: detached tensors, or torch.no_grad(), are needed");
}
const Tensor* get(const Maybe& t) { return t ? &*t : nullptr; }
// What a call has written to: autograd then knows of it where it kept the former values.  (Tensors of inference mode have no
// version.)
void written(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// A tensor that is written: no element of it twice, and none of it also an input's unless it is that input (`same`) as a whole.
void check_written(const char* name, const Tensor& t, const Tensor* same, std::initializer_list<const Tensor*> others) {
  if (at::has_internal_overlap(t) == at::MemOverlap::Yes) value_error(std::string(name) + " must not hold an element twice");
  if (same && at::get_overlap_status(t, *same) == at::MemOverlapStatus::Partial)
    value_error(std::string(name) + " must be the input itself or share no memory with it");
  for (const Tensor* o : others) {
    const at::MemOverlapStatus s = at::get_overlap_status(t, *o);
    if (s == at::MemOverlapStatus::Partial || s == at::MemOverlapStatus::Full)
      value_error(std::string(name) + " must share no memory with the call's other tensors");
  }
}

int half_code(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return 0;
  if (t.scalar_type() == at::kHalf) return 1;
  refuse(g_error, std::string("unsupported dtype ") + c10::toString(t.scalar_type()));
}

// (torch's own state, asked without Python: a gradient's thread would have to wait for the interpreter's lock)
hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check(int rc, const char* what) {
  if (rc == 0) return;
  PyObject* r = PyObject_CallFunction(g_check, "is", rc, what);
  Py_XDECREF(r);
  throw Raised{};
}

// A call into the library, without the interpreter's lock.
template <class F>
int unlocked(F f) {
  PyThreadState* s = PyEval_SaveThread();
  const int rc = f();
  PyEval_RestoreThread(s);
  return rc;
}

void* ptr(const Maybe& t) { return t ? t->data_ptr() : nullptr; }
int64_t stride(const Maybe& t, int i) { return t ? t->stride(i) : 0; }

// ------------------------------------------------------------------------------------------------- the rotation
int check_turns(const Tensor& turns, int64_t head, const at::Device& dev) {
  if (turns.dim() != 1 || turns.scalar_type() != at::kDouble || !turns.is_contiguous() || turns.device() != dev)
    value_error("turns must be a contiguous float64 vector on the tensors' device (frequencies())");
  const int64_t rot = 2 * turns.size(0);
  if (rot > head) value_error(std::to_string(rot) + " rotated elements in heads of " + std::to_string(head));
  return (int)rot;
}
Tensor check_positions(const Tensor& p, int64_t tokens, const at::Device& dev) {
  if ((p.scalar_type() != at::kLong && p.scalar_type() != at::kInt) || p.device() != dev)
    value_error("positions must be int64 or int32 on the tensors' device");
  if (p.numel() != tokens) value_error(std::to_string(p.numel()) + " positions for " + std::to_string(tokens) + " tokens");
  return p.dim() == 1 && p.is_contiguous() ? p : p.reshape(-1).contiguous();
}

struct How {
  bool interleaved, inverse;
  double mscale;
};
// (called with and without the interpreter's lock: a gradient's thread holds none)
int launch_rotation(const Tensor& x, const Tensor& y, const Tensor& pos, const Tensor& turns, const How& how, hipStream_t s) {
  const int dt = x.scalar_type() == at::kBFloat16 ? 0 : x.scalar_type() == at::kHalf ? 1 : 4;
  return g_entry.rope(dt, x.const_data_ptr(), x.stride(0), x.stride(1), x.stride(2), y.data_ptr(), y.stride(0), y.stride(1),
                      y.stride(2), x.size(0), x.size(1), x.size(2), pos.const_data_ptr(), (int)pos.element_size(),
                      turns.const_data_ptr<double>(), 2 * turns.size(0), how.interleaved, how.mscale, how.inverse, s);
}
Tensor like(const Tensor& x) { return at::empty(x.sizes(), x.options()); }

// f() with the interpreter's lock, wherever the thread comes from; Python's error leaves with it.
template <class F>
auto locked(F f) {
  struct Lock {
    PyGILState_STATE s = PyGILState_Ensure();
    ~Lock() { PyGILState_Release(s); }
  } lock;
  try {
    return f();
  } catch (const Raised&) {
    python_error e;
    e.persist();
    throw e;
  }
}

struct Rotation : torch::autograd::Function<Rotation> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& pos, const Tensor& turns,
                        bool interleaved, double mscale, bool inverse) {
    ctx->save_for_backward({pos, turns});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["mscale"] = mscale;
    ctx->saved_data["inverse"] = inverse;
    const Tensor y = like(x);
    const c10::DeviceGuard guard(x.device());
    const int rc = launch_rotation(x, y, pos, turns, How{interleaved, inverse, mscale}, stream_of(x));
    if (rc != 0) locked([&] { check(rc, "sdc_rope"); });
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dy) {
    const auto saved = ctx->get_saved_variables();
    // the transposed rotation is the one by the negative angle, the factor on the result the same
    const Tensor dx = Rotation::apply(dy[0], saved[0], saved[1], ctx->saved_data["interleaved"].toBool(),
                                      ctx->saved_data["mscale"].toDouble(), !ctx->saved_data["inverse"].toBool());
    return {dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// rotate(x, positions, turns, interleaved, mscale, inverse, out)
PyObject* rotate(PyObject* const* a) {
  const Tensor& x = tensor(a[0], "x");
  const Tensor& positions = tensor(a[1], "positions");
  const Tensor& turns = tensor(a[2], "turns");
  const How how{truth(a[3]), truth(a[5]), number(a[4])};
  const Maybe out = maybe(a[6], "out");
  if (x.dim() < 3) value_error("x must be (..., tokens, heads, head size)");
  no_gradient("turns", {&turns});
  no_tangent("rotate", {&x, get(out)});
  const at::Device dev = x.device();
  check_turns(turns, x.size(-1), dev);
  const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 2);
  Tensor pos = positions;
  if (pos.sizes() != lead && pos.dim() < (int64_t)lead.size() && pos.sizes() == lead.slice(lead.size() - pos.dim()))
    pos = pos.expand(lead);
  else if (lead.size() > 1 && pos.dim() > 1 && pos.sizes() != lead)
    value_error("positions are of the leading dimensions' shape, of the last of them, or one row for all tokens");
  const Tensor x3 = x.dim() > 3 ? x.flatten(0, -3) : x;
  pos = check_positions(pos, x3.size(0), dev);
  if (x.scalar_type() != at::kFloat) half_code(x);
  const c10::DeviceGuard guard(dev);
  const bool grad = at::GradMode::is_enabled();
  if (out) {
    if (out->sizes() != x.sizes() || out->scalar_type() != x.scalar_type() || out->device() != dev)
      value_error("out must have x's shape, type and device");
    if (grad && (x.requires_grad() || out->requires_grad())) value_error("out takes no gradient: rotate without it");
    check_written("out", *out, &x, {});
    const Tensor o3 = x.dim() > 3 ? out->view(x3.sizes()) : *out;
    const hipStream_t s = stream_of(x);
    check(unlocked([&] { return launch_rotation(x3, o3, pos, turns, how, s); }), "sdc_rope");
    written({&*out});
    Py_INCREF(a[6]);
    return a[6];
  }
  Tensor y;
  if (grad && x.requires_grad()) {
    y = Rotation::apply(x3, pos, turns, how.interleaved, how.mscale, how.inverse);
  } else {
    y = like(x3);
    const hipStream_t s = stream_of(x);
    check(unlocked([&] { return launch_rotation(x3, y, pos, turns, how, s); }), "sdc_rope");
  }
  return THPVariable_Wrap(x.dim() > 3 ? y.view(x.sizes()) : y);
}

// ------------------------------------------------------------------------------------------------- the paged cache
struct Step {
  Tensor qsl, lens, bt;
};
Step step(PyObject* qsl, PyObject* lens, PyObject* bt, const at::Device& dev) {
  Step s{tensor(qsl, "qsl"), tensor(lens, "seq_lens"), tensor(bt, "bt")};
  Tensor* t[3] = {&s.qsl, &s.lens, &s.bt};
  const char* name[3] = {"qsl", "seq_lens", "bt"};
  for (int i = 0; i < 3; ++i)
    if ((t[i]->scalar_type() != at::kInt && t[i]->scalar_type() != at::kLong) || t[i]->device() != dev)
      value_error(std::string(name[i]) + " must be an integer tensor on the tensors' device");
  if (s.lens.dim() != 1 || s.qsl.dim() != 1 || s.qsl.size(0) != s.lens.size(0) + 1 || s.bt.dim() != 2 ||
      s.bt.size(0) < s.lens.size(0))
    value_error("a step is qsl (requests + 1), seq_lens (requests) and bt (at least requests, pages)");
  for (Tensor* p : t)
    if (p->scalar_type() != at::kInt) *p = p->to(at::kInt);
  if (!s.qsl.is_contiguous()) s.qsl = s.qsl.contiguous();
  if (!s.lens.is_contiguous()) s.lens = s.lens.contiguous();
  if (s.bt.stride(1) != 1) s.bt = s.bt.contiguous();
  return s;
}

constexpr int E4M3 = 0, I8 = 1, SIXTEEN = 2;
int check_cache(const Tensor& kv, const Maybe& scales, std::optional<at::ScalarType> own, int64_t head, const at::Device& dev) {
  if (kv.dim() != 4 || kv.size(3) != 2 * head || kv.stride(3) != 1 || kv.size(0) < 1 || kv.device() != dev)
    value_error("a cache is (pages, kv heads, slots, 2 * head size) with the last dimension contiguous");
  const at::ScalarType t = kv.scalar_type();
  const int code = t == at::kFloat8_e4m3fn ? E4M3 : t == at::kChar ? I8 : own && t == *own ? SIXTEEN : -1;
  if (code < 0)
    value_error(std::string("a cache of ") + c10::toString(t) + ": float8_e4m3fn, int8, or the keys' own 16 bits");
  if (code != SIXTEEN && (!scales || scales->dim() != 3 || scales->size(0) != kv.size(0) || scales->size(1) != kv.size(1) ||
                          scales->size(2) != 2 || scales->scalar_type() != at::kFloat || scales->device() != dev ||
                          scales->stride(2) != 1))
    value_error("scales must be (pages, kv heads, 2) fp32 with the last dimension contiguous");
  return code;
}

// append(key, value, kv, scales, qsl, seq_lens, bt, turns, positions, interleaved, mscale, query, query_out)
PyObject* append(PyObject* const* a) {
  const Tensor &key = tensor(a[0], "key"), &value = tensor(a[1], "value"), &kv = tensor(a[2], "kv");
  const Maybe scales = maybe(a[3], "scales"), turns = maybe(a[7], "turns"), query = maybe(a[11], "query");
  Maybe positions = maybe(a[8], "positions"), out = maybe(a[12], "query_out");
  const bool interleaved = truth(a[9]);
  const double mscale = number(a[10]);
  no_gradient("kv_append", {&key, &value, &kv, get(scales), get(turns), get(query), get(out)});
  const at::Device dev = key.device();
  if (key.dim() != 3 || value.sizes() != key.sizes() || value.scalar_type() != key.scalar_type())
    value_error("key and value must be (tokens, kv heads, head size) of one type");
  const int64_t T = key.size(0), Hkv = key.size(1), D = key.size(2);
  const int dt = half_code(key);
  if (value.device() != dev || kv.dim() < 2 || kv.size(1) != Hkv)
    value_error("key, value and cache must have the same kv heads, on one device");
  const int code = check_cache(kv, scales, key.scalar_type(), D, dev);
  const int rot = turns ? check_turns(*turns, D, dev) : 0;
  const Step st = step(a[4], a[5], a[6], dev);
  if (positions) positions = check_positions(*positions, T, dev);
  int64_t Hq = 0;
  bool made = false;
  const c10::DeviceGuard guard(dev);
  if (!query) {
    if (out) value_error("query_out without query");
  } else {
    if (query->dim() != 3 || query->size(0) != T || query->size(2) != D || query->scalar_type() != key.scalar_type() ||
        query->device() != dev)
      value_error("query must be (tokens, heads, head size) of the keys' type");
    Hq = query->size(1);
    if (!out) {
      out = like(*query);
      made = true;
    } else if (out->sizes() != query->sizes() || out->scalar_type() != query->scalar_type() || out->device() != dev) {
      value_error("query_out must have query's shape, type and device");
    } else {
      check_written("query_out", *out, &*query, {&key, &value, &kv});
    }
  }
  check_written("kv", kv, nullptr, {&key, &value});
  if (code != SIXTEEN) check_written("scales", *scales, nullptr, {});
  const hipStream_t s = stream_of(key);
  const Maybe sc = code == SIXTEEN ? Maybe() : scales;
  check(unlocked([&] {
          return g_entry.append(
              dt, code, key.const_data_ptr(), key.stride(0), key.stride(1), key.stride(2), value.const_data_ptr(),
              value.stride(0), value.stride(1), value.stride(2), T, Hkv, D, kv.data_ptr(), kv.stride(0), kv.stride(1),
              kv.stride(2), kv.size(0), kv.size(2), (float*)ptr(sc), stride(sc, 0), stride(sc, 1),
              st.qsl.const_data_ptr<int32_t>(), st.lens.const_data_ptr<int32_t>(), st.lens.size(0),
              st.bt.const_data_ptr<int32_t>(), st.bt.stride(0), st.bt.size(1), ptr(positions),
              positions ? (int)positions->element_size() : 0, (const double*)ptr(turns), rot, interleaved, mscale, ptr(query),
              stride(query, 0), stride(query, 1), stride(query, 2), ptr(out), stride(out, 0), stride(out, 1), stride(out, 2),
              Hq, s);
        }),
        "sdc_kv_append");
  written({&kv, get(sc), made ? nullptr : get(out)});
  if (!query) Py_RETURN_NONE;
  if (made) return THPVariable_Wrap(*out);
  Py_INCREF(a[12]);
  return a[12];
}

// attend(q, kv, scales, qsl, seq_lens, bt, scale, window, max_seq_len, out, return_lse)
PyObject* attend(PyObject* const* a) {
  const Tensor &q = tensor(a[0], "q"), &kv = tensor(a[1], "kv");
  const Maybe scales = maybe(a[2], "scales");
  Maybe out = maybe(a[9], "out");
  const int64_t window = integer(a[7]);
  const bool want = truth(a[10]);
  no_gradient("kv_attend", {&q, &kv, get(scales), get(out)});
  if (q.dim() != 3) value_error("q must be (tokens, heads, head size)");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  const at::Device dev = q.device();
  const int dt = half_code(q);
  const int code = check_cache(kv, scales, std::nullopt, D, dev);
  const int64_t Hkv = kv.size(1), N = kv.size(2);
  if (Hkv < 1 || Hq < 1 || Hq % Hkv || D > 256)
    value_error(std::to_string(Hq) + " heads of " + std::to_string(D) + " over " + std::to_string(Hkv) +
                " kv heads: a multiple of them, and head sizes up to 256");
  if (window < 0) value_error("window must not be negative (0: none)");
  const float scale = a[6] == Py_None ? (float)(1.0 / std::sqrt((double)D)) : (float)number(a[6]);
  if (!std::isfinite(scale)) value_error("scale must be a finite number");
  const Step st = step(a[3], a[4], a[5], dev);
  const int64_t R = st.lens.size(0), W = st.bt.size(1);
  int64_t most = W * N;
  if (a[8] != Py_None) most = std::min(most, integer(a[8]));
  if (most < 0) value_error("max_seq_len must not be negative");
  const c10::DeviceGuard guard(dev);
  bool made = false;
  if (!out) {
    out = at::empty({T, Hq, D}, q.options());
    made = true;
  } else if (out->sizes() != q.sizes() || out->scalar_type() != q.scalar_type() || out->device() != dev) {
    value_error("out must have q's shape, type and device");
  } else {
    check_written("out", *out, &q, {&kv});
  }
  Tensor lse, ws;
  if (want) lse = at::empty({T, Hq}, q.options().dtype(at::kFloat));
  // (a workspace of the call's own: the allocator orders its memory by stream, and within a captured graph keeps it)
  const int64_t need = g_entry.workspace(T, R, Hq, Hkv, D, N, most, window);
  if (need) ws = at::empty({need}, q.options().dtype(at::kByte));
  const hipStream_t s = stream_of(q);
  check(unlocked([&] {
          return g_entry.attend(dt, code, q.const_data_ptr(), q.stride(0), q.stride(1), q.stride(2), out->data_ptr(),
                                out->stride(0), out->stride(1), out->stride(2), want ? lse.data_ptr<float>() : nullptr, Hq, T,
                                Hq, D, kv.const_data_ptr(), kv.stride(0), kv.stride(1), kv.stride(2), kv.size(0), Hkv, N,
                                (const float*)ptr(scales), stride(scales, 0), stride(scales, 1),
                                st.qsl.const_data_ptr<int32_t>(), st.lens.const_data_ptr<int32_t>(), R,
                                st.bt.const_data_ptr<int32_t>(), st.bt.stride(0), W, scale, window, most,
                                need ? ws.data_ptr() : nullptr, need, s);
        }),
        "sdc_kv_attend");
  PyObject* o = a[9];
  if (made) {
    o = THPVariable_Wrap(*out);
  } else {
    written({&*out});
    Py_INCREF(o);
  }
  if (!want || !o) return o;
  PyObject* e = THPVariable_Wrap(lse);
  if (!e) {
    Py_DECREF(o);
    return nullptr;
  }
  PyObject* r = PyTuple_Pack(2, o, e);
  Py_DECREF(o);
  Py_DECREF(e);
  return r;
}

// ------------------------------------------------------------------------------------------------------- the module
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, not %zd", N, n);
    return nullptr;
  }
  if (!g_entry.rope) {
    PyErr_SetString(PyExc_RuntimeError, "the library is not bound");
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Raised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// bind(addresses of sdc_rope, sdc_kv_append, sdc_kv_attend_workspace, sdc_kv_attend; check; HipLibraryError)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "6 arguments expected");
    return nullptr;
  }
  void* p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an entry point is missing");
      return nullptr;
    }
  }
  g_entry = Entry{(decltype(&sdc_rope))p[0], (decltype(&sdc_kv_append))p[1], (decltype(&sdc_kv_attend_workspace))p[2],
                  (decltype(&sdc_kv_attend))p[3]};
  PyObject** keep[2] = {&g_check, &g_error};
  for (int i = 0; i < 2; ++i) {
    Py_INCREF(a[4 + i]);
    Py_XSETREF(*keep[i], a[4 + i]);
  }
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"bind", (PyCFunction)(void*)bind, METH_FASTCALL, nullptr},
    {"rotate", (PyCFunction)(void*)call<rotate, 7>, METH_FASTCALL, nullptr},
    {"append", (PyCFunction)(void*)call<append, 13>, METH_FASTCALL, nullptr},
    {"attend", (PyCFunction)(void*)call<attend, 11>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&g_module); }
