// The paged cache's operators as Python calls them: operand checks and argument structs in C++.  A served step of single
// tokens is over in microseconds, and the same checks took eight of them in Python.  Built against torch's headers as a
// CPython module (dark_amd/_bind.so); the entry points of libdark_hip.so are handed over by address (init), so that it works
// on whichever build of the library dark_amd/_hip.py has loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/dark_hip.h"

namespace {

decltype(&dark_qk_norm_rope) f_norm_rope = nullptr;
decltype(&dark_kv_append) f_append = nullptr;
decltype(&dark_paged_attention) f_attend = nullptr;
decltype(&dark_paged_attention_workspace_bytes) f_workspace = nullptr;
decltype(&dark_hip_last_error) f_error = nullptr;
PyObject* dark_error = nullptr;

struct Refusal : std::runtime_error {
  PyObject* type;
  Refusal(PyObject* t, const std::string& m) : std::runtime_error(m), type(t) {}
};
[[noreturn]] void refuse(const std::string& m) { throw Refusal(PyExc_ValueError, m); }
void need(bool ok, const char* m) {
  if (!ok) refuse(m);
}

std::string shape_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}
std::string name_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return std::string("torch.") + at::toString(t);
  }
}

const at::Tensor* given(PyObject* o, const char* name) {   // nullptr: None
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) throw Refusal(PyExc_TypeError, std::string(name) + " must be a tensor, got " + Py_TYPE(o)->tp_name);
  return &THPVariable_Unpack(o);
}
const at::Tensor& wanted(PyObject* o, const char* name) {
  const at::Tensor* t = given(o, name);
  if (!t) throw Refusal(PyExc_TypeError, std::string(name) + " must be a tensor, got NoneType");
  return *t;
}

struct Call {
  c10::Device dev = c10::Device(c10::kCPU);
  at::ScalarType dt = at::kFloat;
  int64_t es = 4;
  bool grad = c10::GradMode::is_enabled();
  bool tangents = c10::AutogradState::get_tls_state().get_fw_grad_mode();

  void open(const at::Tensor& t) {
    if (!t.is_cuda()) throw Refusal(PyExc_RuntimeError, "dark_amd runs on a HIP device only");
    dt = t.scalar_type();
    if (dt != at::kFloat && dt != at::kBFloat16) refuse("dtype " + name_of(dt) + ": float32 and bfloat16 only");
    es = dt == at::kFloat ? 4 : 2;
    dev = t.device();
  }
  int32_t dtype() const { return dt == at::kBFloat16 ? DARK_BF16 : DARK_F32; }

  void check(const at::Tensor& t, const char* name, at::ScalarType type, int64_t dim) const {
    if (t.device() != dev) refuse(std::string(name) + " is on " + t.device().str() + ", expected " + dev.str());
    if (t.scalar_type() != type) refuse(std::string(name) + " is " + name_of(t.scalar_type()) + ", expected " + name_of(type));
    if (t.dim() != dim) refuse(std::string(name) + " has " + std::to_string(t.dim()) + " dimensions, expected " + std::to_string(dim));
    if (grad && t.requires_grad())
      throw Refusal(PyExc_RuntimeError, std::string(name) + " requires gradients: the cache's operators have no backward (use torch.no_grad())");
    if (tangents && (type == at::kFloat || type == at::kBFloat16) && t._fw_grad(0).defined())   // (whole numbers have none)
      throw Refusal(PyExc_RuntimeError, std::string(name) + " carries a forward-mode tangent: the cache's operators have no derivative");
  }

  // 16-byte pointer and strides, contiguous last dimension (a dimension of one has no stride of its own)
  bool fits(const at::Tensor& t) const {
    const int64_t n = t.dim();
    if ((uintptr_t)t.data_ptr() & 15) return false;
    if (t.stride(n - 1) != 1 && t.size(n - 1) > 1) return false;
    for (int64_t i = 0; i + 1 < n; ++i)
      if (t.size(i) > 1 && t.stride(i) * es % 16 != 0) return false;
    return true;
  }
  void writable(const at::Tensor& t, const char* name) const {
    if (t.numel() == 0) return;
    if (!fits(t)) refuse(std::string(name) + ": pointer and strides must be multiples of 16 bytes, the last dimension contiguous");
    for (int64_t i = 0; i + 1 < t.dim(); ++i)
      if (t.size(i) > 1 && t.stride(i) <= 0) refuse(std::string(name) + ": an expanded tensor cannot be written");
  }
  // what a call wrote into a tensor of the caller's: autograd refuses to go back through what it saved of it before
  static void wrote(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  static int64_t stride(const at::Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 0; }

  // a [T, heads, HD] input, copied only where its strides or its alignment do not fit
  at::Tensor rows(const at::Tensor& t, const char* name, int64_t T, int64_t HD) const {
    check(t, name, dt, 3);
    if (t.size(0) != T || t.size(2) != HD)
      refuse(std::string(name) + " is " + shape_of(t) + ", expected [" + std::to_string(T) + ", heads, " + std::to_string(HD) + "]");
    return fits(t) ? t : t.detach().clone(at::MemoryFormat::Contiguous);
  }
  at::Tensor out(const at::Tensor* t, const char* name, const at::Tensor& like) const {
    if (!t) return at::empty(like.sizes(), like.options().requires_grad(false));
    check(*t, name, dt, 3);
    if (t->sizes() != like.sizes()) refuse(std::string(name) + " is " + shape_of(*t) + ", expected " + shape_of(like));
    writable(*t, name);
    return *t;
  }
  const void* vec(PyObject* o, const char* name, at::ScalarType type, int64_t n) const {
    const at::Tensor* t = given(o, name);
    if (!t) return nullptr;
    check(*t, name, type, 1);
    if (t->size(0) != n || !t->is_contiguous()) refuse(std::string(name) + " must be contiguous with " + std::to_string(n) + " elements");
    return t->data_ptr();
  }
  struct Turn {
    const float *cos = nullptr, *sin = nullptr;
    const int32_t* pos = nullptr;
    int32_t n = 0;
  };
  Turn tables(PyObject* c, PyObject* s, PyObject* p, int64_t T, int64_t HD) const {
    Turn r;
    if (c == Py_None && s == Py_None) return r;
    need(c != Py_None && s != Py_None && p != Py_None, "cos, sin and pos go together");
    const at::Tensor &tc = wanted(c, "cos"), &ts = wanted(s, "sin");
    check(tc, "cos", at::kFloat, 2);
    check(ts, "sin", at::kFloat, 2);
    if (tc.size(0) < 1 || tc.size(0) >= (1ll << 31) || tc.size(1) * 2 != HD || ts.sizes() != tc.sizes() || !tc.is_contiguous() || !ts.is_contiguous())
      refuse("cos and sin must be contiguous [max_pos, " + std::to_string(HD / 2) + "]");
    r.cos = tc.const_data_ptr<float>();
    r.sin = ts.const_data_ptr<float>();
    r.pos = (const int32_t*)vec(p, "pos", at::kInt, T);
    r.n = (int32_t)tc.size(0);
    return r;
  }
  dark_paged_kv cache(PyObject* ko, PyObject* vo) const {
    const at::Tensor &k = wanted(ko, "k_cache"), &v = wanted(vo, "v_cache");
    check(k, "k_cache", dt, 4);
    check(v, "v_cache", dt, 4);
    need(k.sizes() == v.sizes() && k.strides() == v.strides(), "k_cache and v_cache must have the same shape and strides");
    const int64_t page = k.size(1);
    if (page < 1 || (page & (page - 1))) refuse("page size " + std::to_string(page) + " must be a power of two");
    need(k.size(0) < (1ll << 31) && page < (1ll << 31) && k.size(2) < (1ll << 31) && k.size(3) < (1ll << 31), "the cache is too large");
    writable(k, "k_cache");
    writable(v, "v_cache");
    dark_paged_kv kv = {};
    kv.k = k.data_ptr();
    kv.v = v.data_ptr();
    kv.page_stride = stride(k, 0);
    kv.slot_stride = stride(k, 1);
    kv.head_stride = stride(k, 2);
    kv.dtype = dtype();
    kv.n_pages = (int32_t)k.size(0);
    kv.page_size = (int32_t)page;
    kv.n_kv_heads = (int32_t)k.size(2);
    kv.head_dim = (int32_t)k.size(3);
    return kv;
  }
};

void done(int rc) {
  if (rc != DARK_OK) throw Refusal(dark_error, "dark_hip error " + std::to_string(rc) + ": " + f_error());
}
int64_t whole(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refusal(nullptr, name);
  if (v < 0 || v >= (1ll << 31)) refuse(std::string(name) + "=" + std::to_string(v) + " is out of range");
  return v;
}
float real(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refusal(nullptr, name);
  return (float)v;
}

template <typename F>
PyObject* guarded(F body) {
  try {
    if (!f_attend) throw Refusal(PyExc_RuntimeError, "the HIP library is not bound");
    return body();
  } catch (const Refusal& e) {
    if (e.type) PyErr_SetString(e.type, e.what());   // (null: Python has set the error)
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// (stream, q, k, q_weight, k_weight, cos, sin, pos, eps, q_out, k_out)
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 11, "qk_norm_rope: 11 arguments");
    Call c;
    const at::Tensor &q0 = wanted(a[1], "q"), &k0 = wanted(a[2], "k");
    c.open(q0);
    const int64_t T = q0.dim() == 3 ? q0.size(0) : 0, HD = q0.dim() == 3 ? q0.size(2) : 0;
    const at::Tensor q = c.rows(q0, "q", T, HD), k = c.rows(k0, "k", T, HD);
    const at::Tensor qo = c.out(given(a[9], "q_out"), "q_out", q0), ko = c.out(given(a[10], "k_out"), "k_out", k0);
    dark_qk_norm_rope_args p = {};
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.q_out = qo.data_ptr(); p.k_out = ko.data_ptr();
    p.q_w = (const float*)c.vec(a[3], "q_weight", at::kFloat, HD);
    p.k_w = (const float*)c.vec(a[4], "k_weight", at::kFloat, HD);
    const Call::Turn t = c.tables(a[5], a[6], a[7], T, HD);
    p.rope_cos = t.cos; p.rope_sin = t.sin; p.pos = t.pos; p.max_pos = t.n;
    p.q_ts = c.stride(q, 0); p.q_hs = c.stride(q, 1); p.k_ts = c.stride(k, 0); p.k_hs = c.stride(k, 1);
    p.qo_ts = c.stride(qo, 0); p.qo_hs = c.stride(qo, 1); p.ko_ts = c.stride(ko, 0); p.ko_hs = c.stride(ko, 1);
    need(T < (1ll << 30) && q.size(1) < (1ll << 30) && k.size(1) < (1ll << 30) && HD < (1ll << 30), "too large");
    p.dtype = c.dtype(); p.n_tokens = (int32_t)T; p.n_heads = (int32_t)q.size(1); p.n_kv_heads = (int32_t)k.size(1); p.head_dim = (int32_t)HD;
    p.eps = real(a[8], "eps");
    void* st = PyLong_AsVoidPtr(a[0]);
    const c10::DeviceGuard guard(c.dev);
    done(f_norm_rope(&p, st));
    if (a[9] != Py_None) c.wrote(qo);
    if (a[10] != Py_None) c.wrote(ko);
    PyObject *x = a[9] == Py_None ? THPVariable_Wrap(qo) : (Py_INCREF(a[9]), a[9]);
    PyObject *y = a[10] == Py_None ? THPVariable_Wrap(ko) : (Py_INCREF(a[10]), a[10]);
    PyObject* r = PyTuple_Pack(2, x, y);
    Py_DECREF(x);
    Py_DECREF(y);
    return r;
  });
}

// (stream, k, v, k_cache, v_cache, slots, cos, sin, pos, q, q_out, q_weight, k_weight, eps)
PyObject* append_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 14, "append_kv: 14 arguments");
    Call c;
    const at::Tensor &k0 = wanted(a[1], "k"), &v0 = wanted(a[2], "v");
    c.open(k0);
    const int64_t T = k0.dim() == 3 ? k0.size(0) : 0, HD = k0.dim() == 3 ? k0.size(2) : 0;
    dark_kv_append_args p = {};
    p.kv = c.cache(a[3], a[4]);
    const at::Tensor k = c.rows(k0, "k", T, HD), v = c.rows(v0, "v", T, HD);
    if (p.kv.n_kv_heads != k.size(1) || p.kv.head_dim != HD || v.size(1) != k.size(1))
      refuse("k is " + shape_of(k0) + ", v " + shape_of(v0) + ", the cache holds " + std::to_string(p.kv.n_kv_heads) + " heads of " +
             std::to_string(p.kv.head_dim));
    const at::Tensor *q0 = given(a[9], "q"), *qo0 = given(a[10], "q_out");
    at::Tensor q, qo;
    if (q0) {
      q = c.rows(*q0, "q", T, HD);
      qo = c.out(qo0, "q_out", *q0);
      p.q = q.data_ptr(); p.q_out = qo.data_ptr(); p.n_heads = (int32_t)q.size(1);
      p.q_ts = c.stride(q, 0); p.q_hs = c.stride(q, 1); p.qo_ts = c.stride(qo, 0); p.qo_hs = c.stride(qo, 1);
    } else {
      need(!qo0, "q_out without q");
    }
    p.k = k.data_ptr(); p.v = v.data_ptr();
    p.k_ts = c.stride(k, 0); p.k_hs = c.stride(k, 1); p.v_ts = c.stride(v, 0); p.v_hs = c.stride(v, 1);
    wanted(a[5], "slots");
    p.slots = (const int64_t*)c.vec(a[5], "slots", at::kLong, T);
    const Call::Turn t = c.tables(a[6], a[7], a[8], T, HD);
    p.rope_cos = t.cos; p.rope_sin = t.sin; p.pos = t.pos; p.max_pos = t.n;
    p.q_w = (const float*)c.vec(a[11], "q_weight", at::kFloat, HD);
    p.k_w = (const float*)c.vec(a[12], "k_weight", at::kFloat, HD);
    p.eps = real(a[13], "eps");
    need(T < (1ll << 30), "too many tokens");
    p.n_tokens = (int32_t)T;
    void* st = PyLong_AsVoidPtr(a[0]);
    const c10::DeviceGuard guard(c.dev);
    // (empty vectors have no pointer)
    if (T > 0) {
      done(f_append(&p, st));
      c.wrote(*given(a[3], "k_cache"));
      c.wrote(*given(a[4], "v_cache"));
      if (qo0) c.wrote(qo);
    }
    if (!q0) Py_RETURN_NONE;
    if (a[10] != Py_None) return Py_INCREF(a[10]), a[10];
    return THPVariable_Wrap(qo);
  });
}

// (stream, q, k_cache, v_cache, block_table, cu_q, kv_len, max_q, max_kv, q_index, key_mask, causal, scale, out, return_lse)
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 15, "paged_attention: 15 arguments");
    Call c;
    const at::Tensor& q0 = wanted(a[1], "q");
    c.open(q0);
    const int64_t T = q0.dim() == 3 ? q0.size(0) : 0, HD = q0.dim() == 3 ? q0.size(2) : 0;
    dark_paged_attention_args p = {};
    p.kv = c.cache(a[2], a[3]);
    const at::Tensor q = c.rows(q0, "q", T, HD);
    const int64_t H = q.size(1);
    if (p.kv.head_dim != HD || p.kv.n_kv_heads < 1 || H % p.kv.n_kv_heads)
      refuse("q is " + shape_of(q0) + ", the cache holds " + std::to_string(p.kv.n_kv_heads) + " heads of " + std::to_string(p.kv.head_dim));
    const at::Tensor& table = wanted(a[4], "block_table");
    c.check(table, "block_table", at::kInt, 2);
    const int64_t B = table.size(0), width = table.size(1);
    need(B < (1ll << 31) && width < (1ll << 31) && T < (1ll << 30) && H < (1ll << 31), "too large");
    need(width <= 1 || table.stride(1) == 1, "block_table rows must be contiguous");
    p.block_table = (const int32_t*)table.data_ptr();
    p.table_stride = B > 1 ? table.stride(0) : width;
    need(p.table_stride >= 0, "block_table rows must be contiguous");
    p.max_q = (int32_t)whole(a[7], "max_q");
    p.max_kv = (int32_t)whole(a[8], "max_kv");
    if (const at::Tensor* m = given(a[10], "key_mask")) {
      const at::ScalarType mt = m->scalar_type();
      if (mt != at::kByte && mt != at::kBool) refuse("key_mask is " + name_of(mt) + ", expected uint8 or bool");
      c.check(*m, "key_mask", mt, 2);
      if (m->size(0) != B || m->size(1) < p.max_kv || (m->size(1) > 1 && m->stride(1) != 1) || m->stride(0) < 0)
        refuse("key_mask is " + shape_of(*m) + ", expected [" + std::to_string(B) + ", >= " + std::to_string(p.max_kv) + "] with contiguous rows");
      p.key_mask = (const uint8_t*)m->data_ptr();
      p.mask_stride = B > 1 ? m->stride(0) : 0;
    }
    wanted(a[5], "cu_q");
    wanted(a[6], "kv_len");
    p.cu_q = (const int32_t*)c.vec(a[5], "cu_q", at::kInt, B + 1);
    p.kv_len = (const int32_t*)c.vec(a[6], "kv_len", at::kInt, B);
    p.q_index = (const int32_t*)c.vec(a[9], "q_index", at::kInt, T);
    const at::Tensor out = c.out(given(a[13], "out"), "out", q0);
    need(out.numel() == 0 || out.data_ptr() != q.data_ptr(), "out must not overlap q");
    at::Tensor lse;
    const int want = PyObject_IsTrue(a[14]), causal = PyObject_IsTrue(a[11]);
    if (want < 0 || causal < 0) throw Refusal(nullptr, "");
    if (want) {
      lse = at::empty({T, H}, q0.options().dtype(at::kFloat).requires_grad(false));
      p.lse = lse.data_ptr<float>();
    }
    p.q = q.data_ptr(); p.out = out.data_ptr();
    p.q_ts = c.stride(q, 0); p.q_hs = c.stride(q, 1); p.o_ts = c.stride(out, 0); p.o_hs = c.stride(out, 1);
    p.n_tokens = (int32_t)T; p.n_heads = (int32_t)H; p.n_seqs = (int32_t)B; p.table_width = (int32_t)width;
    p.causal = causal;
    p.scale = a[12] == Py_None ? (float)(1.0 / std::sqrt((double)HD)) : real(a[12], "scale");
    void* st = PyLong_AsVoidPtr(a[0]);
    const c10::DeviceGuard guard(c.dev);
    at::Tensor ws;
    if (const size_t bytes = f_workspace(&p)) {   // (torch's allocator orders its reuse behind this stream's work)
      ws = at::empty({(int64_t)bytes}, q0.options().dtype(at::kByte).requires_grad(false));
      p.workspace = ws.data_ptr();
      p.workspace_bytes = (int64_t)bytes;
    }
    if (T > 0) {
      done(f_attend(&p, st));
      if (a[13] != Py_None) c.wrote(out);
    }
    PyObject* o = a[13] == Py_None ? THPVariable_Wrap(out) : (Py_INCREF(a[13]), a[13]);
    if (!want) return o;
    PyObject* l = THPVariable_Wrap(lse);
    PyObject* r = PyTuple_Pack(2, o, l);
    Py_DECREF(o);
    Py_DECREF(l);
    return r;
  });
}

// (DarkHipError, addresses of dark_qk_norm_rope, dark_kv_append, dark_paged_attention, its workspace_bytes, dark_hip_last_error)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "init: 6 arguments");
    return nullptr;
  }
  Py_INCREF(a[0]);
  Py_XDECREF(dark_error);
  dark_error = a[0];
  f_norm_rope = (decltype(f_norm_rope))PyLong_AsVoidPtr(a[1]);
  f_append = (decltype(f_append))PyLong_AsVoidPtr(a[2]);
  f_attend = (decltype(f_attend))PyLong_AsVoidPtr(a[3]);
  f_workspace = (decltype(f_workspace))PyLong_AsVoidPtr(a[4]);
  f_error = (decltype(f_error))PyLong_AsVoidPtr(a[5]);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"init", (PyCFunction)(void (*)(void))init, METH_FASTCALL, nullptr},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))qk_norm_rope, METH_FASTCALL, nullptr},
    {"append_kv", (PyCFunction)(void (*)(void))append_kv, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind(void) {
  PyObject* m = PyModule_Create(&module);
  // (the argument structs this file was compiled with: whoever binds the library compares)
  if (m && PyModule_AddIntConstant(m, "ABI_VERSION", DARK_HIP_ABI_VERSION) < 0) Py_CLEAR(m);
  return m;
}
