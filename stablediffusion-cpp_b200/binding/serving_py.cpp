// serving_py.cpp - the calls of the operators for several requests at once, from torch tensors
// to the C ABI. At one token a call's GPU time is 2 to 8 us, and tests of a dozen tensors and 25
// converted arguments cost 10 us in Python. Each function tests its arguments, allocates what the
// caller did not bring, and calls the library on the current stream. It returns the outputs, the
// library's error code, or None where an argument does not fit: backend.py then names the fault.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <mutex>

namespace {

using at::ScalarType;
using at::Tensor;

// The library's functions, by address (bind).
int (*set_stream)(void*);
int (*qk_norm_rope)(int64_t, const void*, int64_t, int, const void*, int64_t, int, int, int64_t, int64_t, const float*,
                    const float*, float, const float*, const float*, int64_t, const int32_t*, int, void*, int64_t, void*,
                    int64_t, int);
int64_t (*lora_workspace)(int64_t, int64_t, int64_t, const void*, int64_t, int, const uint16_t*, int64_t, int64_t, int64_t,
                          const uint16_t*, int64_t, const uint16_t*, int64_t);
int (*linear_lora)(int64_t, int64_t, int64_t, const void*, int64_t, int, const uint16_t*, int64_t, const float*,
                   const int32_t*, int64_t, int64_t, const uint16_t*, int64_t, const uint16_t*, int64_t, const float*, void*,
                   int64_t, int, void*, int64_t);
int64_t (*attention_workspace)(int, int64_t, int64_t, int, int, int64_t);
int (*attention_ragged)(const void*, int64_t, const void*, int64_t, const void*, int64_t, int, void*, int64_t, int, int64_t,
                        int64_t, int, const int32_t*, const int32_t*, const int32_t*, const int32_t*, int64_t, int64_t, int,
                        int, int64_t, float, float, const float*, int, const int32_t*, void*, int64_t);

// One call at a time: the library's first call of a kind sets attributes for all.
std::mutex call_mutex;

struct Refused {};  // an argument does not fit

void want(bool ok) {
  if (!ok) throw Refused{};
}
const Tensor& tensor(PyObject* o) {
  want(THPVariable_Check(o));
  return THPVariable_Unpack(o);
}
ScalarType dtype_of(PyObject* o) {
  want(THPDtype_Check(o));
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
int code(ScalarType t) {  // SDB200_F32, SDB200_BF16, SDB200_F16
  want(t == ScalarType::Float || t == ScalarType::BFloat16 || t == ScalarType::Half);
  return t == ScalarType::Float ? 0 : t == ScalarType::BFloat16 ? 1 : 2;
}
bool strided(const Tensor& t) { return t.layout() == at::kStrided; }
int current_device_of(const Tensor& t) {
  want(t.is_cuda() && strided(t));
  const int dev = t.get_device();
  want(dev == c10::cuda::current_device());
  return dev;
}
void on(const Tensor& t, int dev, ScalarType type) {
  want(t.is_cuda() && strided(t) && t.get_device() == dev && t.scalar_type() == type);
}
// A contiguous vector, or null for None.
template <class T>
const T* vec(PyObject* o, int dev, ScalarType type, int64_t n) {
  if (o == Py_None) return nullptr;
  const Tensor& t = tensor(o);
  on(t, dev, type);
  want(t.dim() == 1 && t.size(0) == n && t.is_contiguous());
  return static_cast<const T*>(t.data_ptr());
}
const int32_t* index(PyObject* o, int dev, int64_t n) {
  want(o != Py_None);
  return vec<int32_t>(o, dev, ScalarType::Int, n);
}
// Row pitches, in elements, of dense heads, dense rows and adapters one after another.
int64_t head_pitch(const Tensor& t) {
  const int64_t h = t.size(1), d = t.size(2);
  want((t.stride(2) == 1 || d <= 1) && (t.stride(1) == d || h <= 1));
  return t.size(0) > 1 ? t.stride(0) : h * d;
}
int64_t row_pitch(const Tensor& t) {
  want(t.stride(1) == 1 || t.size(1) <= 1);
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}
int64_t stack_pitch(const Tensor& t) {
  const int64_t n = t.size(0), rows = t.size(1), cols = t.size(2);
  if (t.numel() == 0) return cols;
  const int64_t ld = rows > 1 ? t.stride(1) : n > 1 ? t.stride(0) : cols;
  want((t.stride(2) == 1 || cols <= 1) && (n <= 1 || t.stride(0) == rows * ld));
  return ld;
}
double number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw Refused{};
  return x;
}
int64_t integer(PyObject* o) {
  int over = 0;
  const long long x = PyLong_AsLongLongAndOverflow(o, &over);
  if (x == -1 && !over && PyErr_Occurred()) throw Refused{};
  return over ? (over > 0 ? std::numeric_limits<int64_t>::max() : std::numeric_limits<int64_t>::min()) : x;
}
bool flag(PyObject* o) {
  const int x = PyObject_IsTrue(o);
  want(x >= 0);
  return x != 0;
}
Tensor empty(at::IntArrayRef size, const Tensor& like, ScalarType type) { return at::empty(size, like.options().dtype(type)); }

// The call on the current stream, without the interpreter's lock (a launch may wait for room).
template <class F>
int run(int dev, F call) {
  void* const stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  {
    std::lock_guard<std::mutex> lock(call_mutex);
    rc = set_stream(stream);
    if (rc == 0) rc = call();
  }
  Py_END_ALLOW_THREADS;
  return rc;
}

template <class F>
PyObject* guarded(F body) {
  try {
    return body();
  } catch (const Refused&) {
    PyErr_Clear();
    Py_RETURN_NONE;
  } catch (const std::exception& e) {  // an allocation failed
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// q, k, cos, sin, gq, gk, eps, pos, interleaved, out_dtype, q_out, k_out
PyObject* py_qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    want(nargs == 12);
    const Tensor& q = tensor(a[0]);
    const ScalarType in = q.scalar_type();
    const int in_code = code(in), dev = current_device_of(q);
    want(q.dim() == 3);
    const int64_t T = q.size(0), heads = q.size(1), d = q.size(2);
    const Tensor &cos = tensor(a[2]), &sin = tensor(a[3]);
    on(cos, dev, ScalarType::Float);
    on(sin, dev, ScalarType::Float);
    want(cos.dim() == 2 && cos.is_contiguous() && sin.is_contiguous() && sin.sizes() == cos.sizes());
    const float *gq = vec<float>(a[4], dev, ScalarType::Float, d), *gk = vec<float>(a[5], dev, ScalarType::Float, d);
    const int32_t* pos = vec<int32_t>(a[7], dev, ScalarType::Int, T);
    ScalarType out = in;
    if (a[9] != Py_None)
      out = dtype_of(a[9]);
    else if (a[10] != Py_None)
      out = tensor(a[10]).scalar_type();
    const int out_code = code(out);
    const float eps = static_cast<float>(number(a[6]));
    const bool inter = flag(a[8]);
    // Views must fit before anything is allocated.
    Tensor q_out, k_out;
    int64_t ldqo = heads * d, kv = 0, ldk = 0, ldko = 0;
    const int64_t ldq = head_pitch(q);
    const bool have_k = a[1] != Py_None;
    if (a[10] != Py_None) {
      q_out = tensor(a[10]);
      on(q_out, dev, out);
      want(q_out.sizes() == q.sizes());
      ldqo = head_pitch(q_out);
    }
    if (have_k) {
      const Tensor& k = tensor(a[1]);
      on(k, dev, in);
      want(k.dim() == 3 && k.size(0) == T && k.size(2) == d);
      kv = k.size(1);
      ldk = head_pitch(k);
      ldko = kv * d;
      if (a[11] != Py_None) {
        k_out = tensor(a[11]);
        on(k_out, dev, out);
        want(k_out.sizes() == k.sizes());
        ldko = head_pitch(k_out);
      } else {
        k_out = empty({T, kv, d}, q, out);
      }
    } else if (a[11] != Py_None) {
      on(tensor(a[11]), dev, out);
    }
    if (!q_out.defined()) q_out = empty({T, heads, d}, q, out);
    const void *qp = q.data_ptr(), *kp = have_k ? tensor(a[1]).data_ptr() : nullptr;
    void *qo = q_out.data_ptr(), *ko = have_k ? k_out.data_ptr() : nullptr;
    const float *cp = static_cast<const float*>(cos.data_ptr()), *sp = static_cast<const float*>(sin.data_ptr());
    const int64_t n_pos = cos.size(0), rot = cos.size(1);
    const int rc = run(dev, [&]() {
      return qk_norm_rope(T, qp, ldq, (int)heads, kp, ldk, (int)kv, in_code, d, rot, gq, gk, eps, cp, sp, n_pos, pos,
                          inter ? 1 : 0, qo, ldqo, ko, ldko, out_code);
    });
    if (rc) return PyLong_FromLong(rc);
    PyObject* r = PyTuple_New(2);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, a[10] != Py_None ? Py_NewRef(a[10]) : THPVariable_Wrap(std::move(q_out)));
    PyTuple_SET_ITEM(r, 1, !have_k ? Py_NewRef(Py_None) : a[11] != Py_None ? Py_NewRef(a[11]) : THPVariable_Wrap(std::move(k_out)));
    return r;
  });
}

// x, W, A, B, rows, scale, bias, out_dtype, out
PyObject* py_linear_lora(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    want(nargs == 9);
    const Tensor &x = tensor(a[0]), &W = tensor(a[1]), &A = tensor(a[2]), &B = tensor(a[3]);
    const ScalarType in = x.scalar_type();
    want(in == ScalarType::Float || in == ScalarType::BFloat16);
    const int dev = current_device_of(x);
    want(x.dim() == 2 && W.dim() == 2 && A.dim() == 3 && B.dim() == 3);
    const int64_t T = x.size(0), K = x.size(1), N = W.size(0), n = A.size(0), r = A.size(1);
    want(W.size(1) == K && A.size(2) == K && B.size(0) == n && B.size(1) == N && B.size(2) == r);
    on(W, dev, ScalarType::BFloat16);
    on(A, dev, ScalarType::BFloat16);
    on(B, dev, ScalarType::BFloat16);
    const int32_t* rows = index(a[4], dev, T);
    const float *scale = vec<float>(a[5], dev, ScalarType::Float, n), *bias = vec<float>(a[6], dev, ScalarType::Float, N);
    const int64_t ldx = row_pitch(x), ldw = row_pitch(W), lda = stack_pitch(A), ldb = stack_pitch(B);
    int64_t ldy = N;
    Tensor y;
    if (a[8] != Py_None) {
      y = tensor(a[8]);
      on(y, dev, y.scalar_type());
      want(y.dim() == 2 && y.size(0) == T && y.size(1) == N);
      ldy = row_pitch(y);
    }
    const ScalarType out = y.defined() ? y.scalar_type() : dtype_of(a[7]);
    want(out == ScalarType::Float || out == ScalarType::BFloat16);
    const void* xp = x.data_ptr();
    const auto *wp = static_cast<const uint16_t*>(W.data_ptr()), *ap = static_cast<const uint16_t*>(A.data_ptr()),
               *bp = static_cast<const uint16_t*>(B.data_ptr());
    const int x_bf16 = in == ScalarType::BFloat16, y_bf16 = out == ScalarType::BFloat16;
    const int64_t need = lora_workspace(T, N, K, xp, ldx, x_bf16, wp, ldw, n, r, ap, lda, bp, ldb);
    if (!y.defined()) y = empty({T, N}, x, out);
    Tensor ws;
    if (need > 0) ws = empty({need}, x, ScalarType::Byte);
    void *yp = y.data_ptr(), *wsp = need > 0 ? ws.data_ptr() : nullptr;
    const int rc = run(dev, [&]() {
      return linear_lora(T, N, K, xp, ldx, x_bf16, wp, ldw, bias, rows, n, r, ap, lda, bp, ldb, scale, yp, ldy, y_bf16, wsp,
                         need);
    });
    if (rc) return PyLong_FromLong(rc);
    return a[8] != Py_None ? Py_NewRef(a[8]) : THPVariable_Wrap(std::move(y));
  });
}

// q, k, v, q_begin, q_len, kv_begin, kv_len, max_q, max_kv, scale, causal, prefix, cap, slopes, out_dtype, out
PyObject* py_attention_ragged(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    want(nargs == 16);
    const Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]);
    const ScalarType in = q.scalar_type();
    want(in == ScalarType::BFloat16 || in == ScalarType::Half);
    const int dev = current_device_of(q);
    want(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes());
    const int64_t Tq = q.size(0), heads = q.size(1), d = q.size(2), Tkv = k.size(0), kv_heads = k.size(1);
    want(k.size(2) == d);
    on(k, dev, in);
    on(v, dev, in);
    const int64_t n = tensor(a[3]).numel();
    const int32_t *qb = index(a[3], dev, n), *ql = index(a[4], dev, n), *kb = index(a[5], dev, n), *kl = index(a[6], dev, n);
    const int64_t max_q = std::min(integer(a[7]), Tq), max_kv = std::min(integer(a[8]), Tkv);
    const float scale = a[9] == Py_None ? (float)(1.0 / std::sqrt((double)d)) : (float)number(a[9]);
    const bool causal = flag(a[10]);
    const int32_t* prefix = vec<int32_t>(a[11], dev, ScalarType::Int, n);
    const float cap = (float)number(a[12]);
    const float* slopes = vec<float>(a[13], dev, ScalarType::Float, heads);
    const int64_t ldq = head_pitch(q), ldk = head_pitch(k), ldv = head_pitch(v);
    int64_t ldo = heads * d;
    Tensor o;
    if (a[15] != Py_None) {
      o = tensor(a[15]);
      on(o, dev, o.scalar_type());
      want(o.sizes() == q.sizes());
      ldo = head_pitch(o);
    }
    const ScalarType out = o.defined() ? o.scalar_type() : a[14] != Py_None ? dtype_of(a[14]) : in;
    want(out == ScalarType::BFloat16 || out == ScalarType::Half);
    const int64_t need = attention_workspace((int)std::min<int64_t>(n, 1 << 30), max_q, max_kv, (int)heads, (int)kv_heads, d);
    if (!o.defined()) o = at::zeros({Tq, heads, d}, q.options().dtype(out));
    Tensor ws;
    if (need > 0) ws = empty({need}, q, ScalarType::Byte);
    const void *qp = q.data_ptr(), *kp = k.data_ptr(), *vp = v.data_ptr();
    void *op = o.data_ptr(), *wsp = need > 0 ? ws.data_ptr() : nullptr;
    const int in_code = code(in), out_code = code(out);
    const int rc = run(dev, [&]() {
      return attention_ragged(qp, ldq, kp, ldk, vp, ldv, in_code, op, ldo, out_code, Tq, Tkv,
                              (int)std::min<int64_t>(n, 1 << 30), qb, ql, kb, kl, max_q, max_kv, (int)heads, (int)kv_heads, d,
                              scale, cap, slopes, causal ? 1 : 0, prefix, wsp, need);
    });
    if (rc) return PyLong_FromLong(rc);
    return a[15] != Py_None ? Py_NewRef(a[15]) : THPVariable_Wrap(std::move(o));
  });
}

// The addresses of the library's functions, in the order above.
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 6) {
    PyErr_SetString(PyExc_TypeError, "bind: six addresses");
    return nullptr;
  }
  void* p[6];
  for (int i = 0; i < 6; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: null address");
      return nullptr;
    }
  }
  set_stream = reinterpret_cast<decltype(set_stream)>(p[0]);
  qk_norm_rope = reinterpret_cast<decltype(qk_norm_rope)>(p[1]);
  lora_workspace = reinterpret_cast<decltype(lora_workspace)>(p[2]);
  linear_lora = reinterpret_cast<decltype(linear_lora)>(p[3]);
  attention_workspace = reinterpret_cast<decltype(attention_workspace)>(p[4]);
  attention_ragged = reinterpret_cast<decltype(attention_ragged)>(p[5]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_bind)), METH_FASTCALL, nullptr},
    {"qk_norm_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_qk_norm_rope)), METH_FASTCALL, nullptr},
    {"linear_lora", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_linear_lora)), METH_FASTCALL, nullptr},
    {"attention_ragged", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_attention_ragged)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving() { return PyModule_Create(&module); }
