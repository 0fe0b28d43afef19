// CPython binding of the entry points that launch work: torch tensors in, tri_* call, status out.
//
// What it replaces and why: filling the tri_tensor structs from Python through ctypes took 0.7 us per tensor and 8 to
// 25 us per call, more than most kernels of a decode step run (RMSNorm of 16 rows: 10.2 us a call of which the GPU
// worked 3.0).  Reading sizes and strides from the tensor object takes some 20 ns.
//
// Every function takes the tensors (or descriptors of them) in the order of the C entry point (None where it allows
// NULL), then its scalars, then the stream as an integer, and returns the status; trinity_amd/ext.py turns a status into
// an exception.
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "../../include/trinity_amd.h"

namespace {

constexpr int kMaxTensors = 12;

struct Tensors {
  tri_tensor v[kMaxTensors];
  tri_tensor* p[kMaxTensors];
};

// o = tensor, None, or a tensor's descriptor as ext.as_tri makes it; int32 tensors are lengths and nothing else
bool to_tri(PyObject* o, tri_tensor& v, tri_tensor*& p, bool lengths) {
  if (o == Py_None) {
    p = nullptr;
    return true;
  }
  if (!THPVariable_Check(o)) {
    Py_buffer b;
    if (strcmp(Py_TYPE(o)->tp_name, "TriTensor") != 0 || PyObject_GetBuffer(o, &b, PyBUF_SIMPLE) != 0) {
      PyErr_Format(PyExc_TypeError, "expected a tensor or None, got %.100s", Py_TYPE(o)->tp_name);
      return false;
    }
    const bool whole = b.len == (Py_ssize_t)sizeof v;
    if (whole) memcpy(&v, b.buf, sizeof v);
    else PyErr_SetString(PyExc_TypeError, "not the TriTensor of this library");
    PyBuffer_Release(&b);
    p = &v;
    return whole;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  switch (t.scalar_type()) {
    case at::kHalf: v.dtype = TRI_F16; break;
    case at::kBFloat16: v.dtype = TRI_BF16; break;
    case at::kFloat: v.dtype = TRI_F32; break;
    case at::kByte: v.dtype = TRI_U8; break;
    case at::kFloat8_e4m3fn: v.dtype = TRI_FP8_E4M3; break;
    default:
      if (lengths && t.scalar_type() == at::kInt) {
        v.dtype = TRI_I32;
        break;
      }
      PyErr_Format(PyExc_TypeError, "unsupported dtype %s", at::toString(t.scalar_type()));
      return false;
  }
  const int64_t nd = t.dim();
  if (nd > 4) {
    PyErr_SetString(PyExc_ValueError, "at most 4 dimensions");
    return false;
  }
  v.ptr = t.data_ptr();
  v.ndim = (int32_t)nd;
  for (int i = 0; i < 4; ++i) {
    v.shape[i] = i < nd ? t.size(i) : 0;
    v.stride[i] = i < nd ? t.stride(i) : 0;
  }
  p = &v;
  return true;
}

// lens_at: which of the tensors holds lengths of sequences
bool marshal(PyObject* const* args, Py_ssize_t nargs, int ntensors, int nscalars, Tensors& t, int lens_at = -1) {
  if (nargs != ntensors + nscalars + 1) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", ntensors + nscalars + 1, nargs);
    return false;
  }
  for (int i = 0; i < ntensors; ++i) {
    if (!to_tri(args[i], t.v[i], t.p[i], i == lens_at)) return false;
  }
  return true;
}

// The tensors of a call are on one GPU (a length or a scale read from host memory would fault it), which is the current one
// while the call launches.
struct OneDevice {
  c10::OptionalDeviceGuard guard;
  bool ok = true;
  OneDevice(PyObject* const* args, int ntensors) {
    const at::Tensor* first = nullptr;
    for (int i = 0; i < ntensors && ok; ++i) {
      if (!THPVariable_Check(args[i])) continue;
      const at::Tensor& t = THPVariable_Unpack(args[i]);
      if (first == nullptr) first = &t;
      ok = t.is_cuda() && t.device() == first->device();
    }
    if (!ok) PyErr_SetString(PyExc_ValueError, "the tensors of a call have to be on one GPU");
    else if (first != nullptr) guard.reset_device(first->device());
  }
};

// the bytes of a ctypes structure (tri_attn_params, tri_cache_params)
template <class T>
struct ParamsOf {
  static_assert(sizeof(tri_attn_params) != sizeof(tri_cache_params), "told apart by their sizes");
  Py_buffer buf{};
  const T* p = nullptr;
  explicit ParamsOf(PyObject* o) {
    if (PyObject_GetBuffer(o, &buf, PyBUF_SIMPLE) != 0) return;
    if (buf.len == (Py_ssize_t)sizeof(T)) p = static_cast<const T*>(buf.buf);
    else PyErr_SetString(PyExc_TypeError, sizeof(T) == sizeof(tri_attn_params) ? "expected TriAttnParams" : "expected TriCacheParams");
  }
  ~ParamsOf() { if (buf.obj != nullptr) PyBuffer_Release(&buf); }
};
using Params = ParamsOf<tri_attn_params>;
using CacheParams = ParamsOf<tri_cache_params>;

void* stream_of(PyObject* o) { return PyLong_AsVoidPtr(o); }

// Other Python threads run while the library works (a launch may wait for room in a stream's queue, and what that queue
// waits for may need the interpreter: a host callback in Python, a thread that feeds another stream).
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};
template <class F>
int call(F f) {
  if (PyErr_Occurred() != nullptr) return 0;
  const NoGil nogil;
  return f();
}

template <class F>
PyObject* run(F f) {
  try {
    const int st = f();
    return PyErr_Occurred() != nullptr ? nullptr : PyLong_FromLong(st);
  } catch (const std::exception& e) {  // (a tensor without storage, for instance)
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

#define TRI_BIND(name) PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n)

TRI_BIND(rmsnorm) {
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 3, 1, t)) return 0;
    const double eps = PyFloat_AsDouble(a[3]);
    void* s = stream_of(a[4]);
    return call([&] { return tri_rmsnorm(t.p[0], t.p[1], t.p[2], (float)eps, s); });
  });
}
TRI_BIND(ffn_swiglu) {
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 7, 0, t)) return 0;
    void* s = stream_of(a[7]);
    return call([&] { return tri_ffn_swiglu(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], t.p[6], s); });
  });
}
TRI_BIND(gateup_swiglu) {
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 6, 0, t)) return 0;
    void* s = stream_of(a[6]);
    return call([&] { return tri_gateup_swiglu(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], s); });
  });
}
TRI_BIND(matmul) {
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 5, 0, t)) return 0;
    void* s = stream_of(a[5]);
    return call([&] { return tri_matmul(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], s); });
  });
}
TRI_BIND(ffn_gelu) {
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 6, 0, t)) return 0;
    void* s = stream_of(a[6]);
    return call([&] { return tri_ffn_gelu(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], s); });
  });
}
TRI_BIND(ffn_block) {
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 12, 0, t)) return 0;
    void* s = stream_of(a[12]);
    return call([&] {
      return tri_ffn_block(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], t.p[6], t.p[7], t.p[8], t.p[9], t.p[10], t.p[11], s);
    });
  });
}
TRI_BIND(qkv_attention) {
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 10, 1, t)) return 0;
    const Params p(a[10]);
    void* s = stream_of(a[11]);
    return call([&] {
      return tri_qkv_attention(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], t.p[6], t.p[7], t.p[8], t.p[9], p.p, s);
    });
  });
}
TRI_BIND(qkv_attention_static) {
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 9, 1, t)) return 0;
    const Params p(a[9]);
    void* s = stream_of(a[10]);
    return call([&] {
      return tri_qkv_attention_static(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], t.p[6], t.p[7], t.p[8], p.p, s);
    });
  });
}
TRI_BIND(keyformer) {
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 11, 1, t)) return 0;
    const Params p(a[11]);
    void* s = stream_of(a[12]);
    return call([&] {
      return tri_keyformer(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], t.p[6], t.p[7], t.p[8], t.p[9], t.p[10], p.p, s);
    });
  });
}
TRI_BIND(roco) {  // (as_mean_var comes before the parameters, as in the C entry point)
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 11, 2, t)) return 0;
    const long mean_var = PyLong_AsLong(a[11]);
    const Params p(a[12]);
    void* s = stream_of(a[13]);
    return call([&] {
      return tri_roco(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], t.p[6], t.p[7], t.p[8], t.p[9], t.p[10],
                      (int32_t)mean_var, p.p, s);
    });
  });
}
TRI_BIND(cache_append) {
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 7, 1, t, 6)) return 0;
    const OneDevice device(a, 7);
    if (!device.ok) return 0;
    const CacheParams p(a[7]);
    void* s = stream_of(a[8]);
    return call([&] { return tri_cache_append(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], t.p[6], p.p, s); });
  });
}
TRI_BIND(cache_read) {
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 7, 1, t, 4)) return 0;
    const OneDevice device(a, 7);
    if (!device.ok) return 0;
    const CacheParams p(a[7]);
    void* s = stream_of(a[8]);
    return call([&] { return tri_cache_read(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], t.p[6], p.p, s); });
  });
}
TRI_BIND(cache_attention) {
  return run([&] {
    Tensors t;
    if (!marshal(a, n, 9, 1, t, 5)) return 0;
    const OneDevice device(a, 9);
    if (!device.ok) return 0;
    const CacheParams p(a[9]);
    void* s = stream_of(a[10]);
    return call([&] {
      return tri_cache_attention(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], t.p[6], t.p[7], t.p[8], p.p, s);
    });
  });
}
#undef TRI_BIND

// ---- blocks.CachedAttention: the sizes of a call are read off its tensors here, and what it returns is made here - from
// Python that takes as long as the rest of a call without its launch.  Each takes the heads and the mask as TriCacheParams,
// its tensors, kv_len (None: all rows of the cache) and the stream; a status other than 0 is returned as an integer.
struct CacheCall {
  tri_cache_params p{};
  bool ok = false;
  // rows: of all sequences together, or (each) of every one
  CacheCall(PyObject* params, PyObject* cache, int64_t rows, bool each, PyObject* kv_len) {
    const CacheParams given(params);
    if (PyErr_Occurred() != nullptr) return;
    if (!THPVariable_Check(cache)) {
      PyErr_Format(PyExc_TypeError, "the cache has to be a tensor, not %.100s", Py_TYPE(cache)->tp_name);
      return;
    }
    const at::Tensor& c = THPVariable_Unpack(cache);
    const int64_t batch = c.dim() == 4 ? c.size(0) : 1;
    const int64_t len = kv_len != Py_None ? PyLong_AsLongLong(kv_len) : (c.dim() >= 2 ? c.size(-2) : 0);
    if (PyErr_Occurred() != nullptr) return;
    if (!each && batch > 0 && rows % batch != 0) {
      PyErr_Format(PyExc_ValueError, "%lld rows are not as many for each of %lld sequences", (long long)rows, (long long)batch);
      return;
    }
    const int64_t seq = each ? rows : (batch > 0 ? rows / batch : 0);
    if (batch > INT32_MAX || seq > INT32_MAX || len > INT32_MAX || seq < INT32_MIN || len < INT32_MIN) {
      PyErr_SetString(PyExc_ValueError, "sizes beyond 32 bits");
      return;
    }
    p = *given.p;
    p.batch = (int32_t)batch;
    p.seq = (int32_t)seq;
    p.kv_len = (int32_t)len;
    ok = true;
  }
};

at::Tensor new_tensor(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
  return at::empty(sizes, like.options().dtype(type));
}
tri_tensor describe(const at::Tensor& t, int32_t dtype) {
  tri_tensor d{};
  d.ptr = t.data_ptr();
  d.ndim = (int32_t)t.dim();
  d.dtype = dtype;
  for (int i = 0; i < d.ndim; ++i) {
    d.shape[i] = t.size(i);
    d.stride[i] = t.stride(i);
  }
  return d;
}
const at::Tensor* tensor_of(PyObject* o, const char* what) {
  if (THPVariable_Check(o)) return &THPVariable_Unpack(o);
  PyErr_Format(PyExc_TypeError, "%s has to be a tensor, not %.100s", what, Py_TYPE(o)->tp_name);
  return nullptr;
}
template <class F>
PyObject* run_new(F f) {
  try {
    return f();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// (k, v, k_cache, k_scales, v_cache, v_scales, lens, kv_len, parameters, stream) -> 0
PyObject* cache_append_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return run_new([&]() -> PyObject* {
    Tensors t;
    if (!marshal(a, n, 7, 2, t, 6)) return nullptr;
    const at::Tensor* const k = tensor_of(a[0], "k");
    if (k == nullptr) return nullptr;
    const CacheCall c(a[8], a[2], k->dim() > 0 ? k->size(0) : 0, false, a[7]);
    if (!c.ok) return nullptr;
    const OneDevice device(a, 7);
    void* s = stream_of(a[9]);
    if (!device.ok || PyErr_Occurred() != nullptr) return nullptr;
    return PyLong_FromLong(call([&] { return tri_cache_append(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], t.p[6], &c.p, s); }));
  });
}

// (k_cache, k_scales, v_cache, v_scales, lens, rows (None: kv_len), whether in bfloat16, kv_len, parameters, stream) -> (k, v)
PyObject* cache_read_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return run_new([&]() -> PyObject* {
    Tensors t;
    if (!marshal(a, n, 5, 4, t, 4)) return nullptr;
    const at::Tensor* const cache = tensor_of(a[0], "the cache");
    if (cache == nullptr) return nullptr;
    CacheCall c(a[8], a[0], a[5] != Py_None ? PyLong_AsLongLong(a[5]) : 0, true, a[7]);
    if (!c.ok) return nullptr;
    if (a[5] == Py_None) c.p.seq = c.p.kv_len;
    const bool bf16 = PyObject_IsTrue(a[6]) == 1;
    const OneDevice device(a, 5);
    void* s = stream_of(a[9]);
    if (!device.ok || PyErr_Occurred() != nullptr) return nullptr;
    // one allocation, the two halves of it as tensors (taking and returning memory costs a microsecond and a half a tensor)
    const int64_t sizes[5] = {2, c.p.batch, c.p.n_kv_heads, c.p.seq < 0 ? 0 : c.p.seq, c.p.head_dim};
    const at::Tensor both = new_tensor(*cache, sizes, bf16 ? at::kBFloat16 : at::kHalf);
    at::Tensor out[2];
    tri_tensor d[2];
    for (int i = 0; i < 2; ++i) {
      out[i] = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(both.storage()), both.key_set(), both.dtype());
      out[i].unsafeGetTensorImpl()->set_sizes_contiguous(at::IntArrayRef(sizes + 1, 4));
      out[i].unsafeGetTensorImpl()->set_storage_offset(i * (both.numel() / 2));
      d[i] = describe(out[i], bf16 ? TRI_BF16 : TRI_F16);
    }
    const int st = call([&] { return tri_cache_read(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], &d[0], &d[1], &c.p, s); });
    if (st != 0) return PyLong_FromLong(st);
    PyObject *const k = THPVariable_Wrap(out[0]), *const v = THPVariable_Wrap(out[1]);
    PyObject* const r = k != nullptr && v != nullptr ? PyTuple_Pack(2, k, v) : nullptr;
    Py_XDECREF(k);
    Py_XDECREF(v);
    return r;
  });
}

// (q, k_cache, k_scales, v_cache, v_scales, lens, scratch, out or None, want_lse, kv_len, parameters, stream) -> out, or (out, lse);
// or, where the scratch is smaller than the call's best plan wants or on another device, the bytes that it wants (nothing is
// launched then)
PyObject* cache_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return run_new([&]() -> PyObject* {
    Tensors t;
    if (!marshal(a, n, 8, 3, t, 5)) return nullptr;
    const at::Tensor* const q = tensor_of(a[0], "q");
    if (q == nullptr) return nullptr;
    const CacheCall c(a[10], a[1], q->dim() > 0 ? q->size(0) : 0, false, a[9]);
    const bool want_lse = PyObject_IsTrue(a[8]) == 1;
    void* s = stream_of(a[11]);
    if (!c.ok || PyErr_Occurred() != nullptr) return nullptr;
    const int64_t need = tri_cache_scratch_bytes(&c.p, t.p[2] != nullptr);
    if (need < 0) return PyLong_FromLongLong(need);
    PyObject* with[8];
    for (int i = 0; i < 8; ++i) with[i] = i == 6 ? Py_None : a[i];  // (the scratch may be anywhere: another is asked for then)
    const OneDevice device(with, 8);
    if (!device.ok) return nullptr;
    if (need > 0 && (t.p[6] == nullptr || t.p[6]->shape[0] < need || THPVariable_Unpack(a[6]).device() != q->device()))
      return PyLong_FromLongLong(need);
    at::Tensor made, lse;
    tri_tensor o, l;
    tri_tensor *out = t.p[7], *lp = nullptr;
    if (out == nullptr) {
      made = new_tensor(*q, {q->dim() > 0 ? q->size(0) : 0, (int64_t)c.p.n_q_heads * c.p.head_dim}, q->scalar_type());
      o = describe(made, t.p[0]->dtype);
      out = &o;
    }
    if (want_lse) {
      lse = new_tensor(*q, {c.p.batch, c.p.n_q_heads, c.p.seq}, at::kFloat);
      l = describe(lse, TRI_F32);
      lp = &l;
    }
    const int st = call([&] {
      return tri_cache_attention(t.p[0], t.p[1], t.p[2], t.p[3], t.p[4], t.p[5], need > 0 ? t.p[6] : nullptr, lp, out, &c.p, s);
    });
    if (st != 0) return PyLong_FromLong(st);
    PyObject* r = made.defined() ? THPVariable_Wrap(made) : a[7];
    if (!made.defined()) Py_INCREF(r);
    if (r == nullptr || !want_lse) return r;
    PyObject* const x = THPVariable_Wrap(lse);
    PyObject* const both = x != nullptr ? PyTuple_Pack(2, r, x) : nullptr;
    Py_DECREF(r);
    Py_XDECREF(x);
    return both;
  });
}

PyObject* cache_scratch_bytes(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) return PyErr_Format(PyExc_TypeError, "expected 2 arguments, got %zd", n);
  const CacheParams p(a[0]);
  const long four_bit = PyLong_AsLong(a[1]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  return PyLong_FromLongLong(tri_cache_scratch_bytes(p.p, four_bit != 0));
}
PyObject* qkv_scratch_bytes(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) return PyErr_Format(PyExc_TypeError, "expected 2 arguments, got %zd", n);
  const Params p(a[0]);
  const long long n_model = PyLong_AsLongLong(a[1]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  return PyLong_FromLongLong(tri_qkv_scratch_bytes(p.p, n_model));
}
template <int64_t (*F)(int64_t, int64_t, int64_t)>
PyObject* workspace_bytes(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) return PyErr_Format(PyExc_TypeError, "expected 3 arguments, got %zd", n);
  const long long x = PyLong_AsLongLong(a[0]), y = PyLong_AsLongLong(a[1]), z = PyLong_AsLongLong(a[2]);
  if (PyErr_Occurred() != nullptr) return nullptr;
  return PyLong_FromLongLong(F(x, y, z));
}

#define TRI_METHOD(name, fn) {name, (PyCFunction)(void (*)(void))(PyObject* (*)(PyObject*, PyObject* const*, Py_ssize_t))(fn), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    TRI_METHOD("rmsnorm", rmsnorm), TRI_METHOD("ffn_swiglu", ffn_swiglu), TRI_METHOD("gateup_swiglu", gateup_swiglu),
    TRI_METHOD("matmul", matmul), TRI_METHOD("ffn_gelu", ffn_gelu), TRI_METHOD("ffn_block", ffn_block),
    TRI_METHOD("qkv_attention", qkv_attention), TRI_METHOD("qkv_attention_static", qkv_attention_static),
    TRI_METHOD("keyformer", keyformer), TRI_METHOD("roco", roco), TRI_METHOD("qkv_scratch_bytes", qkv_scratch_bytes),
    TRI_METHOD("gemm_workspace_bytes", workspace_bytes<tri_gemm_workspace_bytes>),
    TRI_METHOD("ffn_workspace_bytes", workspace_bytes<tri_ffn_workspace_bytes>),
    TRI_METHOD("cache_append", cache_append), TRI_METHOD("cache_read", cache_read),
    TRI_METHOD("cache_attention", cache_attention), TRI_METHOD("cache_append_rows", cache_append_rows),
    TRI_METHOD("cache_read_rows", cache_read_rows), TRI_METHOD("cache_attend", cache_attend), TRI_METHOD("cache_scratch_bytes", cache_scratch_bytes),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
