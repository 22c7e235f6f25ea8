// torch_calls.cpp -- a short way from torch tensors to the entry points of paged and packed
// attention, for calls that take less time on the GPU than their checks in Python (single tokens).
//
// Every function makes the checks of the wrapper of its name in ops.py on the tensors themselves and
// calls the C entry on the current stream. It returns the entry's code, or None where anything is
// not as the wrapper wants it (or the call has a workspace): the wrapper then goes its own way, which
// says what is wrong. The entry points come as addresses (init), so this links with no CUDA code.
#include <Python.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/srdit_b200.h"

namespace {

decltype(&srdit_kv_write) g_write = nullptr;
decltype(&srdit_kv_read) g_read = nullptr;
decltype(&srdit_seq_attn) g_attn = nullptr;
decltype(&srdit_seq_attn_workspace) g_workspace = nullptr;

// thrown where the wrapper has to go its own way
struct Otherwise {};
void want(bool ok) {
  if (!ok) throw Otherwise{};
}

// The tensors of a call: all on one device, which is the current one.
struct Call {
  int device = -1;
  const at::Tensor& tensor(PyObject* o) {
    want(THPVariable_Check(o));
    const at::Tensor& t = THPVariable_Unpack(o);
    want(t.is_cuda() && t.layout() == at::kStrided);
    if (device < 0) {
      device = t.get_device();
      want(device == c10::cuda::current_device());
    }
    want(t.get_device() == device);
    return t;
  }
  cudaStream_t stream() const {
    return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
  }
  // contiguous int32 [n], or null for None
  const int32_t* ints(PyObject* o, int64_t n, bool may_lack) {
    if (o == Py_None && may_lack) return nullptr;
    const at::Tensor& t = tensor(o);
    want(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous());
    return static_cast<const int32_t*>(t.data_ptr());
  }
};

int as_int(int64_t n) {
  want(n >= 0 && n <= INT32_MAX);
  return static_cast<int>(n);
}
int half_type(at::ScalarType t) {
  want(t == at::kBFloat16 || t == at::kHalf);
  return t == at::kBFloat16 ? SRDIT_BF16 : SRDIT_FP16;
}

// _pages of ops.py; rows of the cache go to or from `rows`
srdit_kv_pages pages(Call& c, PyObject* const* o, PyObject* ks, PyObject* vs,
                     at::ScalarType rows) {
  const at::Tensor &k = c.tensor(o[0]), &v = c.tensor(o[1]), &table = c.tensor(o[2]);
  want(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type());
  want(k.stride(3) == 1 && v.stride(3) == 1);
  want(table.dim() == 2 && table.scalar_type() == at::kInt &&
       (table.stride(1) == 1 || table.size(1) <= 1));
  srdit_kv_pages p = {};
  p.dtype = half_type(rows);
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  if (k.scalar_type() == rows) {
    want(ks == Py_None && vs == Py_None);
    p.code = SRDIT_KV_PLAIN;
  } else {
    want(k.scalar_type() == at::kChar || k.scalar_type() == at::kFloat8_e4m3fn);
    p.code = k.scalar_type() == at::kChar ? SRDIT_Q_INT8 : SRDIT_Q_E4M3;
    const at::Tensor &a = c.tensor(ks), &b = c.tensor(vs);
    want(a.scalar_type() == at::kFloat && b.scalar_type() == at::kFloat && a.dim() == 3 &&
         a.sizes() == b.sizes() && a.sizes() == k.sizes().slice(0, 3));
    p.k_scale = static_cast<float*>(a.data_ptr());
    p.v_scale = static_cast<float*>(b.data_ptr());
    for (int i = 0; i < 3; ++i) {
      p.ks_stride[i] = a.stride(i);
      p.vs_stride[i] = b.stride(i);
    }
  }
  p.pages = as_int(k.size(0));
  p.page_size = as_int(k.size(1));
  p.Hkv = as_int(k.size(2));
  p.D = as_int(k.size(3));
  for (int i = 0; i < 3; ++i) {
    p.k_stride[i] = k.stride(i);
    p.v_stride[i] = v.stride(i);
  }
  p.table = static_cast<const int32_t*>(table.data_ptr());
  p.table_stride = table.stride(0);
  p.table_width = as_int(table.size(1));
  p.B = as_int(table.size(0));
  return p;
}

// packed rows [T, Hkv, D] with unit stride: {token, head}
void row_strides(const at::Tensor& t, long long st[2]) {
  want(t.stride(2) == 1);
  st[0] = t.stride(0);
  st[1] = t.stride(1);
}

template <typename F>
PyObject* guarded(F f) {
  try {
    return PyLong_FromLong(f());
  } catch (...) {
    PyErr_Clear();  // (of an argument's __bool__; the wrapper meets it again)
    Py_RETURN_NONE;
  }
}

// kv_write(k, v, k_pages, v_pages, table, kv_lens, cu_q, k_scale, v_scale)
PyObject* kv_write(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&] {
    want(n == 9 && g_write);
    Call c;
    const at::Tensor &k = c.tensor(o[0]), &v = c.tensor(o[1]);
    const srdit_kv_pages p = pages(c, o + 2, o[7], o[8], k.scalar_type());
    want(k.dim() == 3 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() &&
         k.size(1) == p.Hkv && k.size(2) == p.D);
    long long ks[2], vs[2];
    row_strides(k, ks);
    row_strides(v, vs);
    const int32_t* lens = c.ints(o[5], p.B, false);
    const int32_t* cu = c.ints(o[6], p.B + 1ll, true);
    return g_write(&p, k.data_ptr(), ks, v.data_ptr(), vs, as_int(k.size(0)), cu, lens, c.stream());
  });
}

// kv_read(k_pages, v_pages, table, cu_k, k, v, k_scale, v_scale)
PyObject* kv_read(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&] {
    want(n == 8 && g_read);
    Call c;
    const at::Tensor &k = c.tensor(o[4]), &v = c.tensor(o[5]);
    const srdit_kv_pages p = pages(c, o, o[6], o[7], k.scalar_type());
    want(k.dim() == 3 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() &&
         k.size(1) == p.Hkv && k.size(2) == p.D);
    long long ks[2], vs[2];
    row_strides(k, ks);
    row_strides(v, vs);
    return g_read(&p, k.data_ptr(), ks, v.data_ptr(), vs, as_int(k.size(0)),
                  c.ints(o[3], p.B + 1ll, false), c.stream());
  });
}

// what both attentions have: q, out, causal, scale, status
void attention(Call& c, srdit_seq_attn_args& a, PyObject* q_, PyObject* out_, PyObject* causal,
               PyObject* scale, PyObject* status) {
  const at::Tensor &q = c.tensor(q_), &out = c.tensor(out_);
  want(q.dim() == 3 && q.size(2) == a.D && a.Hkv > 0 && q.size(1) % a.Hkv == 0);
  want(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type());
  row_strides(q, a.q_stride);
  row_strides(out, a.o_stride);
  a.dtype = half_type(q.scalar_type());
  a.q = q.data_ptr();
  a.out = out.data_ptr();
  a.T = as_int(q.size(0));
  a.H = as_int(q.size(1));
  const int yes = PyObject_IsTrue(causal);
  want(yes >= 0);
  a.causal = yes;
  if (scale == Py_None) {
    a.scale = static_cast<float>(std::pow(static_cast<double>(a.D), -0.5));
  } else {
    want(PyFloat_CheckExact(scale));
    a.scale = static_cast<float>(PyFloat_AS_DOUBLE(scale));
  }
  if (status != Py_None) a.status = static_cast<uint32_t*>(c.tensor(status).data_ptr());
}
int whole(PyObject* o) {
  want(PyLong_CheckExact(o));
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Otherwise{};
  }
  want(v >= INT32_MIN && v <= INT32_MAX);
  return static_cast<int>(v);
}
int run(const srdit_seq_attn_args& a, const Call& c) {
  want(g_workspace(&a) == 0);
  return g_attn(&a, c.stream());
}

// paged_attn(q, k_pages, v_pages, table, kv_lens, out, cu_q, max_q, max_kv, causal, k_scale, v_scale,
//            scale, status)
PyObject* paged_attn(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&] {
    want(n == 14 && g_attn && g_workspace);
    Call c;
    const srdit_kv_pages p = pages(c, o + 1, o[10], o[11], c.tensor(o[0]).scalar_type());
    srdit_seq_attn_args a = {};
    a.pages = &p;
    a.B = p.B;
    a.Hkv = p.Hkv;
    a.D = p.D;
    attention(c, a, o[0], o[5], o[9], o[12], o[13]);
    a.kv_lens = c.ints(o[4], p.B, false);
    a.cu_q = c.ints(o[6], p.B + 1ll, true);
    a.max_q = o[7] != Py_None ? whole(o[7]) : a.cu_q || p.B == 0 ? a.T : a.T / p.B;
    a.max_kv = o[8] != Py_None
                   ? whole(o[8])
                   : as_int(static_cast<int64_t>(p.table_width) * p.page_size);
    return run(a, c);
  });
}

// packed_attn(q, k, v, cu_q, out, cu_k, causal, scale, status)
PyObject* packed_attn(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&] {
    want(n == 9 && g_attn && g_workspace);
    Call c;
    const at::Tensor &q = c.tensor(o[0]), &k = c.tensor(o[1]), &v = c.tensor(o[2]);
    want(k.dim() == 3 && v.sizes() == k.sizes() && k.scalar_type() == q.scalar_type() &&
         v.scalar_type() == q.scalar_type());
    const at::Tensor& cu = c.tensor(o[3]);
    srdit_seq_attn_args a = {};
    a.B = as_int(cu.numel() - 1);
    a.Hkv = as_int(k.size(1));
    a.D = as_int(k.size(2));
    attention(c, a, o[0], o[4], o[6], o[7], o[8]);
    row_strides(k, a.k_stride);
    row_strides(v, a.v_stride);
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.Tk = as_int(k.size(0));
    a.cu_q = c.ints(o[3], a.B + 1ll, false);
    a.cu_k = c.ints(o[5], a.B + 1ll, true);
    want(a.cu_k || a.Tk == a.T);
    return run(a, c);
  });
}

// init(addresses of srdit_kv_write, srdit_kv_read, srdit_seq_attn, srdit_seq_attn_workspace)
PyObject* init(PyObject*, PyObject* const* o, Py_ssize_t n) {
  void* p[4];
  if (n != 4) return PyErr_Format(PyExc_TypeError, "four addresses");
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(o[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g_write = reinterpret_cast<decltype(g_write)>(p[0]);
  g_read = reinterpret_cast<decltype(g_read)>(p[1]);
  g_attn = reinterpret_cast<decltype(g_attn)>(p[2]);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(p[3]);
  Py_RETURN_NONE;
}

#define SRDIT_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {SRDIT_METHOD(init),       SRDIT_METHOD(kv_write),
                           SRDIT_METHOD(kv_read),    SRDIT_METHOD(paged_attn),
                           SRDIT_METHOD(packed_attn), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_srdit_calls", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__srdit_calls(void) { return PyModule_Create(&g_module); }
