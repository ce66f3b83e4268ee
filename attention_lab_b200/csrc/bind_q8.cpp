// Python binding of the 8-bit cache's operators (the module attention_lab_b200._q8_bind): argument checks, outputs and
// the call of the C ABI, in one step from Python. The same through ctypes took 12 to 17 us of host time a call, more
// than a decode step's kernels take on the device; this takes 4 to 6. The operators' contracts are documented in
// attention_lab_b200/q8.py, which passes every argument by position.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/attention_lab_b200.h"

namespace {

constexpr int64_t kBlock = 64;

[[noreturn]] void raise_status(int rc) {
  const char* msg = al_last_error();
  if (rc == AL_EINVAL || rc == AL_EUNSUPPORTED) TORCH_CHECK_VALUE(false, msg);
  TORCH_CHECK(false, msg);
}
void check(int rc) {
  if (rc != AL_OK) raise_status(rc);
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o, const char* what) {
  TORCH_CHECK_TYPE(PyIndex_Check(o), what, " must be an integer, got ", Py_TYPE(o)->tp_name);
  PyObject* i = PyNumber_Index(o);
  if (!i) throw python_error();
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(i, &overflow);
  Py_DECREF(i);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  TORCH_CHECK_VALUE(overflow == 0, what, " is out of range");
  return v;
}
// An integer that the C ABI takes as int: out of its range is out of every range.
int small(PyObject* o, const char* what) {
  const int64_t v = integer(o, what);
  TORCH_CHECK_VALUE(v >= INT32_MIN && v <= INT32_MAX, what, " = ", v, " is out of range");
  return (int)v;
}
int size32(int64_t v, const char* what) {
  TORCH_CHECK_VALUE(v <= INT32_MAX, what, " = ", v, " is too large");
  return (int)v;
}

void on_device(const at::Tensor& t, int dev) {
  TORCH_CHECK_VALUE(t.is_cuda(), "every tensor must live on a CUDA device (the CUDA path has no CPU fallback)");
  TORCH_CHECK_VALUE(t.get_device() == dev, "all inputs must live on the same device");
}
int cuda_ordinal(const at::Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), "every tensor must live on a CUDA device (the CUDA path has no CPU fallback)");
  return t.get_device();
}
int code_of(at::ScalarType t, const char* what) {
  TORCH_CHECK_VALUE(t == at::kFloat || t == at::kBFloat16, what, " must be float32 or bfloat16, got ", t);
  return t == at::kFloat ? AL_F32 : AL_BF16;
}

// t itself when its rows can be read in 16-byte pieces, else a contiguous copy.
at::Tensor rows(const at::Tensor& t) {
  const int64_t unit = 16 / t.element_size(), n = t.dim();
  int64_t bits = 0;
  for (int64_t i = 0; i + 1 < n; ++i) bits |= t.stride(i);
  auto aligned = [](const at::Tensor& x) { return (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0; };
  if (t.stride(n - 1) == 1 && (bits & (unit - 1)) == 0 && aligned(t)) return t;
  at::Tensor c = t.contiguous();
  return aligned(c) ? c : c.clone();
}

struct Cache {
  const at::Tensor *k, *v, *ke, *ve;
  int B, G, C, d, dev;
};
Cache cache_of(PyObject* o) {
  TORCH_CHECK_TYPE(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 4, "the cache must be a Q8Cache (k, v, k_exp, v_exp)");
  Cache c;
  c.k = &tensor(PyTuple_GET_ITEM(o, 0), "k");
  c.v = &tensor(PyTuple_GET_ITEM(o, 1), "v");
  c.ke = &tensor(PyTuple_GET_ITEM(o, 2), "k_exp");
  c.ve = &tensor(PyTuple_GET_ITEM(o, 3), "v_exp");
  TORCH_CHECK_VALUE(c.k->dim() == 4 && c.v->sizes() == c.k->sizes(), "the codes must be [B,G,C,d] of one shape, got ",
                    c.k->sizes(), " and ", c.v->sizes());
  TORCH_CHECK_VALUE(c.k->scalar_type() == at::kFloat8_e4m3fn && c.v->scalar_type() == at::kFloat8_e4m3fn,
                    "the codes must be float8_e4m3fn, got ", c.k->scalar_type(), " and ", c.v->scalar_type());
  const auto s = c.k->sizes();
  c.B = size32(s[0], "B"); c.G = size32(s[1], "G"); c.C = size32(s[2], "C"); c.d = size32(s[3], "d");
  auto exps_ok = [&](const at::Tensor& e) {
    return e.dim() == 3 && e.size(0) == s[0] && e.size(1) == s[1] && e.size(2) == (s[2] + kBlock - 1) / kBlock &&
           e.scalar_type() == at::kChar;
  };
  TORCH_CHECK_VALUE(exps_ok(*c.ke) && exps_ok(*c.ve), "the exponents must be int8 [B,G,ceil(C/64)]");
  TORCH_CHECK_VALUE(c.k->is_contiguous() && c.v->is_contiguous() && c.ke->is_contiguous() && c.ve->is_contiguous(),
                    "codes and exponents must be contiguous");
  c.dev = cuda_ordinal(*c.k);
  on_device(*c.v, c.dev); on_device(*c.ke, c.dev); on_device(*c.ve, c.dev);
  return c;
}

struct Lengths {
  const int* ptr;
  int all;
};
Lengths lengths_of(PyObject* o, const Cache& c, const char* what, int64_t least) {
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == c.B && t.is_contiguous(),
                      "lengths must be an int or a contiguous int32 tensor [B]");
    on_device(t, c.dev);
    return {t.data_ptr<int>(), 0};
  }
  const int64_t n = integer(o, "lengths");
  TORCH_CHECK_VALUE(least <= n && n <= c.C, what, ": length ", n, " outside [", least, ", ", c.C, "]");
  return {nullptr, (int)n};
}

struct Table {
  const float* ptr;
  int rows, rot;
};
Table table_of(const at::Tensor& t, int dev) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.scalar_type() == at::kFloat && t.is_contiguous(),
                    "the rotary table must be a contiguous float32 [length, rotary_dim] tensor");
  on_device(t, dev);
  return {t.data_ptr<float>(), size32(t.size(0), "table length"), size32(t.size(1), "rotary_dim")};
}

void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

// rotary_embed(q, k | None, table, positions, layout, inverse) -> (q', k' | None)
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6, "rotary_embed takes 6 arguments");
  const at::Tensor& q0 = tensor(a[0], "q");
  const at::Tensor& tab = tensor(a[2], "table");
  const int dev = cuda_ordinal(q0);
  const Table t = table_of(tab, dev);
  TORCH_CHECK_VALUE(q0.dim() == 4, "q must be [B,H,T,d], got ", q0.sizes());
  const int B = size32(q0.size(0), "B"), H = size32(q0.size(1), "H"), T = size32(q0.size(2), "T"), d = size32(q0.size(3), "d");
  const int code = code_of(q0.scalar_type(), "q");
  const c10::cuda::OptionalCUDAGuard guard(q0.device());
  const at::Tensor q = rows(q0);
  at::Tensor k, k_out;
  int Hk = 0;
  int64_t ks[3] = {0, 0, 0};
  if (a[1] != Py_None) {
    const at::Tensor& k0 = tensor(a[1], "k");
    on_device(k0, dev);
    TORCH_CHECK_VALUE(k0.dim() == 4 && k0.size(0) == B && k0.size(2) == T && k0.size(3) == d &&
                          k0.scalar_type() == q0.scalar_type(), "k must be [B,G,T,d] of q's dtype");
    k = rows(k0);
    Hk = size32(k.size(1), "G");
    for (int i = 0; i < 3; ++i) ks[i] = k.stride(i);
    k_out = at::empty({B, Hk, T, d}, q.options());
  }
  const int64_t* pos = nullptr;
  int64_t pst[2] = {0, 0}, start = 0;
  at::Tensor p;
  if (THPVariable_Check(a[3])) {
    p = THPVariable_Unpack(a[3]);
    TORCH_CHECK_VALUE(p.scalar_type() == at::kLong, "positions must be int64");
    on_device(p, dev);
    // [B,T], [T] or [1,T], or a single position for every row
    const int64_t pd = p.dim();
    TORCH_CHECK_VALUE(p.numel() == 1 || ((pd == 1 || (pd == 2 && (p.size(0) == B || p.size(0) == 1))) && p.size(pd - 1) == T),
                      "positions must be [B,T] = [", B, ",", T, "], got ", p.sizes());
    if (p.numel() == 1) p = p.reshape({});
    p = p.expand({B, T});
    pos = p.data_ptr<int64_t>();
    pst[0] = p.stride(0); pst[1] = p.stride(1);
  } else {
    start = integer(a[3], "positions");
    TORCH_CHECK_VALUE(start >= 0 && start <= (int64_t)t.rows - T, T, " positions from ", start, " on lie outside the table's ", t.rows, " rows");
  }
  at::Tensor out = at::empty({B, H, T, d}, q.options());
  check(al_rotary(q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), H, Hk ? k.data_ptr() : nullptr, ks[0], ks[1], ks[2],
                  Hk, code, t.ptr, t.rows, t.rot, small(a[4], "layout"), pos, pst[0], pst[1], start, B, T, d,
                  PyObject_IsTrue(a[5]), out.data_ptr(), Hk ? k_out.data_ptr() : nullptr, stream_of(dev)));
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(out)));
  if (a[1] != Py_None) PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(k_out)));
  else PyTuple_SET_ITEM(r, 1, Py_NewRef(Py_None));
  return r;
  END_HANDLE_TH_ERRORS
}

// append_q8(cache, lengths, k_new, v_new, q | None, table | None, layout) -> q' | None
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "append_q8 takes 7 arguments");
  const Cache c = cache_of(a[0]);
  const at::Tensor& k0 = tensor(a[2], "k_new");
  const at::Tensor& v0 = tensor(a[3], "v_new");
  TORCH_CHECK_VALUE(k0.dim() == 4 && k0.size(0) == c.B && k0.size(1) == c.G && k0.size(3) == c.d && v0.sizes() == k0.sizes(),
                    "k_new and v_new must be [B,G,T,d] matching the cache");
  TORCH_CHECK_VALUE(v0.scalar_type() == k0.scalar_type(), "k_new and v_new must share one dtype");
  on_device(k0, c.dev); on_device(v0, c.dev);
  const int T = size32(k0.size(2), "T"), code = code_of(k0.scalar_type(), "k_new");
  const Lengths len = lengths_of(a[1], c, "append", T);
  Table t = {nullptr, 0, 0};
  if (a[5] != Py_None) t = table_of(tensor(a[5], "table"), c.dev);
  const c10::cuda::OptionalCUDAGuard guard(k0.device());
  at::Tensor q, q_out;
  int h = 0;
  int64_t qs[4] = {0, 0, 0, 0};
  if (a[4] != Py_None) {
    const at::Tensor& q0 = tensor(a[4], "q");
    TORCH_CHECK_VALUE(t.ptr != nullptr, "q is rotated: it needs a table");
    on_device(q0, c.dev);
    TORCH_CHECK_VALUE(q0.dim() == 5 && q0.size(0) == c.B && q0.size(1) == c.G && q0.size(3) == T && q0.size(4) == c.d &&
                          q0.scalar_type() == k0.scalar_type(), "q must be [B,G,h,T,d] of k_new's dtype");
    q = rows(q0);
    h = size32(q.size(2), "h");
    for (int i = 0; i < 4; ++i) qs[i] = q.stride(i);
    q_out = at::empty({c.B, c.G, h, T, c.d}, q.options());
  }
  const at::Tensor k = rows(k0), v = rows(v0);
  const bool has_q = h > 0;
  check(al_append_q8(c.k->data_ptr(), c.v->data_ptr(), c.ke->data_ptr(), c.ve->data_ptr(), len.ptr, len.all,
                     k.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.data_ptr(), v.stride(0), v.stride(1), v.stride(2),
                     code, t.ptr, t.rows, t.rot, small(a[6], "layout"), has_q ? q.data_ptr() : nullptr, qs[0], qs[1], qs[2],
                     qs[3], h, has_q ? q_out.data_ptr() : nullptr, c.B, c.G, T, c.C, c.d, stream_of(c.dev)));
  if (a[4] == Py_None) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(q_out));
  END_HANDLE_TH_ERRORS
}

// read_q8(cache, lo, hi, is_f32) -> (k, v)
PyObject* py_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 4, "read_q8 takes 4 arguments");
  const Cache c = cache_of(a[0]);
  const int64_t lo = integer(a[1], "lo"), hi = integer(a[2], "hi");
  TORCH_CHECK_VALUE(0 <= lo && lo <= hi && hi <= c.C, "need 0 <= lo <= hi <= capacity ", c.C, ", got lo=", lo, " hi=", hi);
  const bool f32 = PyObject_IsTrue(a[3]);
  const c10::cuda::OptionalCUDAGuard guard(c.k->device());
  const auto opt = c.k->options().dtype(f32 ? at::kFloat : at::kBFloat16);
  at::Tensor k = at::empty({c.B, c.G, hi - lo, c.d}, opt), v = at::empty({c.B, c.G, hi - lo, c.d}, opt);
  check(al_read_q8(c.k->data_ptr(), c.v->data_ptr(), c.ke->data_ptr(), c.ve->data_ptr(), c.B, c.G, c.C, c.d, (int)lo, (int)hi,
                   f32 ? AL_F32 : AL_BF16, k.data_ptr(), v.data_ptr(), stream_of(c.dev)));
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(k)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(v)));
  return r;
  END_HANDLE_TH_ERRORS
}

// attend_q8(q, cache, lengths, window, sinks, scale | None, max_length | None) -> out
PyObject* py_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "attend_q8 takes 7 arguments");
  const Cache c = cache_of(a[1]);
  const at::Tensor& q0 = tensor(a[0], "q");
  TORCH_CHECK_VALUE(q0.dim() == 5 && q0.size(0) == c.B && q0.size(1) == c.G && q0.size(4) == c.d,
                    "q must be [B,G,h,T,d] matching the cache, got ", q0.sizes());
  on_device(q0, c.dev);
  const int h = size32(q0.size(2), "h"), T = size32(q0.size(3), "T"), code = code_of(q0.scalar_type(), "q");
  const int window = small(a[3], "window"), sinks = small(a[4], "sinks");
  TORCH_CHECK_VALUE(window >= 0 && sinks >= 0, "window and sinks must not be negative, got ", window, " and ", sinks);
  const Lengths len = lengths_of(a[2], c, "attend", 0);
  const int most = !len.ptr ? len.all : a[6] == Py_None ? c.C : small(a[6], "max_length");
  double scale = 1.0 / std::sqrt((double)c.d);
  if (a[5] != Py_None) {
    TORCH_CHECK_TYPE(PyNumber_Check(a[5]), "scale must be a number, got ", Py_TYPE(a[5])->tp_name);
    scale = PyFloat_AsDouble(a[5]);
    if (scale == -1.0 && PyErr_Occurred()) throw python_error();
  }
  const c10::cuda::OptionalCUDAGuard guard(q0.device());
  const at::Tensor q = rows(q0);
  at::Tensor out = at::empty({c.B, c.G, h, T, c.d}, q.options()), work;
  size_t need = 0;
  check(al_attend_q8_workspace(c.B, c.G, h, T, c.C, window, sinks, most, &need));
  if (need) work = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
  check(al_attend_q8(q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), q.stride(3), code, c.k->data_ptr(),
                     c.v->data_ptr(), c.ke->data_ptr(), c.ve->data_ptr(), len.ptr, len.all, c.B, c.G, h, T, c.C, c.d, window,
                     sinks, (float)scale, most, out.data_ptr(), need ? work.data_ptr() : nullptr, need, stream_of(c.dev)));
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"rotary_embed", (PyCFunction)(void (*)(void))py_rotary, METH_FASTCALL, nullptr},
    {"append_q8", (PyCFunction)(void (*)(void))py_append, METH_FASTCALL, nullptr},
    {"read_q8", (PyCFunction)(void (*)(void))py_read, METH_FASTCALL, nullptr},
    {"attend_q8", (PyCFunction)(void (*)(void))py_attend, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_q8_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyMODINIT_FUNC PyInit__q8_bind(void) { return PyModule_Create(&module); }
