// The calls of leapquant_amd/attn.py: checks of the tensors and the launch, without the interpreter's time for each attribute
// of each tensor.  Arguments that the kernels do not take raise; no C++ exception leaves.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>
#include <string>

#include "../../include/lq_attn.h"

namespace {

struct Raised {};                        // a Python exception is set

template <typename... A> [[noreturn]] void raise(PyObject* type, const char* format, A... a) {
  PyErr_Format(type, format, a...);
  throw Raised();
}
std::string shape_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
std::string strides_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.stride(i));
  return s + ")";
}
std::string type_of(const at::Tensor& t) { return c10::toString(t.scalar_type()); }

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s: a tensor expected, got %s", name, Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
long long integer(PyObject* o, const char* name) {
  if (!PyLong_Check(o)) raise(PyExc_TypeError, "%s: an integer expected, got %s", name, Py_TYPE(o)->tp_name);
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}
double number(PyObject* o, const char* name) {
  if (!PyFloat_Check(o) && !PyLong_Check(o)) raise(PyExc_TypeError, "%s: a number expected, got %s", name, Py_TYPE(o)->tp_name);
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised();
  return v;
}
bool aligned(const at::Tensor& t, int bytes) { return (uintptr_t)t.data_ptr() % bytes == 0; }

// every tensor of a call on the GPU `dev`, the first one's
struct Device {
  const int dev;
  explicit Device(const at::Tensor& t) : dev(t.is_cuda() ? (int)t.get_device() : -1) {}
  void on(const at::Tensor& t, const char* name) const {
    const int d = t.is_cuda() ? (int)t.get_device() : -1;
    if (d != dev) raise(PyExc_ValueError, "%s is on %s, expected %s", name, t.device().str().c_str(),
                        dev >= 0 ? ("cuda:" + std::to_string(dev)).c_str() : "cpu");
  }
  void gpu() const { if (dev < 0) raise(PyExc_ValueError, "liblq_attn takes GPU tensors only, got cpu tensors"); }
};

// `dev` current while this lives: a launch on a default stream goes to the current device, whatever its tensors are on
struct Current {
  const c10::DeviceIndex dev, was;
  explicit Current(int d) : dev((c10::DeviceIndex)d), was(c10::hip::ExchangeDevice(dev)) {}
  ~Current() { if (was != dev) (void)c10::hip::SetDevice(was); }
};
void* stream(int dev) { return (void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream(); }

// bf16 [T, H, D] with packed heads whose start and strides are multiples of 16 bytes
lq_rows rows(const at::Tensor& t, const Device& dev, long long T, long long H, long long D, const char* name) {
  dev.on(t, name);
  if (t.scalar_type() != at::kBFloat16) raise(PyExc_TypeError, "%s: dtype %s, expected torch.bfloat16", name, type_of(t).c_str());
  if (t.dim() != 3 || t.size(0) != T || t.size(1) != H || t.size(2) != D)
    raise(PyExc_ValueError, "%s: shape %s, expected (%lld, %lld, %lld)", name, shape_of(t).c_str(), T, H, D);
  const long long ld = T < 2 ? H * D : t.stride(0), hd = H < 2 ? D : t.stride(1);
  if (t.stride(2) != 1 || ld % 8 || hd % 8 || !aligned(t, 16))
    raise(PyExc_ValueError, "%s: packed heads expected, with their start and strides aligned to 16 bytes (strides %s)", name,
          strides_of(t).c_str());
  return {t.data_ptr(), ld, hd};
}
void apart(const lq_rows& r, long long T, long long H, long long D) {
  const bool ok = (T < 2 || r.ld >= D) && (H < 2 || r.hd >= D) &&
                  (T < 2 || H < 2 || (r.ld >= r.hd ? r.ld >= (H - 1) * r.hd + D : r.hd >= (T - 1) * r.ld + D));
  if (!ok) raise(PyExc_ValueError, "out: heads that overlap each other (strides %lld, %lld)", r.ld, r.hd);
}

// Integers of another type as int32.  Wider ones are held to its range, where the kernels take them for what they are: outside the
// cache, or past the last token.  (As they are, 2^32 would become page 0.)
at::Tensor narrowed(const at::Tensor& t) {
  const auto type = t.scalar_type();
  if (type != at::kLong && type != at::ScalarType::UInt32 && type != at::ScalarType::UInt64) return t.to(at::kInt).contiguous();
  at::Tensor wide = t.to(at::kLong);
  if (type == at::ScalarType::UInt64) wide = wide.masked_fill(wide.lt(0), 0x7fffffff);          // 2^63 and more
  return wide.clamp(-0x80000000ll, 0x7fffffffll).to(at::kInt).contiguous();
}
// an int32 index tensor; other integer types are converted
at::Tensor index(const at::Tensor& t, const Device& dev, long long n, const char* name) {
  dev.on(t, name);
  if (t.dim() != 1 || t.size(0) != n) raise(PyExc_ValueError, "%s: 1-D with %lld elements expected, got shape %s", name, n, shape_of(t).c_str());
  if (t.scalar_type() == at::kInt && t.is_contiguous()) return t;
  if (!at::isIntegralType(t.scalar_type(), false)) raise(PyExc_TypeError, "%s: integers expected, got %s", name, type_of(t).c_str());
  return narrowed(t);
}

struct Batch {
  at::Tensor table, loc, lens;
  lq_batch b;
};
Batch batch(PyObject* table, PyObject* loc, PyObject* lens, const Device& dev, long long T) {
  Batch r;
  const at::Tensor& t = tensor(table, "table");
  dev.on(t, "table");
  if (t.dim() != 2) raise(PyExc_ValueError, "table: [N, pages] expected, got shape %s", shape_of(t).c_str());
  if (!at::isIntegralType(t.scalar_type(), false)) raise(PyExc_TypeError, "table: integers expected, got %s", type_of(t).c_str());
  const long long N = t.size(0), width = t.size(1);
  if (N >= 0x7fffffff || T >= 0x7fffffff || width >= 0x7fffffff) raise(PyExc_ValueError, "at most 2^31 - 2 sequences, tokens and pages a sequence");
  r.table = t.scalar_type() == at::kInt && (width < 2 || t.stride(1) == 1) ? t : narrowed(t);
  r.loc = index(tensor(loc, "loc"), dev, N + 1, "loc");
  r.lens = index(tensor(lens, "lens"), dev, N, "lens");
  r.b = {(const int*)r.loc.data_ptr(), (const int*)r.lens.data_ptr(), (const int*)r.table.data_ptr(), N < 2 ? width : r.table.stride(0),
         (int)width, (int)N, (int)T};
  return r;
}

// (k, v, k_scale, v_scale)
lq_pages pages(PyObject* o, const Device& dev) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) raise(PyExc_TypeError, "pages: Pages(k, v, k_scale, v_scale) expected, got %s", Py_TYPE(o)->tp_name);
  const at::Tensor &k = tensor(PyTuple_GET_ITEM(o, 0), "pages.k"), &v = tensor(PyTuple_GET_ITEM(o, 1), "pages.v");
  const bool int8 = k.scalar_type() == at::kChar;
  if (!int8 && k.scalar_type() != at::kBFloat16) raise(PyExc_TypeError, "pages.k: torch.bfloat16 or torch.int8 expected, got %s", type_of(k).c_str());
  if (v.scalar_type() != k.scalar_type()) raise(PyExc_TypeError, "pages.v: dtype %s, pages.k has %s", type_of(v).c_str(), type_of(k).c_str());
  if (k.dim() != 4 || k.size(0) < 1 || k.size(1) < 1 || k.size(2) < 1)
    raise(PyExc_ValueError, "pages.k: [pages, page, heads, D] expected, got shape %s", shape_of(k).c_str());
  const long long NP = k.size(0), page = k.size(1), HK = k.size(2), D = k.size(3);
  if (D != 64 && D != 128 && D != 256) raise(PyExc_ValueError, "heads of 64, 128 or 256 expected, got %lld", D);
  if (page % 16) raise(PyExc_ValueError, "pages of a multiple of 16 tokens expected, got %lld", page);
  if (v.sizes() != k.sizes() || v.strides() != k.strides())
    raise(PyExc_ValueError, "pages.v: laid out as pages.k expected, got shape %s strides %s", shape_of(v).c_str(), strides_of(v).c_str());
  const int unit = int8 ? 16 : 8;
  const long long page_ld = NP < 2 ? page * HK * D : k.stride(0), head_ld = HK < 2 ? D : k.stride(2), row_ld = k.stride(1);
  if (k.stride(3) != 1 || page_ld % unit || row_ld % unit || head_ld % unit || !aligned(k, 16) || !aligned(v, 16))
    raise(PyExc_ValueError, "pages: packed heads expected, with their start and strides aligned to 16 bytes (strides %s)", strides_of(k).c_str());
  if (NP > 0x7fffffff || HK > 0x7fffffff || page > 1 << 24 || (page - 1) * row_ld + (HK - 1) * head_ld + D > 1 << 29)
    raise(PyExc_ValueError, "pages: the elements of a page within 2^29 expected (shape %s, strides %s)", shape_of(k).c_str(), strides_of(k).c_str());
  lq_pages p = {k.data_ptr(), v.data_ptr(), nullptr, nullptr, page_ld, row_ld, head_ld, 0, 0, 0, (int)NP, (int)page, (int)HK, (int)D, int8};
  PyObject *ks = PyTuple_GET_ITEM(o, 2), *vs = PyTuple_GET_ITEM(o, 3);
  if (int8) {
    const at::Tensor &a = tensor(ks, "pages.k_scale"), &b = tensor(vs, "pages.v_scale");
    for (const at::Tensor* t : {&a, &b}) {
      if (t->scalar_type() != at::kFloat) raise(PyExc_TypeError, "pages: fp32 scales expected, got %s", type_of(*t).c_str());
      if (t->dim() != 3 || t->size(0) != NP || t->size(1) != page || t->size(2) != HK || t->strides() != a.strides())
        raise(PyExc_ValueError, "pages: scales [%lld, %lld, %lld] laid out alike expected, got shape %s strides %s", NP, page, HK,
              shape_of(*t).c_str(), strides_of(*t).c_str());
      dev.on(*t, "pages' scales");
    }
    p.k_scale = (float*)a.data_ptr();
    p.v_scale = (float*)b.data_ptr();
    p.s_page_ld = a.stride(0); p.s_row_ld = a.stride(1); p.s_head_ld = a.stride(2);
  } else if (ks != Py_None || vs != Py_None) {
    raise(PyExc_ValueError, "pages: scales belong to pages in 8 bits");
  }
  dev.on(k, "pages.k");
  dev.on(v, "pages.v");
  return p;
}
void limits(const lq_batch& b, const lq_pages& p, long long most) {
  if ((long long)b.width * p.page > most || (unsigned long long)b.width * p.page * (unsigned long long)p.page >= 1ull << 40)
    raise(PyExc_ValueError, "table: %d pages of %d tokens are more than the kernels' places hold", b.width, p.page);
}
// a weight of D elements in fp32 or bf16 (true)
bool weight(const at::Tensor& t, const Device& dev, long long D, const char* name) {
  dev.on(t, name);
  const bool bf16 = t.scalar_type() == at::kBFloat16;
  if (t.dim() != 1 || t.size(0) != D || !t.is_contiguous() || (!bf16 && t.scalar_type() != at::kFloat) || !aligned(t, 16))
    raise(PyExc_ValueError, "%s: contiguous, 16-byte aligned fp32 or bf16 [%lld] expected, got %s %s", name, D, type_of(t).c_str(), shape_of(t).c_str());
  return bf16;
}

template <typename F> PyObject* status(const char* name, F call) {
  try {
    const int rc = call();
    if (rc == 0) Py_RETURN_NONE;
    PyErr_Format(PyExc_RuntimeError, "%s failed: %s (status %d)", name,
                 rc == LQ_ERR_ARG ? "bad argument (unsupported shape / size / pointer)" : "HIP launch error", rc);
  } catch (const Raised&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_Clear();
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_Clear();
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_Clear();
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_Clear();
    PyErr_Format(PyExc_RuntimeError, "%s: unknown error", name);
  }
  return nullptr;
}
void arguments(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) raise(PyExc_TypeError, "%zd arguments expected, got %zd", want, got);
}
// [T, H, D] of a query tensor
void heads_of(const at::Tensor& q) {
  if (q.dim() != 3 || q.size(1) < 1) raise(PyExc_ValueError, "q: [T, heads, D] expected, got shape %s", shape_of(q).c_str());
  if (q.size(0) >= 0x7fffffff || q.size(1) > 1 << 20) raise(PyExc_ValueError, "q: at most 2^31 - 2 tokens and 2^20 heads, got shape %s", shape_of(q).c_str());
}

// (q, k, v, q_weight, k_weight, inv_freq, pages, table, loc, lens, out, eps, offset, interleaved)
PyObject* rope_norm(PyObject*, PyObject* const* arg, Py_ssize_t count) {
  return status("lq_rope_norm", [&] {
    arguments(count, 14);
    const at::Tensor& q = tensor(arg[0], "q");
    const Device dev(q);
    const lq_pages p = pages(arg[6], dev);
    heads_of(q);
    const long long T = q.size(0), HQ = q.size(1), D = p.D, HK = p.HK;
    lq_rope r = {};
    r.q = rows(q, dev, T, HQ, D, "q");
    r.k = rows(tensor(arg[1], "k"), dev, T, HK, D, "k");
    r.v = rows(tensor(arg[2], "v"), dev, T, HK, D, "v");
    r.out = rows(tensor(arg[10], "out"), dev, T, HQ, D, "out");
    apart(r.out, T, HQ, D);
    const at::Tensor &qw = tensor(arg[3], "q_weight"), &kw = tensor(arg[4], "k_weight"), &f = tensor(arg[5], "inv_freq");
    r.weight_bf16 = weight(qw, dev, D, "q_weight") + 2 * weight(kw, dev, D, "k_weight");
    r.q_weight = qw.data_ptr();
    r.k_weight = kw.data_ptr();
    dev.on(f, "inv_freq");
    r.freq64 = f.scalar_type() == at::kDouble;
    if (f.dim() != 1 || !f.is_contiguous() || (!r.freq64 && f.scalar_type() != at::kFloat))
      raise(PyExc_ValueError, "inv_freq: contiguous fp32 or fp64 [rot / 2] expected, got %s %s", type_of(f).c_str(), shape_of(f).c_str());
    if (2 * f.size(0) > D || f.size(0) % 8) raise(PyExc_ValueError, "inv_freq: a multiple of 8 elements, at most %lld, expected, got %lld", D / 2, (long long)f.size(0));
    r.inv_freq = f.data_ptr();
    r.HQ = (int)HQ;
    r.rot = 2 * (int)f.size(0);
    r.eps = (float)number(arg[11], "eps");
    if (!(r.eps >= 0.f)) raise(PyExc_ValueError, "eps: 0 or more expected");
    r.offset = (float)number(arg[12], "offset");
    r.interleaved = truth(arg[13]);
    const Batch b = batch(arg[7], arg[8], arg[9], dev, T);
    limits(b.b, p, 0x7ffffffell);
    dev.gpu();
    const Current current(dev.dev);
    return lq_rope_norm(&r, &p, &b.b, stream(dev.dev));
  });
}

// (q, pages, table, loc, lens, out, scale, window, gate, longest)
PyObject* attend(PyObject*, PyObject* const* arg, Py_ssize_t count) {
  return status("lq_attend", [&] {
    arguments(count, 10);
    const at::Tensor& q = tensor(arg[0], "q");
    const Device dev(q);
    const lq_pages p = pages(arg[1], dev);
    heads_of(q);
    const long long T = q.size(0), HQ = q.size(1), D = p.D;
    if (HQ % p.HK) raise(PyExc_ValueError, "%d heads of the pages do not divide %lld heads of q", p.HK, HQ);
    lq_attention a = {};
    a.q = rows(q, dev, T, HQ, D, "q");
    a.out = rows(tensor(arg[5], "out"), dev, T, HQ, D, "out");
    apart(a.out, T, HQ, D);
    if (arg[8] != Py_None) a.gate = rows(tensor(arg[8], "gate"), dev, T, HQ, D, "gate");
    a.HQ = (int)HQ;
    const double scale = arg[6] == Py_None ? 1.0 / std::sqrt((double)D) : number(arg[6], "scale");
    a.scale = (float)scale;
    if (!(a.scale > 0.f) || a.scale >= 0x1p127f) raise(PyExc_ValueError, "scale: positive and below 2^127 expected");
    const long long window = integer(arg[7], "window"), longest = arg[9] == Py_None ? 0 : integer(arg[9], "longest");
    if (window < 0 || window > 0x7fffffff) raise(PyExc_ValueError, "window: 0 (none) or a number of tokens expected, got %lld", window);
    if (longest < 0) raise(PyExc_ValueError, "longest: a number of tokens expected, got %lld", longest);
    a.window = (int)window;
    const Batch b = batch(arg[2], arg[3], arg[4], dev, T);
    limits(b.b, p, 0x7fffffffll - 4096);
    dev.gpu();
    const Current current(dev.dev);
    const int most = (int)(longest < T ? longest : T);
    const long long need = lq_attend_workspace(&a, &p, &b.b, most);
    if (need < 0) return (int)need;
    at::Tensor work;
    if (need > 0) work = at::empty({need}, at::TensorOptions().dtype(at::kByte).device(q.device()));
    return lq_attend(&a, &p, &b.b, most, need > 0 ? work.data_ptr() : nullptr, need, stream(dev.dev));
  });
}

PyMethodDef methods[] = {{"rope_norm", (PyCFunction)(void (*)())rope_norm, METH_FASTCALL, nullptr},
                         {"attend", (PyCFunction)(void (*)())attend, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "lq_attn_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_lq_attn_call() {
  PyObject* m = PyModule_Create(&module);
  if (!m) return nullptr;
  PyModule_AddIntConstant(m, "ABI", LQ_ATTN_ABI_VERSION);
  PyModule_AddStringConstant(m, "TORCH", LQ_TORCH_VERSION);      // whose tensors the functions read
  return m;
}
