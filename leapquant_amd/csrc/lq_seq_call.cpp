// The calls of leapquant_amd/seq.py whose arguments are as the kernels read them, without the interpreter's time for each
// attribute of each tensor (a call on small tensors is mostly host time: 10.8 -> 5.1 us for the rule's steps, 6.1 -> 3.4 for a
// norm).
// Each function checks all that the Python operator checks.  It returns the C entry's status, or NOT_PLAIN, having done
// nothing: the operator then goes on in Python, which converts what may be converted and says what is wrong with the rest.
// No C++ exception leaves; the only Python one is that of the callable that `delta` calls.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/lq_seq.h"

namespace {

constexpr int NOT_PLAIN = 1;
struct NotPlain {};
struct Raised {};                        // a Python exception is set
void need(bool ok) { if (!ok) throw NotPlain(); }

const at::Tensor& tensor(PyObject* o) {
  need(THPVariable_CheckExact(o));
  return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o) { return o == Py_None ? nullptr : &tensor(o); }
long long integer(PyObject* o) {
  need(PyLong_Check(o));
  const long long v = PyLong_AsLongLong(o);
  need(v != -1 || !PyErr_Occurred());
  return v;
}
double number(PyObject* o) {
  need(PyFloat_Check(o) || PyLong_Check(o));
  const double v = PyFloat_AsDouble(o);
  need(v != -1.0 || !PyErr_Occurred());
  return v;
}
bool aligned(const at::Tensor& t, int bytes) { return (uintptr_t)t.data_ptr() % bytes == 0; }
bool bf16(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16; }
void on(int dev, const at::Tensor& t) { need(t.is_cuda() && t.get_device() == dev); }

// row stride of a bf16 [T, C] with packed rows whose start and stride are multiples of `align` elements
long long row_stride(const at::Tensor& t, int dev, long long T, long long C, int align) {
  on(dev, t);
  need(bf16(t) && t.dim() == 2 && t.size(0) == T && t.size(1) == C && (t.stride(1) == 1 || C <= 1));
  const long long ld = T < 2 ? (C + align - 1) / align * align : t.stride(0);
  need(ld >= C && ld % align == 0 && aligned(t, 2 * align));
  return ld;
}
const int* index(const at::Tensor& t, int dev, long long n) {
  on(dev, t);
  need(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous());
  return (const int*)t.data_ptr();
}
lq_seqs batch(PyObject* idx, PyObject* loc, PyObject* src, int dev, long long T) {
  const at::Tensor& i = tensor(idx);
  need(i.dim() == 1 && i.size(0) < 0x7fffffff && T <= 0x7fffffff);
  const at::Tensor* s = maybe(src);
  const long long N = i.size(0);
  return {index(tensor(loc), dev, N + 1), index(i, dev, N), s ? index(*s, dev, N) : nullptr, (int)N, (int)T};
}
// a gate parameter: n values, fp32 or bf16 (returns 1)
int gate(const at::Tensor& t, int dev, long long n) {
  on(dev, t);
  need(t.numel() == n && t.is_contiguous() && (bf16(t) || t.scalar_type() == at::kFloat));
  return bf16(t);
}
void* stream(int dev) { return (void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream(); }

// `dev` current while this lives: a launch on a default stream goes to the current device, whatever its tensors are on
struct Current {
  const c10::DeviceIndex dev, was;
  explicit Current(int d) : dev((c10::DeviceIndex)d), was(c10::hip::ExchangeDevice(dev)) {}
  ~Current() { if (was != dev) (void)c10::hip::SetDevice(was); }
};

template <typename F> PyObject* status(F call) {
  int rc = NOT_PLAIN;
  try {
    rc = call();
  } catch (const Raised&) {
    return nullptr;
  } catch (...) {
    PyErr_Clear();
  }
  return PyLong_FromLong(rc);
}

// (S, mixed, a, b, A_log, dt_bias, idx, loc, out, src, H, scale, kda, glb, chunks, before): `before`, None or a callable, is
// called once nothing is left that refuses the call, right before the launch
PyObject* delta(PyObject*, PyObject* const* arg, Py_ssize_t count) {
  return status([&] {
    need(count == 16);
    const at::Tensor& S = tensor(arg[0]);
    need(S.is_cuda() && S.scalar_type() == at::kFloat && S.dim() == 4);
    const int dev = S.get_device();
    const long long NS = S.size(0), HV = S.size(1), V = S.size(2), K = S.size(3), H = integer(arg[10]);
    const bool kda = arg[12] == Py_True, chunks = arg[14] == Py_True;
    need((kda || arg[12] == Py_False) && (chunks || arg[14] == Py_False));
    need((K == 128 && V == 128) || (!kda && K == 64 && (V == 128 || V == 64)));
    need(H > 0 && HV > 0 && HV % H == 0 && NS <= 0x7fffffff && HV <= 0x7fffffff / 256);
    const long long SS = NS < 2 ? HV * V * K : S.stride(0), KA = kda ? K : 1;
    need(S.stride(1) == V * K && S.stride(2) == K && S.stride(3) == 1 && aligned(S, 16) && SS % 4 == 0 && SS >= HV * V * K);
    const at::Tensor &mixed = tensor(arg[1]), &a = tensor(arg[2]), &b = tensor(arg[3]), &out = tensor(arg[8]);
    need(mixed.dim() == 2);
    const long long T = mixed.size(0), mixed_ld = row_stride(mixed, dev, T, 2 * H * K + HV * V, 8);
    const long long b_ld = row_stride(b, dev, T, HV, 1);
    long long a_ld;
    if (kda && a.dim() == 3) {                   // packed rows [HV, K]
      on(dev, a);
      need(bf16(a) && a.size(0) == T && a.size(1) == HV && a.size(2) == K && a.stride(1) == K && a.stride(2) == 1);
      a_ld = T < 2 ? HV * K : a.stride(0);
      need(a_ld >= HV * K && a_ld % 4 == 0 && aligned(a, 8));
    } else {
      a_ld = row_stride(a, dev, T, HV * KA, kda ? 4 : 1);
    }
    on(dev, out);
    need(bf16(out) && out.dim() == 3 && out.size(0) == T && out.size(1) == HV && out.size(2) == V && out.is_contiguous());
    need(aligned(out, 16) && (!chunks || (T * HV <= 1 << 30 && mixed_ld <= 1 << 24)));
    const at::Tensor &A_log = tensor(arg[4]), &dt_bias = tensor(arg[5]);
    const int gate_bf16 = gate(A_log, dev, HV) + 2 * gate(dt_bias, dev, HV * KA);
    const lq_seqs s = batch(arg[6], arg[7], arg[9], dev, T);
    const float scale = arg[11] == Py_None ? (float)(1.0 / std::sqrt((double)K)) : (float)number(arg[11]);
    const lq_delta d = {(float*)S.data_ptr(), SS, (int)NS, (int)HV, (int)H, (int)K, (int)V, mixed.data_ptr(), a.data_ptr(),
                        b.data_ptr(), A_log.data_ptr(), dt_bias.data_ptr(), out.data_ptr(), mixed_ld, a_ld, b_ld, scale,
                        gate_bf16, kda, (float)number(arg[13])};
    const Current current(dev);
    if (int rc = lq_delta_check(&d, &s, chunks)) return rc;
    const long long n = chunks ? lq_delta_workspace(&d, &s) : 0;
    at::Tensor work;
    if (n > 0) work = at::empty({n}, at::TensorOptions().dtype(at::kByte).device(S.device()));
    void* const st = stream(dev);
    if (arg[15] != Py_None) {
      PyObject* r = PyObject_CallNoArgs(arg[15]);
      if (!r) throw Raised();
      Py_DECREF(r);
    }
    return chunks ? lq_delta_prefill(&d, &s, n > 0 ? work.data_ptr() : nullptr, n, st) : lq_delta_steps(&d, &s, st);
  });
}

// (x, conv_state, weight, bias, idx, loc, out, src, silu)
PyObject* conv(PyObject*, PyObject* const* arg, Py_ssize_t count) {
  return status([&] {
    need(count == 9);
    const at::Tensor &x = tensor(arg[0]), &st = tensor(arg[1]), &w = tensor(arg[2]), &out = tensor(arg[6]);
    need(x.is_cuda() && x.dim() == 2);
    const int dev = x.get_device();
    const long long T = x.size(0), C = x.size(1), ld = row_stride(x, dev, T, C, 1);
    on(dev, st); on(dev, w); on(dev, out);
    need(C <= 0x7fffffff && bf16(st) && st.dim() == 3 && st.size(1) == C && st.size(2) == 3 && st.size(0) <= 0x7fffffff);
    need(bf16(w) && w.dim() == 2 && w.size(0) == C && w.size(1) == 4 && w.is_contiguous());
    need(bf16(out) && out.dim() == 2 && out.size(0) == T && out.size(1) == C && out.is_contiguous());
    const at::Tensor* bias = maybe(arg[3]);
    if (bias) {
      on(dev, *bias);
      need(bf16(*bias) && bias->numel() == C && bias->is_contiguous());
    }
    const lq_seqs s = batch(arg[4], arg[5], arg[7], dev, T);
    need(arg[8] == Py_True || arg[8] == Py_False);
    const lq_conv cv = {st.data_ptr(), w.data_ptr(), bias ? bias->data_ptr() : nullptr, st.stride(0), st.stride(1), st.stride(2),
                        4, arg[8] == Py_True, (int)st.size(0)};
    const Current current(dev);
    return lq_conv_seq(&cv, &s, x.data_ptr(), ld, out.data_ptr(), (int)C, stream(dev));
  });
}

// (x, z, weight, out, res or None, eps, scale, offset, act, add)
PyObject* norm(PyObject*, PyObject* const* arg, Py_ssize_t count) {
  return status([&] {
    need(count == 10);
    const at::Tensor &x = tensor(arg[0]), &z = tensor(arg[1]), &w = tensor(arg[2]), &out = tensor(arg[3]);
    const at::Tensor* res = maybe(arg[4]);
    const bool add = arg[9] == Py_True;
    need(add || arg[9] == Py_False);
    need(add == (res != nullptr));
    const int64_t nd = x.dim();
    need(x.is_cuda() && bf16(x) && nd >= 1 && nd <= 3);
    const int dev = x.get_device();
    const long long D = x.size(nd - 1), rows = nd > 1 ? x.size(0) : 1, heads = nd > 2 ? x.size(1) : 1;
    need(D >= 1 && D <= 16384 && rows <= 0x7fffffff && heads >= 1 && heads <= 0x7fffffff);
    on(dev, z); on(dev, w); on(dev, out);
    need(bf16(z) && bf16(out) && z.sizes() == x.sizes() && out.sizes() == x.sizes());
    need(D == 1 || (x.stride(nd - 1) == 1 && z.stride(nd - 1) == 1 && out.stride(nd - 1) == 1));
    need(nd < 2 || rows < 2 || out.stride(0) >= D);        // rows and heads of their own
    need(nd < 3 || heads < 2 || out.stride(1) >= D);
    if (res) {
      on(dev, *res);
      need(bf16(*res) && res->sizes() == x.sizes() && res->strides() == out.strides());
    }
    const bool wide = w.scalar_type() == at::kFloat;
    need(w.dim() == 1 && w.size(0) == D && w.is_contiguous() && (wide || bf16(w)));
    auto row = [&](const at::Tensor& t) { return nd > 1 ? (long long)t.stride(0) : 0; };
    auto head = [&](const at::Tensor& t) { return nd > 2 ? (long long)t.stride(1) : 0; };
    const lq_norm n = {x.data_ptr(), z.data_ptr(), w.data_ptr(), res ? res->data_ptr() : nullptr, out.data_ptr(),
                       row(x), head(x), row(z), head(z), row(out), head(out), (int)rows, (int)heads, (int)D,
                       (float)number(arg[5]), (float)number(arg[6]), (float)number(arg[7]), (int)integer(arg[8]), !wide};
    const Current current(dev);
    return add ? lq_add_norm(&n, stream(dev)) : lq_gated_norm(&n, stream(dev));
  });
}

PyMethodDef methods[] = {{"delta", (PyCFunction)(void (*)())delta, METH_FASTCALL, nullptr},
                         {"conv", (PyCFunction)(void (*)())conv, METH_FASTCALL, nullptr},
                         {"norm", (PyCFunction)(void (*)())norm, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "lq_seq_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_lq_seq_call() {
  PyObject* m = PyModule_Create(&module);
  if (!m) return nullptr;
  PyModule_AddIntConstant(m, "NOT_PLAIN", NOT_PLAIN);
  PyModule_AddIntConstant(m, "ABI", LQ_SEQ_ABI_VERSION);
  PyModule_AddStringConstant(m, "TORCH", LQ_TORCH_VERSION);      // whose tensors the functions read
  return m;
}
