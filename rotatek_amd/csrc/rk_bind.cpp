// rk_bind.cpp -- host path of the quantised and shared-prefix calls: torch
// tensors to rk_tensor descriptors, output and workspace from torch's allocator,
// and the library's entry point, in one C++ call from Python.
//
// The smallest of these calls keep the GPU busy for 8 to 14 us.  Formed in Python
// (ten descriptors, two allocations, a ctypes call) a decode call took 20 us to
// issue; two launches of about 3.5 us each are what it cannot do without.
//
// Module `rotatek_amd._bind`, loaded by _lib.bind(), which hands it the addresses
// of the entry points of the library that ctypes has loaded.  A call returns its
// result or, as an int, the status that refused it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "rotatek_hip.h"

namespace {

constexpr int kOtherDevice = -1000;  // a tensor is not on the call's GPU: the caller words the error

struct Entries {
  decltype(&rk_mx_write) write;
  decltype(&rk_mx_read) read;
  decltype(&rk_mx_append) append;
  decltype(&rk_quantized_decode_check) decode_check;
  decltype(&rk_quantized_decode) decode;
  decltype(&rk_shared_prefix_decode_check) shared_check;
  decltype(&rk_shared_prefix_decode) shared;
} g_entry;

PyObject *g_codes, *g_scales, *g_head_dim, *g_fmt;  // attribute names of MXRows

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return RK_F16;
    case at::kBFloat16: return RK_BF16;
    case at::kFloat: return RK_F32;
    case at::kDouble: return RK_F64;
    case at::kByte:
    case at::kBool: return RK_U8;
    case at::kInt: return RK_I32;
    case at::kLong: return RK_I64;
    default: return -1;
  }
}

// What a call writes is asked for as mutable: a tensor that shares its memory
// until it is written (copy-on-write) gets its own then.
enum Use { kRead, kWrite };

int describe(const at::Tensor& t, int64_t device, rk_tensor* d, Use use) {
  if (!t.device().is_cuda() || t.get_device() != device) return kOtherDevice;
  const int64_t nd = t.dim();
  const int32_t code = dtype_code(t.scalar_type());
  if (nd > 4) return RK_ERR_RANK;
  if (code < 0) return RK_ERR_DTYPE;
  memset(d, 0, sizeof(*d));
  d->data = t.numel() == 0 ? nullptr : use == kWrite ? t.mutable_data_ptr() : const_cast<void*>(t.const_data_ptr());
  d->dtype = code;
  d->ndim = (int32_t)nd;
  for (int64_t i = 0; i < nd; ++i) {
    d->shape[i] = t.size(i);
    d->stride[i] = t.stride(i);
  }
  return RK_OK;
}

// An optional tensor argument: its descriptor, or null for None.
struct Arg {
  rk_tensor d;
  const rk_tensor* p = nullptr;
  int set(PyObject* o, int64_t device, Use use = kRead) {
    if (o == Py_None) return RK_OK;
    if (!THPVariable_Check(o)) return RK_ERR_ARG;
    p = &d;
    return describe(THPVariable_Unpack(o), device, &d, use);
  }
};

int format_of(PyObject* fmt) {
  if (!PyUnicode_Check(fmt)) return -1;
  return PyUnicode_CompareWithASCIIString(fmt, "mx8") == 0   ? RK_ROWS_MX8
         : PyUnicode_CompareWithASCIIString(fmt, "mx4") == 0 ? RK_ROWS_MX4
                                                             : -1;
}

// Rows: None, a plain [B, H, S, D] tensor or MXRows.
struct RowsArg {
  rk_rows d;
  const rk_rows* p = nullptr;
  // a Python error is left where MXRows' attributes are not what they should be
  int set(PyObject* o, int64_t device, Use use = kRead) {
    if (o == Py_None) return RK_OK;
    p = &d;
    memset(&d, 0, sizeof(d));
    if (THPVariable_Check(o)) {
      const at::Tensor& t = THPVariable_Unpack(o);
      d.head_dim = t.dim() > 0 ? t.size(-1) : 0;
      d.format = RK_ROWS_PLAIN;
      return describe(t, device, &d.data, use);
    }
    int st = RK_ERR_ARG;
    PyObject* codes = PyObject_GetAttr(o, g_codes);
    PyObject* scales = codes ? PyObject_GetAttr(o, g_scales) : nullptr;
    PyObject* dim = scales ? PyObject_GetAttr(o, g_head_dim) : nullptr;
    PyObject* fmt = dim ? PyObject_GetAttr(o, g_fmt) : nullptr;
    if (fmt && THPVariable_Check(codes) && THPVariable_Check(scales) && PyUnicode_Check(fmt)) {
      d.head_dim = PyLong_AsLongLong(dim);
      d.format = format_of(fmt);
      st = d.format < 0 ? RK_ERR_ARG : describe(THPVariable_Unpack(codes), device, &d.data, use);
      if (st == RK_OK) st = describe(THPVariable_Unpack(scales), device, &d.scales, use);
    }
    Py_XDECREF(codes);
    Py_XDECREF(scales);
    Py_XDECREF(dim);
    Py_XDECREF(fmt);
    return st;
  }
};

// The call's GPU as the current one (a tensor elsewhere is refused later).
struct OnDevice {
  c10::OptionalDeviceGuard guard;
  explicit OnDevice(const at::Tensor& t) {
    if (t.device().is_cuda()) guard.reset_device(t.device());
  }
};

// The interpreter runs other threads while the GPU's queue is waited for.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

PyObject* status(int st) { return PyErr_Occurred() ? nullptr : PyLong_FromLong(st); }

at::TensorOptions on(const at::Tensor& like, at::ScalarType type) { return like.options().dtype(type); }

bool counts(const char* name, Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, not %zd", name, want, n);
  return false;
}

void* stream_of(PyObject* o) { return PyLong_AsVoidPtr(o); }

// write(x, rows, fmt, stream): a status; with rows None new rows, (codes,
// scales), or a status
PyObject* py_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts("write", n, 4)) return nullptr;
  if (!THPVariable_Check(a[0])) return status(RK_ERR_ARG);
  const at::Tensor& t = THPVariable_Unpack(a[0]);
  const int64_t dev = t.get_device();
  Arg x;
  RowsArg r;
  const OnDevice guard(t);
  int st = x.set(a[0], dev);
  if (!st) st = r.set(a[1], dev, kWrite);
  void* stream = stream_of(a[3]);
  if (st || PyErr_Occurred()) return status(st);
  at::Tensor new_codes, new_scales;
  if (!r.p) {
    if (t.dim() != 4) return status(RK_ERR_RANK);
    const int64_t D = t.size(3), blocks = (D + 31) / 32, S = t.size(2);
    memset(&r.d, 0, sizeof(r.d));
    r.d.format = format_of(a[2]);
    r.d.head_dim = D;
    if (r.d.format < 0) return status(RK_ERR_ARG);
    if (D > 128) return status(RK_ERR_HEAD_DIM);
    new_codes = at::empty({t.size(0), t.size(1), S, (r.d.format == RK_ROWS_MX8 ? 32 : 16) * blocks}, on(t, at::kByte));
    new_scales = at::empty({t.size(0), t.size(1), blocks, (S + 31) / 32 * 32}, on(t, at::kByte));
    st = describe(new_codes, dev, &r.d.data, kWrite);
    if (!st) st = describe(new_scales, dev, &r.d.scales, kWrite);
    if (st) return status(st);
  }
  {
    const Unlocked unlocked;
    st = g_entry.write(x.p, r.p ? r.p : &r.d, stream);
  }
  if (st || r.p) return status(st);
  PyObject* c = THPVariable_Wrap(new_codes);
  PyObject* e = c ? THPVariable_Wrap(new_scales) : nullptr;
  PyObject* pair = e ? PyTuple_Pack(2, c, e) : nullptr;
  Py_XDECREF(c);
  Py_XDECREF(e);
  return pair;
  END_HANDLE_TH_ERRORS
}

// read(rows, out, dtype, stream): a status; with out None a new tensor of
// `dtype`, or a status
PyObject* py_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts("read", n, 4)) return nullptr;
  PyObject* codes = PyObject_GetAttr(a[0], g_codes);
  if (!codes) return nullptr;
  const bool tensor = THPVariable_Check(codes);
  const at::Tensor t = tensor ? THPVariable_Unpack(codes) : at::Tensor();
  Py_DECREF(codes);
  if (!tensor) return status(RK_ERR_ARG);
  const int64_t dev = t.get_device();
  RowsArg r;
  Arg x;
  const OnDevice guard(t);
  int st = r.set(a[0], dev);
  if (!st) st = x.set(a[1], dev, kWrite);
  void* stream = stream_of(a[3]);
  if (st || PyErr_Occurred()) return status(st);
  at::Tensor out;
  if (!x.p) {
    if (!THPDtype_Check(a[2])) return status(RK_ERR_DTYPE);
    if (t.dim() != 4) return status(RK_ERR_RANK);
    if (r.d.head_dim < 0) return status(RK_ERR_HEAD_DIM);
    out = at::empty({t.size(0), t.size(1), t.size(2), r.d.head_dim},
                    on(t, reinterpret_cast<THPDtype*>(a[2])->scalar_type));
    st = describe(out, dev, &x.d, kWrite);
    if (st) return status(st);
  }
  {
    const Unlocked unlocked;
    st = g_entry.read(r.p, x.p ? x.p : &x.d, stream);
  }
  if (st || x.p) return status(st);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// A contiguous int32 [B] on the device, or null for None.
int lengths(PyObject* o, int64_t device, int64_t batch, const int32_t** p, Use use = kRead) {
  *p = nullptr;
  if (o == Py_None) return RK_OK;
  if (!THPVariable_Check(o)) return RK_ERR_ARG;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.device().is_cuda() || t.get_device() != device) return kOtherDevice;
  if (t.scalar_type() != at::kInt) return RK_ERR_DTYPE;
  if (t.dim() != 1 || t.size(0) != batch || !t.is_contiguous()) return RK_ERR_SHAPE;
  *p = static_cast<const int32_t*>(use == kWrite ? t.mutable_data_ptr() : t.const_data_ptr());
  return RK_OK;
}

// append(k_new, v_new, k_rows, v_rows, lens, advance, stream)
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts("append", n, 7)) return nullptr;
  if (!THPVariable_Check(a[0])) return status(RK_ERR_ARG);
  const at::Tensor& t = THPVariable_Unpack(a[0]);
  const int64_t dev = t.get_device();
  Arg k, v;
  RowsArg kr, vr;
  const int32_t* lens = nullptr;
  const int advance = PyObject_IsTrue(a[5]);
  if (advance < 0) return nullptr;
  const OnDevice guard(t);
  int st = k.set(a[0], dev);
  if (!st) st = v.set(a[1], dev);
  if (!st) st = kr.set(a[2], dev, kWrite);
  if (!st) st = vr.set(a[3], dev, kWrite);
  if (!st) st = lengths(a[4], dev, t.dim() > 0 ? t.size(0) : 0, &lens, advance ? kWrite : kRead);
  if (st) return status(st);
  void* stream = stream_of(a[6]);
  {
    const Unlocked unlocked;
    st = g_entry.append(k.p, v.p, kr.p, vr.p, const_cast<int32_t*>(lens), advance, stream);
  }
  return status(st);
  END_HANDLE_TH_ERRORS
}

// decode(shared, q, R, delta_mu, k_full, v_full, k_sparse, v_sparse, k_suffix,
// v_suffix, mask, lens, groups, out, stream): out [B, 1, H_q, D], or a status
PyObject* py_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts("decode", n, 15)) return nullptr;
  const bool shared = a[0] == Py_True;
  if (!THPVariable_Check(a[1])) return status(RK_ERR_ARG);
  const at::Tensor& q = THPVariable_Unpack(a[1]);
  const int64_t dev = q.get_device();
  Arg dq, dR, dmu, dmask, dout;
  RowsArg r[6];
  const int32_t* lens = nullptr;
  const OnDevice guard(q);
  int st = dq.set(a[1], dev);
  if (!st) st = dR.set(a[2], dev);
  if (!st) st = dmu.set(a[3], dev);
  for (int i = 0; i < 6 && !st; ++i) st = r[i].set(a[4 + i], dev);
  if (!st) st = dmask.set(a[10], dev);
  if (!st && q.dim() != 3) st = RK_ERR_RANK;
  if (!st) st = lengths(a[11], dev, q.size(0), &lens);
  if (st) return status(st);
  const int64_t groups = PyLong_AsLongLong(a[12]);
  void* stream = stream_of(a[14]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor out;
  if (a[13] == Py_None) {
    out = at::empty({q.size(0), 1, q.size(1), q.size(2)}, on(q, q.scalar_type()));
    dout.p = &dout.d;
    st = describe(out, dev, &dout.d, kWrite);
    dout.d.ndim = 3;
    for (int i = 1; i < 3; ++i) {
      dout.d.shape[i] = out.size(i + 1);
      dout.d.stride[i] = out.stride(i + 1);
    }
    dout.d.shape[3] = dout.d.stride[3] = 0;
  } else {
    st = dout.set(a[13], dev, kWrite);
    if (!st) out = THPVariable_Unpack(a[13]).unsqueeze(1);
  }
  if (st) return status(st);
  size_t bytes = 0;
  st = shared ? g_entry.shared_check(dq.p, dR.p, dmu.p, r[0].p, r[1].p, r[2].p, r[3].p, r[4].p, r[5].p, groups, dout.p,
                                     0, &bytes)
              : g_entry.decode_check(dq.p, dR.p, dmu.p, r[0].p, r[1].p, dmask.p, r[2].p, r[3].p, groups, dout.p, 0,
                                     &bytes);
  if (st) return status(st);
  // the call's own: torch's allocator hands it on in the stream's order
  const at::Tensor ws = at::empty({(int64_t)(bytes > 0 ? bytes : 256)}, on(q, at::kByte));
  {
    const Unlocked unlocked;
    st = shared ? g_entry.shared(dq.p, dR.p, dmu.p, r[0].p, r[1].p, r[2].p, r[3].p, r[4].p, r[5].p, lens, groups,
                                 dout.p, ws.data_ptr(), (size_t)ws.numel(), stream)
                : g_entry.decode(dq.p, dR.p, dmu.p, r[0].p, r[1].p, dmask.p, lens, r[2].p, r[3].p, groups, dout.p,
                                 ws.data_ptr(), (size_t)ws.numel(), stream);
  }
  if (st) return status(st);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// init(write, read, append, decode_check, decode, shared_check, shared): addresses
PyObject* py_init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counts("init", n, 7)) return nullptr;
  void* p[7];
  for (int i = 0; i < 7; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g_entry.write = reinterpret_cast<decltype(g_entry.write)>(p[0]);
  g_entry.read = reinterpret_cast<decltype(g_entry.read)>(p[1]);
  g_entry.append = reinterpret_cast<decltype(g_entry.append)>(p[2]);
  g_entry.decode_check = reinterpret_cast<decltype(g_entry.decode_check)>(p[3]);
  g_entry.decode = reinterpret_cast<decltype(g_entry.decode)>(p[4]);
  g_entry.shared_check = reinterpret_cast<decltype(g_entry.shared_check)>(p[5]);
  g_entry.shared = reinterpret_cast<decltype(g_entry.shared)>(p[6]);
  Py_RETURN_NONE;
}

#define RK_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {RK_METHOD(init),   RK_METHOD(write),  RK_METHOD(read),
                           RK_METHOD(append), RK_METHOD(decode), {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind(void) {
  g_codes = PyUnicode_InternFromString("codes");
  g_scales = PyUnicode_InternFromString("scales");
  g_head_dim = PyUnicode_InternFromString("head_dim");
  g_fmt = PyUnicode_InternFromString("fmt");
  PyObject* m = PyModule_Create(&g_module);
  if (m && PyModule_AddIntConstant(m, "OTHER_DEVICE", kOtherDevice) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
