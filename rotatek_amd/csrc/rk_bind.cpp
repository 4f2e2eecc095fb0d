// rk_bind.cpp -- host path of the quantised, shared-prefix and paged calls: torch
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
#include <ATen/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "rotatek_hip.h"

namespace {

constexpr int kOtherDevice = -1000;  // a tensor is not on the call's GPU: the caller words the error
constexpr int kNeedsGrad = -1001;    // a gradient is asked of a call that has none

struct Entries {
  decltype(&rk_mx_write) write;
  decltype(&rk_mx_read) read;
  decltype(&rk_mx_append) append;
  decltype(&rk_quantized_decode_check) decode_check;
  decltype(&rk_quantized_decode) decode;
  decltype(&rk_shared_prefix_decode_check) shared_check;
  decltype(&rk_shared_prefix_decode) shared;
  decltype(&rk_rotary) rotary;
  decltype(&rk_paged_append) paged_append;
  decltype(&rk_paged_attention_check) paged_check;
  decltype(&rk_paged_attention) paged;
  decltype(&rk_window_attention_check) window_check;
  decltype(&rk_window_attention) window;
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
  if (t.is_neg()) return RK_ERR_ARG;  // its memory holds the negatives (the caller words it)
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

// ---- paged cache

// Whether autograd would record one of these, or follow its tangent (which it does
// without recording too).
template <class... T>
bool needs_grad(T... o) {
  const bool records = c10::GradMode::is_enabled();
  const bool tangents = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (PyObject* x : {o...}) {
    if (!THPVariable_Check(x)) continue;
    const at::Tensor& t = THPVariable_Unpack(x);
    if ((records && t.requires_grad()) || (tangents && t._fw_grad(0).defined())) return true;
  }
  return false;
}

// Marks tensors that a call has written (None among them), for autograd, which may have
// saved them.  Those of inference mode have no count.
template <class... T>
void written(T... o) {
  for (PyObject* x : {o...}) {
    if (!THPVariable_Check(x)) continue;
    const at::Tensor& t = THPVariable_Unpack(x);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
}

// A new tensor, from the allocator of a given one: what at::empty does behind its two
// dispatches (a rotation of one token's queries and Keys 7.1 us with them, 5.9 so).
at::Tensor fresh(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
  c10::Allocator* const from = like.storage().allocator();
  if (!from || !like.is_cuda()) return at::empty(sizes, on(like, type));
  return at::detail::empty_generic(sizes, from, c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}

// A new tensor like t, and its descriptor.
int make_like(const at::Tensor& t, int64_t device, at::Tensor* out, Arg* d) {
  *out = fresh(t, t.sizes(), t.scalar_type());
  d->p = &d->d;
  return describe(*out, device, &d->d, kWrite);
}

// Pairs of each axis, a sequence of integers, or None: one axis of them all.
struct Sections {
  int32_t n[4];
  int32_t axes = 0;
  int set(PyObject* o, int64_t pairs) {
    if (o == Py_None) {
      axes = 1;
      n[0] = (int32_t)(pairs < 0 || pairs > 1024 ? 0 : pairs);
      return RK_OK;
    }
    PyObject* seq = PySequence_Fast(o, "sections must be a sequence of integers");
    if (!seq) return RK_ERR_ARG;
    const Py_ssize_t size = PySequence_Fast_GET_SIZE(seq);
    int st = size < 1 || size > 4 ? RK_ERR_ARG : RK_OK;
    for (Py_ssize_t i = 0; i < size && !st; ++i) {
      const long long x = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq, i));
      if (x < 0 || x > 1024) st = RK_ERR_ARG;
      n[i] = (int32_t)x;
    }
    axes = (int32_t)size;
    Py_DECREF(seq);
    return st;
  }
};

// rotary(q, k, positions, inv_freq, sections, interleaved, inverse, q_out,
// k_out, stream): (q_out, k_out), or a status
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts("rotary", n, 10)) return nullptr;
  if (!THPVariable_Check(a[0])) return status(RK_ERR_ARG);
  if (needs_grad(a[0], a[1], a[3], a[7], a[8])) return status(kNeedsGrad);
  const at::Tensor& t = THPVariable_Unpack(a[0]);
  const int64_t dev = t.get_device();
  Arg q, k, pos, freq, qo, ko;
  Sections sections;
  const int interleaved = PyObject_IsTrue(a[5]), inverse = PyObject_IsTrue(a[6]);
  if (interleaved < 0 || inverse < 0) return nullptr;
  const OnDevice guard(t);
  int st = q.set(a[0], dev);
  if (!st) st = k.set(a[1], dev);
  if (!st) st = pos.set(a[2], dev);
  if (!st) st = freq.set(a[3], dev);
  if (!st) st = sections.set(a[4], freq.p && freq.d.ndim == 1 ? freq.d.shape[0] : 0);
  if (!st) st = qo.set(a[7], dev, kWrite);
  if (!st) st = ko.set(a[8], dev, kWrite);
  void* stream = stream_of(a[9]);
  if (st || PyErr_Occurred()) return status(st);
  at::Tensor new_q, new_k;
  if (!qo.p) st = make_like(t, dev, &new_q, &qo);
  if (!st && k.p && !ko.p) st = make_like(THPVariable_Unpack(a[1]), dev, &new_k, &ko);
  if (st) return status(st);
  {
    const Unlocked unlocked;
    st = g_entry.rotary(q.p, k.p, pos.p, freq.p, sections.n, sections.axes, interleaved, inverse, qo.p, ko.p, stream);
  }
  if (st) return status(st);
  written(a[7], a[8]);
  PyObject* x = new_q.defined() ? THPVariable_Wrap(new_q) : Py_NewRef(a[7]);
  PyObject* y = !x ? nullptr : new_k.defined() ? THPVariable_Wrap(new_k) : Py_NewRef(a[8]);
  PyObject* pair = y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return pair;
  END_HANDLE_TH_ERRORS
}

// Pages, their table and lengths, of the call's device.
struct PagesArg {
  rk_pages d;
  int64_t requests = 0;
  int set(PyObject* k, PyObject* v, PyObject* table, PyObject* lens, int64_t device, Use use = kRead) {
    memset(&d, 0, sizeof(d));
    if (!THPVariable_Check(k) || !THPVariable_Check(v) || !THPVariable_Check(table) || !THPVariable_Check(lens))
      return RK_ERR_ARG;
    const at::Tensor& t = THPVariable_Unpack(table);
    int st = describe(THPVariable_Unpack(k), device, &d.k, use);
    if (!st) st = describe(THPVariable_Unpack(v), device, &d.v, use);
    if (!st) st = describe(t, device, &d.table, kRead);
    requests = t.dim() > 0 ? t.size(0) : 0;
    return st ? st : lengths(lens, device, requests, &d.lens);
  }
};

// paged_append(k_new, v_new, k_pages, v_pages, table, lens, starts, q, q_out,
// positions, inv_freq, sections, interleaved, stream): q_out or None, or a status
PyObject* py_paged_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts("paged_append", n, 14)) return nullptr;
  if (!THPVariable_Check(a[0])) return status(RK_ERR_ARG);
  if (needs_grad(a[0], a[1], a[2], a[3], a[7], a[8], a[10])) return status(kNeedsGrad);
  const at::Tensor& t = THPVariable_Unpack(a[0]);
  const int64_t dev = t.get_device();
  Arg k, v, q, qo, pos, freq;
  PagesArg pages;
  Sections sections;
  const int32_t* starts = nullptr;
  const int interleaved = PyObject_IsTrue(a[12]);
  if (interleaved < 0) return nullptr;
  const OnDevice guard(t);
  int st = k.set(a[0], dev);
  if (!st) st = v.set(a[1], dev);
  if (!st) st = pages.set(a[2], a[3], a[4], a[5], dev, kWrite);
  if (!st) st = lengths(a[6], dev, pages.requests + 1, &starts);
  if (!st) st = q.set(a[7], dev);
  if (!st) st = qo.set(a[8], dev, kWrite);
  if (!st) st = pos.set(a[9], dev);
  if (!st) st = freq.set(a[10], dev);
  if (!st && pos.p) st = sections.set(a[11], freq.p && freq.d.ndim == 1 ? freq.d.shape[0] : 0);
  void* stream = stream_of(a[13]);
  if (st || PyErr_Occurred()) return status(st);
  at::Tensor new_q;
  if (q.p && !qo.p) st = make_like(THPVariable_Unpack(a[7]), dev, &new_q, &qo);
  if (st) return status(st);
  {
    const Unlocked unlocked;
    st = g_entry.paged_append(k.p, v.p, &pages.d, starts, q.p, qo.p, pos.p, freq.p, sections.n, sections.axes,
                              interleaved, stream);
  }
  if (st) return status(st);
  written(a[2], a[3], a[8]);
  return new_q.defined() ? THPVariable_Wrap(new_q) : Py_NewRef(a[8]);
  END_HANDLE_TH_ERRORS
}

// Output, workspace and launch of an attention call: `out` or a status.  A new output
// for q [B, H, D] of single tokens is [B, 1, H, D].
template <class Check, class Launch>
PyObject* attend(PyObject* out_arg, const at::Tensor& q, bool single, int64_t dev, Check check, Launch launch) {
  Arg out;
  at::Tensor made;
  int st = out.set(out_arg, dev, kWrite);
  if (!st && !out.p && single && q.dim() == 3) {
    made = fresh(q, {q.size(0), 1, q.size(1), q.size(2)}, q.scalar_type());
    st = describe(made, dev, &out.d, kWrite);
    for (int i = 1; i < 3; ++i) {
      out.d.shape[i] = out.d.shape[i + 1];
      out.d.stride[i] = out.d.stride[i + 1];
    }
    out.d.ndim = 3;
    out.p = &out.d;
  } else if (!st && !out.p) {
    st = make_like(q, dev, &made, &out);
  }
  if (st) return status(st);
  size_t bytes = 0;
  if ((st = check(out.p, &bytes))) return status(st);
  // the call's own: torch's allocator hands it on in the stream's order
  const at::Tensor ws = bytes > 0 ? fresh(q, {(int64_t)bytes}, at::kByte) : at::Tensor();
  void* const scratch = bytes > 0 ? ws.data_ptr() : nullptr;
  {
    const Unlocked unlocked;
    st = launch(out.p, scratch, bytes);
  }
  if (st) return status(st);
  written(out_arg);
  return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(out_arg);
}

// paged_attention(q, starts, k_pages, v_pages, table, lens, groups, window,
// sinks, out, stream): out, or a status
PyObject* py_paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts("paged_attention", n, 11)) return nullptr;
  if (!THPVariable_Check(a[0])) return status(RK_ERR_ARG);
  if (needs_grad(a[0], a[2], a[3], a[9])) return status(kNeedsGrad);
  const at::Tensor& t = THPVariable_Unpack(a[0]);
  const int64_t dev = t.get_device();
  Arg q;
  PagesArg pages;
  const int32_t* starts = nullptr;
  const OnDevice guard(t);
  int st = q.set(a[0], dev);
  if (!st) st = pages.set(a[2], a[3], a[4], a[5], dev);
  if (!st) st = lengths(a[1], dev, pages.requests + 1, &starts);
  const int64_t groups = PyLong_AsLongLong(a[6]), window = PyLong_AsLongLong(a[7]), sinks = PyLong_AsLongLong(a[8]);
  void* stream = stream_of(a[10]);
  if (st || PyErr_Occurred()) return status(st);
  return attend(
      a[9], t, starts == nullptr, dev,
      [&](const rk_tensor* out, size_t* bytes) {
        return g_entry.paged_check(q.p, starts, &pages.d, groups, window, sinks, out, 0, bytes);
      },
      [&](const rk_tensor* out, void* ws, size_t bytes) {
        return g_entry.paged(q.p, starts, &pages.d, groups, window, sinks, out, ws, bytes, stream);
      });
  END_HANDLE_TH_ERRORS
}

// window_attention(q, k, v, lens, groups, window, sinks, out, stream): out, or a status
PyObject* py_window_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts("window_attention", n, 9)) return nullptr;
  if (!THPVariable_Check(a[0])) return status(RK_ERR_ARG);
  if (needs_grad(a[0], a[1], a[2], a[7])) return status(kNeedsGrad);
  const at::Tensor& t = THPVariable_Unpack(a[0]);
  const int64_t dev = t.get_device();
  Arg q, k, v;
  const int32_t* lens = nullptr;
  const OnDevice guard(t);
  int st = q.set(a[0], dev);
  if (!st) st = k.set(a[1], dev);
  if (!st) st = v.set(a[2], dev);
  if (!st) st = lengths(a[3], dev, t.dim() > 0 ? t.size(0) : 0, &lens);
  const int64_t groups = PyLong_AsLongLong(a[4]), window = PyLong_AsLongLong(a[5]), sinks = PyLong_AsLongLong(a[6]);
  void* stream = stream_of(a[8]);
  if (st || PyErr_Occurred()) return status(st);
  return attend(
      a[7], t, false, dev,
      [&](const rk_tensor* out, size_t* bytes) {
        return g_entry.window_check(q.p, k.p, v.p, lens, groups, window, sinks, out, 0, bytes);
      },
      [&](const rk_tensor* out, void* ws, size_t bytes) {
        return g_entry.window(q.p, k.p, v.p, lens, groups, window, sinks, out, ws, bytes, stream);
      });
  END_HANDLE_TH_ERRORS
}

// init(the entries of `Entries` in its order): addresses
PyObject* py_init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counts("init", n, 13)) return nullptr;
  void* p[13];
  for (int i = 0; i < 13; ++i) {
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
  g_entry.rotary = reinterpret_cast<decltype(g_entry.rotary)>(p[7]);
  g_entry.paged_append = reinterpret_cast<decltype(g_entry.paged_append)>(p[8]);
  g_entry.paged_check = reinterpret_cast<decltype(g_entry.paged_check)>(p[9]);
  g_entry.paged = reinterpret_cast<decltype(g_entry.paged)>(p[10]);
  g_entry.window_check = reinterpret_cast<decltype(g_entry.window_check)>(p[11]);
  g_entry.window = reinterpret_cast<decltype(g_entry.window)>(p[12]);
  Py_RETURN_NONE;
}

#define RK_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {RK_METHOD(init),   RK_METHOD(write),  RK_METHOD(read),
                           RK_METHOD(append), RK_METHOD(decode), RK_METHOD(rotary),
                           RK_METHOD(paged_append), RK_METHOD(paged_attention), RK_METHOD(window_attention),
                           {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind(void) {
  g_codes = PyUnicode_InternFromString("codes");
  g_scales = PyUnicode_InternFromString("scales");
  g_head_dim = PyUnicode_InternFromString("head_dim");
  g_fmt = PyUnicode_InternFromString("fmt");
  PyObject* m = PyModule_Create(&g_module);
  if (m && (PyModule_AddIntConstant(m, "OTHER_DEVICE", kOtherDevice) < 0 ||
            PyModule_AddIntConstant(m, "NEEDS_GRAD", kNeedsGrad) < 0)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
