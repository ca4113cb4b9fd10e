// The decoder's attention and norm, forward and backward, as calls from Python, for the calls that need
// nothing but launches: every tensor on the current CUDA device, in place as the kernels read it.  Checks,
// results, workspace and launch are one call here; anything else (another device, a layout that needs
// a copy, an argument that is to be refused) returns None, and attention.py and norm.py take the call
// from its start, with the copies and the messages.
//
// A small call is bound by the host: forward and backward norm of 900 x 256 take 7.0 us in a CUDA graph, 34 us when
// called in a loop from Python and 11.7 from here; attention of 6 x 13 queries over 600 keys 16.3 us from Python and
// 9.4 from here, which is the GPU's time.
//
// The C ABI's functions come as addresses (init), so that the library that lib() loaded is the one called.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>

#include "s4d_decoder.h"

namespace {

decltype(&s4d_norm_forward) norm_forward_fn;
decltype(&s4d_norm_backward_workspace_bytes) norm_backward_ws_fn;
decltype(&s4d_norm_backward) norm_backward_fn;
decltype(&s4d_attention_forward_workspace_bytes) attention_forward_ws_fn;
decltype(&s4d_attention_forward) attention_forward_fn;
decltype(&s4d_attention_backward_workspace_bytes) attention_backward_ws_fn;
decltype(&s4d_attention_backward) attention_backward_fn;

// The arguments of one call.  ok() is false from the first that does not fit on.
class Args {
 public:
  Args(PyObject* const* args, Py_ssize_t n, Py_ssize_t want) : args_(args), ok_(n == want) {}
  bool ok() const { return ok_; }
  bool need(bool b) { return ok_ = ok_ && b; }
  int device() const { return device_; }
  cudaStream_t stream() const { return c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(device_)).stream(); }

  // A strided tensor on the current device, the same for all of a call; null for None.
  const at::Tensor* tensor(int i, bool optional = false) {
    if (!ok_ || (optional && args_[i] == Py_None)) return nullptr;
    if (!need(THPVariable_Check(args_[i]))) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(args_[i]);
    if (!need(t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch() &&
              !t.is_neg() && !t.is_conj()))
      return nullptr;
    if (device_ < 0) {
      device_ = t.get_device();
      need(device_ == c10::cuda::current_device());
    }
    need(t.get_device() == device_);
    return ok_ ? &t : nullptr;
  }
  // ... contiguous, of this type and shape
  const at::Tensor* tensor(int i, at::ScalarType type, at::IntArrayRef shape, bool optional = false) {
    const at::Tensor* t = tensor(i, optional);
    if (t != nullptr && !need(t->scalar_type() == type && t->sizes() == shape && t->is_contiguous())) return nullptr;
    return t;
  }
  float number(int i) {
    if (!ok_) return 0.0f;
    const double v = PyFloat_Check(args_[i]) || PyLong_Check(args_[i]) ? PyFloat_AsDouble(args_[i]) : NAN;
    if (PyErr_Occurred()) PyErr_Clear();
    need(std::isfinite(v) && (v == 0.0 || float(v) != 0.0f));  // what fp32 makes another number of
    return float(v);
  }
  bool truth(int i) {
    if (!ok_) return false;
    const int v = PyObject_IsTrue(args_[i]);
    if (v < 0) PyErr_Clear();
    need(v >= 0);
    return v == 1;
  }
  bool none(int i) const { return args_[i] == Py_None; }

 private:
  PyObject* const* args_;
  bool ok_;
  int device_ = -1;
};

int dtype_of(at::ScalarType t) {
  return t == at::kFloat ? int(S4D_DTYPE_F32) : t == at::kBFloat16 ? int(S4D_DTYPE_BF16) : t == at::kHalf ? int(S4D_DTYPE_F16) : -1;
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, int device) {
  return at::detail::empty_cuda(shape, type, at::Device(at::kCUDA, c10::DeviceIndex(device)), std::nullopt);
}

void* address(const at::Tensor* t) { return t == nullptr ? nullptr : t->data_ptr(); }

PyObject* wrap(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

PyObject* pack(std::initializer_list<at::Tensor> list) {
  PyObject* tuple = PyTuple_New(Py_ssize_t(list.size()));
  if (tuple == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : list) {
    PyObject* o = wrap(t);
    if (o == nullptr) {
      Py_DECREF(tuple);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple, i++, o);
  }
  return tuple;
}

// A norm's weight or bias: [width] in f32 or the rows' type, the same for both.
bool param(Args& a, const at::Tensor* t, at::ScalarType rows, int64_t width, at::ScalarType* type) {
  if (t == nullptr) return a.ok();
  const at::ScalarType own = t->scalar_type();
  a.need(t->dim() == 1 && t->size(0) == width && t->is_contiguous() && (own == at::kFloat || own == rows) &&
         (*type == at::ScalarType::Undefined || *type == own));
  *type = own;
  return a.ok();
}

// (x, weight or None, bias or None, eps) -> (y, mean, rstd) or None
PyObject* norm_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(args, n, 4);
  const at::Tensor* x = a.tensor(0);
  const at::Tensor *w = a.tensor(1, true), *b = a.tensor(2, true);
  const float eps = a.number(3);
  if (!a.ok() || x->dim() < 1 || !x->is_contiguous() || x->size(-1) < 1 || dtype_of(x->scalar_type()) < 0) Py_RETURN_NONE;
  const int64_t width = x->size(-1), rows = x->numel() / width;
  at::ScalarType type = at::ScalarType::Undefined;
  if (!param(a, w, x->scalar_type(), width, &type) || !param(a, b, x->scalar_type(), width, &type)) Py_RETURN_NONE;
  const auto stats = x->sizes().slice(0, x->dim() - 1);
  at::Tensor y = empty(x->sizes(), x->scalar_type(), a.device());
  at::Tensor mean = empty(stats, at::kFloat, a.device()), rstd = empty(stats, at::kFloat, a.device());
  if (norm_forward_fn(x->data_ptr(), width, dtype_of(x->scalar_type()), address(w), address(b),
                      type == at::ScalarType::Undefined ? int(S4D_DTYPE_F32) : dtype_of(type), y.data_ptr(), width,
                      mean.data_ptr<float>(), rstd.data_ptr<float>(), rows, width, eps, a.stream()) != S4D_OK)
    Py_RETURN_NONE;
  return pack({y, mean, rstd});
  END_HANDLE_TH_ERRORS
}

// (dout, x, weight or None, mean, rstd, need_dx, need_dweight, need_dbias) -> (dx, dweight, dbias) or None
PyObject* norm_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(args, n, 8);
  const at::Tensor* x = a.tensor(1);
  if (!a.ok() || x->dim() < 1 || !x->is_contiguous() || x->size(-1) < 1 || dtype_of(x->scalar_type()) < 0) Py_RETURN_NONE;
  const int64_t width = x->size(-1), rows = x->numel() / width;
  const auto stats = x->sizes().slice(0, x->dim() - 1);
  const at::Tensor *dy = a.tensor(0, x->scalar_type(), x->sizes()), *w = a.tensor(2, true);
  const at::Tensor *mean = a.tensor(3, at::kFloat, stats), *rstd = a.tensor(4, at::kFloat, stats);
  at::ScalarType type = at::ScalarType::Undefined;
  if (!param(a, w, x->scalar_type(), width, &type)) Py_RETURN_NONE;
  if (type == at::ScalarType::Undefined) type = at::kFloat;
  at::Tensor dx, dw, db, ws;
  const bool need_dx = a.truth(5), need_dw = a.truth(6), need_db = a.truth(7);
  if (!a.ok()) Py_RETURN_NONE;
  if (need_dx) dx = empty(x->sizes(), x->scalar_type(), a.device());
  if (need_dw) dw = empty({width}, type, a.device());
  if (need_db) db = empty({width}, type, a.device());
  const size_t need = dw.defined() || db.defined() ? norm_backward_ws_fn(rows, width) : 0;
  if (need > 0) ws = empty({int64_t(need / 4)}, at::kFloat, a.device());
  auto at_of = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  if (norm_backward_fn(dy->data_ptr(), width, x->data_ptr(), width, dtype_of(x->scalar_type()), address(w), dtype_of(type),
                       mean->data_ptr<float>(), rstd->data_ptr<float>(), at_of(dx), width, at_of(dw), at_of(db), rows,
                       width, at_of(ws), need, a.stream()) != S4D_OK)
    Py_RETURN_NONE;
  return pack({dx, dw, db});
  END_HANDLE_TH_ERRORS
}

// q, k or v as the kernels read it: unit stride along dim, the others positive multiples of 8.
bool operand(Args& a, const at::Tensor* t, int64_t* stride) {
  if (!a.need(t->stride(3) == 1 && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0)) return false;
  for (int i = 0; i < 3; ++i) {
    stride[i] = t->stride(i);
    a.need(t->size(i) <= 1 || (stride[i] > 0 && stride[i] % 8 == 0));
  }
  return a.ok();
}

// q, k, v, scale or None, softcap, slopes, q_pos, k_pos, q_segment, k_segment and k_len (the last six or None),
// from argument `at` on.
bool attention_args(Args& a, int at, s4d_attention_args& c) {
  const at::Tensor *q = a.tensor(at), *k = a.tensor(at + 1), *v = a.tensor(at + 2);
  if (!a.ok() || q->dim() != 4 || k->dim() != 4) return false;
  const at::ScalarType type = q->scalar_type();
  c.batch = q->size(0), c.queries = q->size(1), c.heads = q->size(2), c.dim = q->size(3);
  c.keys = k->size(1), c.kv_heads = k->size(2);
  a.need((type == at::kBFloat16 || type == at::kHalf) && k->scalar_type() == type && v->scalar_type() == type &&
         k->size(0) == c.batch && k->size(3) == c.dim && v->sizes() == k->sizes());
  if (!a.ok() || !operand(a, q, c.q_stride) || !operand(a, k, c.k_stride) || !operand(a, v, c.v_stride)) return false;
  c.q = q->data_ptr(), c.k = k->data_ptr(), c.v = v->data_ptr();
  c.dtype = dtype_of(type);
  c.scale = a.none(at + 3) ? float(std::pow(double(c.dim), -0.5)) : a.number(at + 3);
  c.softcap = a.number(at + 4);
  const at::Tensor* slopes = a.tensor(at + 5, true);
  if (slopes != nullptr) {
    const at::Tensor* qp = a.tensor(at + 6);
    if (!a.need(slopes->scalar_type() == at::kFloat && qp != nullptr && qp->dim() == 3)) return false;
    c.pos_dim = qp->size(2);
    qp = a.tensor(at + 6, at::kFloat, {c.batch, c.queries, c.pos_dim});
    const at::Tensor* kp = a.tensor(at + 7, at::kFloat, {c.batch, c.keys, c.pos_dim});
    a.need(c.pos_dim == 1 || c.pos_dim == 2);
    if (slopes->dim() == 1)
      a.need(slopes->size(0) == c.heads), c.slope_stride[2] = slopes->stride(0);
    else if (a.need(slopes->sizes() == at::IntArrayRef({c.batch, c.queries, c.heads})))
      for (int i = 0; i < 3; ++i) c.slope_stride[i] = slopes->stride(i);
    if (!a.ok()) return false;
    c.slopes = slopes->data_ptr<float>(), c.q_pos = qp->data_ptr<float>(), c.k_pos = kp->data_ptr<float>();
    c.dslopes_per_row = slopes->dim() == 3;
  } else if (!a.need(a.none(at + 6) && a.none(at + 7))) {
    return false;
  }
  a.need(a.none(at + 8) == a.none(at + 9));
  c.q_segment = static_cast<const int32_t*>(address(a.tensor(at + 8, at::kInt, {c.batch, c.queries}, true)));
  c.k_segment = static_cast<const int32_t*>(address(a.tensor(at + 9, at::kInt, {c.batch, c.keys}, true)));
  c.k_len = static_cast<const int32_t*>(address(a.tensor(at + 10, at::kInt, {c.batch}, true)));
  return a.ok();
}

// (the eleven arguments above) -> (out, lse) or None
PyObject* attention_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(args, n, 11);
  s4d_attention_args c = {};
  if (!attention_args(a, 0, c)) Py_RETURN_NONE;
  const at::Tensor& q = THPVariable_Unpack(args[0]);
  at::Tensor out = empty(q.sizes(), q.scalar_type(), a.device()), ws;
  at::Tensor lse = empty({c.batch, c.heads, c.queries}, at::kFloat, a.device());
  c.out = out.data_ptr();
  c.lse = lse.data_ptr<float>();
  c.workspace_bytes = attention_forward_ws_fn(&c);
  if (c.workspace_bytes > 0) {
    ws = empty({int64_t(c.workspace_bytes / 4)}, at::kFloat, a.device());
    c.workspace = ws.data_ptr();
  }
  if (attention_forward_fn(&c, a.stream()) != S4D_OK) Py_RETURN_NONE;
  return pack({out, lse});
  END_HANDLE_TH_ERRORS
}

// (dout, q, k, v, out, lse, the other eight of the eleven, need_dkv, need_dslopes) -> (dq, dk, dv, dslopes) or
// None
PyObject* attention_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 16) Py_RETURN_NONE;
  // in attention_args' order: q, k, v and the rest; then dout, out, lse and what is needed
  PyObject* const order[16] = {args[1],  args[2],  args[3],  args[6], args[7], args[8], args[9],  args[10],
                               args[11], args[12], args[13], args[0], args[4], args[5], args[14], args[15]};
  Args a(order, 16, 16);
  s4d_attention_args c = {};
  if (!attention_args(a, 0, c) || c.dtype != S4D_DTYPE_BF16 || c.batch == 0) Py_RETURN_NONE;
  const at::Tensor &q = THPVariable_Unpack(args[1]), &k = THPVariable_Unpack(args[2]);
  const at::Tensor* dout = a.tensor(11);
  if (!a.ok() || dout->scalar_type() != at::kBFloat16 || dout->sizes() != q.sizes() || !operand(a, dout, c.dout_stride))
    Py_RETURN_NONE;
  const at::Tensor *out = a.tensor(12, at::kBFloat16, q.sizes()), *lse = a.tensor(13, at::kFloat, {c.batch, c.heads, c.queries});
  const bool need_dkv = a.truth(14), need_dslopes = a.truth(15);
  if (!a.ok()) Py_RETURN_NONE;
  c.dout = dout->data_ptr(), c.out = out->data_ptr(), c.lse = lse->data_ptr<float>();
  at::Tensor dq = empty(q.sizes(), at::kBFloat16, a.device()), dk, dv, ds, ws;
  c.dq = dq.data_ptr();
  if (need_dkv) {
    dk = empty(k.sizes(), at::kBFloat16, a.device()), dv = empty(k.sizes(), at::kBFloat16, a.device());
    c.dk = dk.data_ptr(), c.dv = dv.data_ptr();
  }
  if (c.slopes != nullptr && need_dslopes) {
    ds = empty(THPVariable_Unpack(args[8]).sizes(), at::kFloat, a.device());
    c.dslopes = ds.data_ptr<float>();
  }
  c.workspace_bytes = attention_backward_ws_fn(&c);
  if (c.workspace_bytes > 0) {
    ws = empty({int64_t(c.workspace_bytes / 4)}, at::kFloat, a.device());
    c.workspace = ws.data_ptr();
  }
  if (attention_backward_fn(&c, a.stream()) != S4D_OK) Py_RETURN_NONE;
  return pack({dq, dk, dv, ds});
  END_HANDLE_TH_ERRORS
}

// (addresses of the seven functions above) -> None
PyObject* init(PyObject*, PyObject* args) {
  unsigned long long at[7];
  if (!PyArg_ParseTuple(args, "KKKKKKK", &at[0], &at[1], &at[2], &at[3], &at[4], &at[5], &at[6])) return nullptr;
  norm_forward_fn = reinterpret_cast<decltype(norm_forward_fn)>(at[0]);
  norm_backward_ws_fn = reinterpret_cast<decltype(norm_backward_ws_fn)>(at[1]);
  norm_backward_fn = reinterpret_cast<decltype(norm_backward_fn)>(at[2]);
  attention_forward_ws_fn = reinterpret_cast<decltype(attention_forward_ws_fn)>(at[3]);
  attention_forward_fn = reinterpret_cast<decltype(attention_forward_fn)>(at[4]);
  attention_backward_ws_fn = reinterpret_cast<decltype(attention_backward_ws_fn)>(at[5]);
  attention_backward_fn = reinterpret_cast<decltype(attention_backward_fn)>(at[6]);
  Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {
    {"init", init, METH_VARARGS, nullptr},
    {"norm_forward", fast(norm_forward), METH_FASTCALL, nullptr},
    {"norm_backward", fast(norm_backward), METH_FASTCALL, nullptr},
    {"attention_forward", fast(attention_forward), METH_FASTCALL, nullptr},
    {"attention_backward", fast(attention_backward), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "s4d_decoder_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_s4d_decoder_calls() { return PyModule_Create(&module); }
