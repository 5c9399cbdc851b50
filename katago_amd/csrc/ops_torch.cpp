// ops_torch.cpp — what katago_amd/ops.py does with a call's tensors, as a Python extension of its own (katago_amd/_ops.so): checks of devices, types and
// shapes, the outputs' allocation, the call into libkatamx.so (katamx_ops.h, which checks the rest). A call on a few rows is bound by the host, where a kernel's
// launch alone is 3.3 us: rms_norm with residual and codes takes 6.3 us (11.8 with these steps in Python), linear8 4.4 (8.4), rotary 5.5 (11.0).
// The library is not linked: bind() is given its entry points' addresses, so that one build of this serves any libkatamx.so.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/katamx_ops.h"

namespace {

constexpr int64_t MX_BLOCK = 32;

// set by bind()
PyObject* streamOf = nullptr;   // device index -> address of its current stream
PyObject* errorType = nullptr;  // KatamxError(code, message)
struct {
  const char* (*lastError)(void);
  decltype(&kmx_rmsnorm) rmsnorm;
  decltype(&kmx_quantize) quantize;
  decltype(&kmx_linear8) linear8;
  decltype(&kmx_rotary) rotary;
} entry;

struct Refused {
  int code;
  std::string why;
};
[[noreturn]] void refuse(const std::string& why) { throw Refused{KMX_ERR_INVALID_ARG, why}; }
struct PythonError {};  // a Python exception is set

// Arguments; None is an undefined tensor. They are the caller's references: alive while the call is.
struct Arg {
  const char* name;
  at::Tensor t;
  bool given() const { return t.defined(); }
  const at::Tensor* operator->() const { return &t; }
};
Arg tensor(const char* name, PyObject* o) {
  if(o == Py_None) return Arg{name, at::Tensor()};
  if(!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
  return Arg{name, THPVariable_Unpack(o)};
}
// The index of the device all of them are on; gradients are refused, forward-mode tangents too (that mode is on in no_grad as well)
int onDevice(std::initializer_list<const Arg*> args) {
  int index = -1;
  const bool grad = c10::GradMode::is_enabled();
  for(const Arg* a : args)
    if(a->given() && a->t._fw_grad(0).defined())
      refuse(std::string(a->name) + " carries a forward-mode tangent and the operators compute none: unpack it first");
  for(const Arg* a : args) {
    if(!a->given()) continue;
    const c10::Device d = a->t.device();
    if(!d.is_cuda()) refuse(std::string(a->name) + " is on " + d.str() + ": the operators work on device tensors");
    if(index >= 0 && d.index() != index) refuse(std::string(a->name) + " is on device " + std::to_string((int)d.index()) + ", the others on " + std::to_string(index));
    index = d.index();
    if(a->t.is_neg()) refuse(std::string(a->name) + " is a view that is negated when it is read: call .resolve_neg() first");
    if(grad && a->t.requires_grad()) refuse(std::string(a->name) + " requires a gradient and the operators compute none: call them under torch.no_grad()");
  }
  return index;
}

std::string shapeOf(at::IntArrayRef s) {
  std::string r = "(";
  for(size_t i = 0; i < s.size(); i++) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}
// A tensor's rows, whose leading dimensions step evenly: [...][channels] with one stride
struct Rows {
  int64_t n, channels, stride;
};
Rows rowsOf(const Arg& a, int64_t channels = -1) {
  const int64_t dims = a->dim();
  if(dims < 1) refuse(std::string(a.name) + " must have a dimension of channels");
  const at::IntArrayRef shape = a->sizes(), strides = a->strides();
  const int64_t c = shape[dims - 1];
  if(channels >= 0 && c != channels) refuse(std::string(a.name) + " has " + std::to_string(c) + " channels, not " + std::to_string(channels));
  if(c > 1 && strides[dims - 1] != 1) refuse(std::string(a.name) + ": channels must be contiguous");
  for(int64_t d = 0; d + 1 < dims; d++)
    if(shape[d] == 0) return Rows{0, c, c};
  int64_t n = 1, stride = c;
  for(int64_t d = dims - 2; d >= 0; d--) {
    if(shape[d] == 1) continue;
    if(n == 1) stride = strides[d];
    else if(strides[d] != stride * n) refuse(std::string(a.name) + ": the rows' strides do not collapse to one");
    n *= shape[d];
  }
  return Rows{n, c, stride};
}
const float* vectorOf(const Arg& a, int64_t length) {
  if(!a.given()) return nullptr;
  if(a->scalar_type() != at::kFloat || a->numel() != length || !a->is_contiguous())
    refuse(std::string(a.name) + " must be " + std::to_string(length) + " contiguous float32 values");
  return (const float*)a->data_ptr();
}
int typeOf(const char* name, at::ScalarType t) {
  if(t == at::kHalf) return KMX_PREC_FP16;
  if(t == at::kBFloat16) return KMX_PREC_BF16;
  if(t == at::kFloat) return KMX_PREC_FP32;
  refuse(std::string(name) + " is " + c10::toString(t) + ", not float16, bfloat16 or float32");
}
void sameAs(const Arg& out, const at::Tensor& like) {
  if(out->scalar_type() != like.scalar_type() || out->sizes() != like.sizes()) refuse(std::string(out.name) + " must be of the input's type and of shape " + shapeOf(like.sizes()));
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if(v == -1.0 && PyErr_Occurred()) throw PythonError();
  return v;
}
long integer(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if(v == -1 && PyErr_Occurred()) throw PythonError();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if(v < 0) throw PythonError();
  return v == 1;
}
void* currentStream(int device) {
  PyObject* const index = PyLong_FromLong(device);
  if(index == nullptr) throw PythonError();
  PyObject* const s = PyObject_CallOneArg(streamOf, index);
  Py_DECREF(index);
  if(s == nullptr) throw PythonError();
  void* const p = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  if(p == nullptr && PyErr_Occurred()) throw PythonError();
  return p;
}
// Other threads of the program run while this lives
class WithoutGil {
 public:
  WithoutGil() : state_(PyEval_SaveThread()) {}
  ~WithoutGil() { PyEval_RestoreThread(state_); }

 private:
  PyThreadState* state_;
};
// A tensor of the caller's has been written: autograd, which may keep it for a backward pass, is told as torch's own in-place operations tell it. (Inference
// tensors have no version.)
void written(const Arg& a) {
  if(a.given() && !a.t.is_inference()) a.t.unsafeGetTensorImpl()->bump_version();
}
// (the message is of this thread's last call)
void check(int rc) {
  if(rc != KMX_OK) throw Refused{rc, entry.lastError()};
}

at::Tensor newLike(const at::Tensor& x, at::IntArrayRef shape, at::ScalarType t) { return at::empty(shape, x.options().dtype(t)); }
void codesFor(const at::Tensor& x, int kind, at::Tensor* codes, at::Tensor* scales) {
  const at::IntArrayRef shape = x.sizes();
  c10::SmallVector<int64_t, 6> lead(shape.begin(), shape.end() - 1);
  if(kind == KMX_SCALES_ROW) *scales = newLike(x, lead, at::kFloat);
  else {
    lead.push_back(shape.back() / MX_BLOCK);
    *scales = newLike(x, lead, at::kFloat8_e8m0fnu);
  }
  *codes = newLike(x, shape, at::kFloat8_e4m3fn);
}
void checkKind(int kind, int64_t channels) {
  if(kind == KMX_SCALES_MX && channels % MX_BLOCK != 0)
    refuse("scales for 32 channels each need a multiple of 32 channels, not " + std::to_string(channels));
}
void count(Py_ssize_t have, Py_ssize_t want) {
  if(have == want) return;
  PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, have);
  throw PythonError();
}
PyObject* wrapped(const at::Tensor& t) { return THPVariable_Wrap(t); }  // (undefined: None)

// rms_norm(x, weight, eps, beta, residual, mask, kind of scales, want_y, sum_out, y_out) -> (sum, y, codes, scales)
PyObject* rmsNorm(PyObject* const* args, Py_ssize_t n) {
  count(n, 10);
  const Arg x = tensor("x", args[0]), weight = tensor("weight", args[1]), beta = tensor("beta", args[3]), residual = tensor("residual", args[4]);
  const Arg mask = tensor("mask", args[5]), sumOut = tensor("sum_out", args[8]), yOut = tensor("y_out", args[9]);
  const int kind = (int)integer(args[6]);
  const bool wantY = args[7] == Py_None ? kind == KMX_SCALES_NONE || yOut.given() : truth(args[7]);
  kmx_rmsnorm_args a = {};
  a.epsilon = (float)number(args[2]);
  if(!x.given()) refuse("x must be a tensor");
  const int device = onDevice({&x, &weight, &beta, &residual, &mask, &sumOut, &yOut});
  a.type = typeOf("x", x->scalar_type());
  a.scale_kind = kind;
  if((yOut.given() && !wantY) || (sumOut.given() && !residual.given())) refuse("an output is given that is not computed");
  const Rows r = rowsOf(x);
  if(r.channels > 0x7fffffff) refuse("x has too many channels");
  a.rows = r.n;
  a.channels = (int32_t)r.channels;
  a.x = x->data_ptr();
  a.x_stride = r.stride;
  a.weight = vectorOf(weight, r.channels);
  a.beta = vectorOf(beta, r.channels);
  a.mask = vectorOf(mask, r.n);
  if(residual.given()) {
    if(residual->scalar_type() != x->scalar_type() || residual->sizes() != x->sizes()) refuse("residual must be of x's type and shape");
    a.residual = residual->data_ptr();
    a.residual_stride = rowsOf(residual).stride;
    if(sumOut.given()) sameAs(sumOut, x.t);
  }
  if(yOut.given()) sameAs(yOut, x.t);
  checkKind(kind, r.channels);
  void* const stream = currentStream(device);
  Arg sum = sumOut, y = yOut;
  at::Tensor codes, scales;
  {
    const WithoutGil others;
    if(residual.given()) {
      if(!sum.given()) sum.t = at::empty_like(x.t);
      a.sum = sum->data_ptr();
      a.sum_stride = rowsOf(sum).stride;
    }
    if(wantY) {
      if(!y.given()) y.t = at::empty_like(x.t);
      a.y = y->data_ptr();
      a.y_stride = rowsOf(y).stride;
    }
    if(kind != KMX_SCALES_NONE) {
      codesFor(x.t, kind, &codes, &scales);
      a.codes = codes.data_ptr();
      a.scales = scales.data_ptr();
      a.codes_stride = r.channels;
    }
    if(r.n > 0) check(entry.rmsnorm(device, stream, &a));
    written(sumOut);
    written(yOut);
  }
  return Py_BuildValue("(NNNN)", wrapped(sum.t), wrapped(y.t), wrapped(codes), wrapped(scales));
}

// quantize(x, kind of scales) -> (codes, scales)
PyObject* quantize(PyObject* const* args, Py_ssize_t n) {
  count(n, 2);
  const Arg x = tensor("x", args[0]);
  if(!x.given()) refuse("x must be a tensor");
  const int kind = (int)integer(args[1]);
  const int device = onDevice({&x}), type = typeOf("x", x->scalar_type());
  const Rows r = rowsOf(x);
  if(r.channels > 0x7fffffff) refuse("x has too many channels");
  checkKind(kind, r.channels);
  void* const stream = currentStream(device);
  at::Tensor codes, scales;
  {
    const WithoutGil others;
    codesFor(x.t, kind, &codes, &scales);
    if(r.n > 0) check(entry.quantize(device, stream, type, kind, r.n, (int)r.channels, x->data_ptr(), r.stride, codes.data_ptr(), r.channels, scales.data_ptr()));
  }
  return Py_BuildValue("(NN)", wrapped(codes), wrapped(scales));
}

int kindOf(const Arg& codes, const Arg& scales, int64_t rows, int64_t k) {
  if(codes->scalar_type() != at::kFloat8_e4m3fn) refuse(std::string(codes.name) + " must be float8_e4m3fn");
  if(!scales->is_contiguous()) refuse(std::string(codes.name) + "'s scales must be contiguous");
  if(scales->scalar_type() == at::kFloat && scales->numel() == rows) return KMX_SCALES_ROW;
  if(scales->scalar_type() == at::kFloat8_e8m0fnu && k % MX_BLOCK == 0 && scales->numel() == rows * (k / MX_BLOCK)) return KMX_SCALES_MX;
  refuse(std::string(codes.name) + "'s scales must be float32 of one a row or float8_e8m0fnu of one for 32 channels");
}

// linear8(codes, scales, weight_codes, weight_scales, bias, out_dtype, out) -> out
PyObject* linear8(PyObject* const* args, Py_ssize_t n) {
  count(n, 7);
  const Arg codes = tensor("codes", args[0]), scales = tensor("scales", args[1]), wCodes = tensor("weight_codes", args[2]), wScales = tensor("weight_scales", args[3]);
  const Arg bias = tensor("bias", args[4]), given = tensor("out", args[6]);
  for(const Arg* a : {&codes, &scales, &wCodes, &wScales})
    if(!a->given()) refuse(std::string(a->name) + " must be a tensor");
  const int device = onDevice({&codes, &scales, &wCodes, &wScales, &bias, &given});
  if(wCodes->dim() != 2) refuse("weight_codes must be [n, k]");
  const Rows w = rowsOf(wCodes), r = rowsOf(codes, w.channels);
  const int64_t outs = wCodes->size(0);
  if(outs > 0x7fffffff || r.channels > 0x7fffffff) refuse("n and k must be below 2^23");
  kmx_linear8_args a = {};
  a.scale_kind = kindOf(codes, scales, r.n, r.channels);
  if(kindOf(wCodes, wScales, outs, r.channels) != a.scale_kind) refuse("the scales of codes and weight_codes are of different kinds");
  c10::SmallVector<int64_t, 6> shape(codes->sizes().begin(), codes->sizes().end() - 1);
  shape.push_back(outs);
  at::ScalarType type;
  if(given.given()) {
    type = given->scalar_type();
    if(given->sizes() != at::IntArrayRef(shape)) refuse("out must be of shape " + shapeOf(shape));
  }
  else {
    if(!THPDtype_Check(args[5])) refuse("out_dtype must be a dtype");
    type = ((THPDtype*)args[5])->scalar_type;
  }
  a.out_type = typeOf(given.given() ? "out" : "out_dtype", type);
  a.rows = r.n;
  a.n = (int32_t)outs;
  a.k = (int32_t)r.channels;
  a.a = codes->data_ptr();
  a.a_scales = scales->data_ptr();
  a.w = wCodes->data_ptr();
  a.w_scales = wScales->data_ptr();
  a.bias = vectorOf(bias, outs);
  a.a_stride = r.stride;
  a.w_stride = w.stride;
  void* const stream = currentStream(device);
  Arg out = given;
  {
    const WithoutGil others;
    if(!out.given()) out.t = newLike(codes.t, shape, type);
    a.out = out->data_ptr();
    a.out_stride = rowsOf(out).stride;
    if(r.n > 0) check(entry.linear8(device, stream, &a));
    written(given);
  }
  return wrapped(out.t);
}

// rotary(q, k, positions, frequencies, half, magnitude, inverse, q_out, k_out) -> (q_out, k_out)
PyObject* rotary(PyObject* const* args, Py_ssize_t n) {
  count(n, 9);
  const Arg q = tensor("q", args[0]), k = tensor("k", args[1]), positions = tensor("positions", args[2]), freqs = tensor("frequencies", args[3]);
  const Arg qOut = tensor("q_out", args[7]), kOut = tensor("k_out", args[8]);
  for(const Arg* a : {&q, &positions, &freqs})
    if(!a->given()) refuse(std::string(a->name) + " must be a tensor");
  kmx_rotary_args a = {};
  a.half = truth(args[4]);
  a.magnitude = (float)number(args[5]);
  a.inverse = truth(args[6]);
  const int device = onDevice({&q, &k, &positions, &freqs, &qOut, &kOut});
  a.type = typeOf("q", q->scalar_type());
  const int64_t lead = q->dim() - 2;
  if(lead != 1 && lead != 2) refuse("q must be [batch, seq, heads, head_dim] or [tokens, heads, head_dim]");
  a.batch = lead == 2 ? q->size(0) : 1;
  a.seq = q->size(lead - 1);
  const int64_t heads = q->size(lead), dim = q->size(lead + 1), kHeads = k.given() && k->dim() == lead + 2 ? k->size(lead) : 0;
  if(freqs->scalar_type() != at::kDouble || !freqs->is_contiguous() || freqs->dim() < 1 || freqs->dim() > 3)
    refuse("frequencies must be contiguous float64 [pairs], [axes, pairs] or [freq_heads, axes, pairs]");
  const int64_t fd = freqs->dim(), pairs = freqs->size(fd - 1), axes = fd >= 2 ? freqs->size(fd - 2) : 1, freqHeads = fd == 3 ? freqs->size(0) : 1;
  for(int64_t v : {heads, dim, kHeads, pairs, axes, freqHeads})
    if(v > 0x7fffffff) refuse("a dimension is out of range");
  if(positions->scalar_type() != at::kInt && positions->scalar_type() != at::kLong) refuse("positions must be int32 or int64");
  // [seq] or [batch, seq], and a last dimension of axes, which may be left out where there is one
  at::IntArrayRef ps = positions->sizes(), pst = positions->strides();
  auto forTokens = [&](at::IntArrayRef s) { return (s.size() == 1 && s[0] == a.seq) || (lead == 2 && s.size() == 2 && s[0] == a.batch && s[1] == a.seq); };
  if((axes > 1 || !forTokens(ps)) && !ps.empty() && ps.back() == axes) {
    a.pos_axis_stride = pst.back();
    ps = ps.slice(0, ps.size() - 1);
    pst = pst.slice(0, ps.size());
  }
  else if(axes > 1) refuse("positions must have a last dimension of " + std::to_string(axes) + " axes");
  if(!forTokens(ps)) refuse("positions must be one for each token: " + shapeOf(positions->sizes()) + " for q's " + shapeOf(q->sizes()));
  a.pos_batch_stride = ps.size() == 2 ? pst[0] : 0;
  a.pos_seq_stride = pst.back();
  if(k.given()) {
    if(k->scalar_type() != q->scalar_type() || k->dim() != lead + 2 || k->size(0) != q->size(0) || k->size(lead - 1) != a.seq || k->size(lead + 1) != dim)
      refuse("k must have q's type, tokens and head_dim");
  }
  else if(kOut.given()) refuse("an output is given that is not computed");
  if(heads == 0 || (k.given() && kHeads == 0)) refuse("q and k must have heads");
  if(qOut.given()) sameAs(qOut, q.t);
  if(kOut.given()) sameAs(kOut, k.t);
  a.q_heads = (int32_t)heads;
  a.k_heads = (int32_t)kHeads;
  a.head_dim = (int32_t)dim;
  a.pairs = (int32_t)pairs;
  a.axes = (int32_t)axes;
  a.freq_heads = (int32_t)freqHeads;
  a.frequencies = (const double*)freqs->data_ptr();
  a.positions = positions->data_ptr();
  a.positions_are_64bit = positions->scalar_type() == at::kLong;
  auto stridesOf = [&](const Arg& t, int64_t (&s)[3]) {
    const at::IntArrayRef st = t->strides();
    if(dim > 1 && st[lead + 1] != 1) refuse(std::string(t.name) + ": channels must be contiguous");
    s[0] = lead == 2 ? st[0] : 0;
    s[1] = st[lead - 1];
    s[2] = st[lead];
  };
  auto side = [&](const Arg& in, const Arg& out) {
    int64_t i[3], o[3];
    stridesOf(in, i);
    stridesOf(out, o);
    return kmx_rotary_tensor{in->data_ptr(), out->data_ptr(), i[0], i[1], i[2], o[0], o[1], o[2]};
  };
  void* const stream = currentStream(device);
  Arg qo = qOut, ko = kOut;
  {
    const WithoutGil others;
    if(!qo.given()) qo.t = at::empty_like(q.t);
    a.q = side(q, qo);
    if(k.given()) {
      if(!ko.given()) ko.t = at::empty_like(k.t);
      a.k = side(k, ko);
    }
    if(a.batch > 0 && a.seq > 0) check(entry.rotary(device, stream, &a));
    written(qOut);
    written(kOut);
  }
  return Py_BuildValue("(NN)", wrapped(qo.t), wrapped(ko.t));
}

// bind(stream of a device, KatamxError, addresses of kmx_last_error, kmx_rmsnorm, kmx_quantize, kmx_linear8, kmx_rotary)
PyObject* bind(PyObject* const* args, Py_ssize_t n) {
  count(n, 7);
  void* at[5];
  for(int i = 0; i < 5; i++) {
    at[i] = PyLong_AsVoidPtr(args[2 + i]);
    if(PyErr_Occurred()) throw PythonError();
    if(at[i] == nullptr) refuse("an entry point is missing");
  }
  entry = {(decltype(entry.lastError))at[0], (decltype(entry.rmsnorm))at[1], (decltype(entry.quantize))at[2], (decltype(entry.linear8))at[3],
           (decltype(entry.rotary))at[4]};
  Py_INCREF(args[0]);
  Py_INCREF(args[1]);
  Py_XDECREF(streamOf);
  Py_XDECREF(errorType);
  streamOf = args[0];
  errorType = args[1];
  Py_RETURN_NONE;
}

// Nothing unwinds into Python: refusals are KatamxError, torch's own errors (out of memory) what they are in Python
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    return F(args, n);
  }
  catch(const Refused& r) {
    PyObject* const e = PyObject_CallFunction(errorType != nullptr ? errorType : PyExc_RuntimeError, "is", r.code, r.why.c_str());
    if(e != nullptr) {
      PyErr_SetObject((PyObject*)Py_TYPE(e), e);
      Py_DECREF(e);
    }
    return nullptr;
  }
  catch(const PythonError&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return PyMethodDef{name, (PyCFunction)(void (*)(void))guarded<F>, METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<rmsNorm>("rms_norm"), method<quantize>("quantize"), method<linear8>("linear8"), method<rotary>("rotary"), method<bind>("bind"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops(void) { return PyModule_Create(&module); }
