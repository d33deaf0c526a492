// kcg_torch.cc — the operators of the 8-bit path on torch tensors: checks of the arguments, outputs, the call.
// A small call is over in 3 to 5 us on the GPU, and the runtime's launch takes the host 3.1; with the same steps in Python a
// call took the host 7.4 to 8.5 us (an output 1.3, a checked operand 0.5), so a decoded token waited for it.  Here a whole call
// takes 3.1 to 3.5 us with the caller's outputs, 3.8 to 4.7 where one or two are made (moe_layer, of two or three launches: 8.6, 11.3).
//
// The module links neither the library nor a HIP runtime: bind() gives it the addresses of the C entry points
// (include/kcg_ops.h), so that both bindings run the one library that the process has loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty_strided.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/kcg_gemm.h"
#include "../../include/kcg_ops.h"

namespace {

using at::ScalarType;

int (*norm_entry)(const kcg_rmsnorm_quant_args*, int, uint64_t);
int (*swiglu_entry)(const kcg_swiglu_quant_args*, int, uint64_t);
int (*matmul_entry)(const kcg_matmul_fp8_args*, int, uint64_t);
int (*moe_entry)(const kcg_moe_layer_args*, int, uint64_t);
int64_t (*moe_workspace)(int64_t, int64_t, int64_t, int64_t, int64_t);
PyObject* stream_of;       // device index -> raw handle of torch's current stream
PyObject* check_status;    // raises what a negative status stands for

int64_t groups(int64_t n) { return (n + 127) / 128; }
int64_t address(const at::Tensor& t) { return (int64_t)(uintptr_t)t.data_ptr(); }

int64_t code_of(ScalarType t) {
  switch (t) {
    case ScalarType::Float: return KCG_DT_FLOAT32;
    case ScalarType::Half: return KCG_DT_FLOAT16;
    case ScalarType::BFloat16: return KCG_DT_BFLOAT16;
    default: return 0;     // no type of an input or a product here
  }
}

const at::Tensor& tensor(const char* name, PyObject* o) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

// The operators have no backward pass.  Results cut off from an argument that wants a gradient would train wrongly without a word,
// so such a call is refused, as torch refuses its own functions with an out argument.
void no_gradient(PyObject* const* a, Py_ssize_t n) {
  if (!c10::GradMode::is_enabled()) return;
  for (Py_ssize_t i = 0; i < n; ++i)
    TORCH_CHECK(!THPVariable_Check(a[i]) || !THPVariable_Unpack(a[i]).requires_grad(),
                "the operators of the 8-bit path have no gradient, and a tensor of the call requires one (shape ", THPVariable_Unpack(a[i]).sizes(),
                "): call under torch.no_grad(), or pass its detach()");
}

void on_gpu(const char* name, const at::Tensor& t) {
  TORCH_CHECK_TYPE(t.is_cuda(), name, " must be on a GPU, got ", t.device().str(), ": the operators have no CPU path");
}

void check_shape(const char* name, const at::Tensor& t, int64_t rows, int64_t cols, ScalarType type, at::Device device) {
  TORCH_CHECK_TYPE(t.scalar_type() == type && t.device() == device, name, " must be ", c10::toString(type), " on ", device.str(), ", got ",
                   c10::toString(t.scalar_type()), " on ", t.device().str());
  TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, name, " must have shape (", rows, ", ", cols,
                    "), got ", t.sizes());
}

// a matrix whose rows are contiguous -> its row stride
int64_t matrix(const char* name, const at::Tensor& t, int64_t rows, int64_t cols, ScalarType type, at::Device device) {
  check_shape(name, t, rows, cols, type, device);
  TORCH_CHECK_VALUE(t.stride(1) == 1 || cols <= 1, name, ": the elements of a row must lie side by side, got strides ", t.strides());
  return t.stride(0);
}

// What an argument stands for: the tensor given, checked, or a new one whose rows are `ld` apart.
struct Matrix {
  int64_t address = 0, row = 0, col = 0;
  PyObject* object = nullptr;                // a new reference, or null
  bool theirs = false;                       // an output that the caller passed in
  Matrix() = default;
  Matrix(const Matrix&) = delete;
  ~Matrix() { Py_XDECREF(object); }
  PyObject* release() {
    PyObject* o = object ? object : Py_NewRef(Py_None);
    object = nullptr;
    return o;
  }
  void made(int64_t rows, int64_t cols, int64_t ld, ScalarType type, at::Device device) {
    at::Tensor t = at::empty_strided({rows, cols}, {ld, 1}, at::TensorOptions().dtype(type).device(device));
    address = ::address(t);
    row = ld;
    col = 1;
    object = THPVariable_Wrap(std::move(t));
    if (!object) throw python_error();
  }
  // a tensor of the caller's has been written: what autograd has saved of it counts as changed (a tensor of inference mode keeps
  // no such count)
  void written() const {
    if (!theirs) return;
    const at::Tensor& t = THPVariable_Unpack(object);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  void given(const char* name, PyObject* o, int64_t rows, int64_t cols, ScalarType type, at::Device device) {
    const at::Tensor& t = tensor(name, o);
    row = matrix(name, t, rows, cols, type, device);
    col = 1;
    address = ::address(t);
    object = Py_NewRef(o);
  }
  void given_any_strides(const char* name, PyObject* o, int64_t rows, int64_t cols, at::Device device) {
    const at::Tensor& t = tensor(name, o);
    check_shape(name, t, rows, cols, ScalarType::Float, device);
    row = t.stride(0);
    col = t.stride(1);
    address = ::address(t);
    object = Py_NewRef(o);
  }
  void output(const char* name, PyObject* o, int64_t rows, int64_t cols, int64_t ld, ScalarType type, at::Device device) {
    if (o == Py_None)
      made(rows, cols, ld, type, device);
    else
      given(name, o, rows, cols, type, device);
    theirs = o != Py_None;
  }
  void output_scales(PyObject* o, int64_t rows, int64_t cols, at::Device device) {
    if (o == Py_None)
      made(rows, cols, cols, ScalarType::Float, device);
    else
      given_any_strides("scale", o, rows, cols, device);
    theirs = o != Py_None;
  }
};

int64_t ld16(int64_t cols) { return (cols + 15) / 16 * 16; }

// raises what a negative status stands for
void raise_status(int status) {
  PyObject* r = PyObject_CallFunction(check_status, "i", status);
  Py_XDECREF(r);
  if (r) PyErr_Format(PyExc_RuntimeError, "status %d", status);
}

// false: a Python error is set
template <class Args>
bool run(int (*entry)(const Args*, int, uint64_t), const Args& args, int device) {
  PyObject* index = PyLong_FromLong(device);
  PyObject* handle = index ? PyObject_CallOneArg(stream_of, index) : nullptr;
  Py_XDECREF(index);
  const uint64_t stream = handle ? PyLong_AsUnsignedLongLongMask(handle) : 0;
  Py_XDECREF(handle);
  if (!handle || PyErr_Occurred()) return false;
  TORCH_CHECK(entry, "_kcg_torch is not bound to the library: call the operators through codegendemo_amd.kcg.Operators");
  int status;
  Py_BEGIN_ALLOW_THREADS                     // (a launch waits where the device's queue is full)
  status = entry(&args, device, stream);
  Py_END_ALLOW_THREADS
  if (status >= 0) return true;
  raise_status(status);
  return false;
}

bool count(const char* name, Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, n);
  return false;
}

PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count("bind", n, 7)) return nullptr;
  uint64_t entries[5];
  for (int i = 0; i < 5; ++i) entries[i] = PyLong_AsUnsignedLongLong(a[i]);
  if (PyErr_Occurred()) return nullptr;
  norm_entry = (decltype(norm_entry))(uintptr_t)entries[0];
  swiglu_entry = (decltype(swiglu_entry))(uintptr_t)entries[1];
  matmul_entry = (decltype(matmul_entry))(uintptr_t)entries[2];
  moe_entry = (decltype(moe_entry))(uintptr_t)entries[3];
  moe_workspace = (decltype(moe_workspace))(uintptr_t)entries[4];
  Py_XDECREF(stream_of);
  Py_XDECREF(check_status);
  stream_of = Py_NewRef(a[5]);
  check_status = Py_NewRef(a[6]);
  Py_RETURN_NONE;
}

// (x, weight, eps, residual, residual_out, q, scale, y, want_y) -> (q, scale, y, residual_out)
PyObject* rmsnorm_quant(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!count("rmsnorm_quant", n, 9)) return nullptr;
  no_gradient(a, n);
  const at::Tensor& x = tensor("x", a[0]);
  on_gpu("x", x);
  TORCH_CHECK_VALUE(x.dim() == 2, "x must be a matrix, got shape ", x.sizes());
  const ScalarType type = x.scalar_type();
  TORCH_CHECK_TYPE(code_of(type), "x must be bfloat16, float16 or float32, got ", c10::toString(type));
  const at::Device device = x.device();
  kcg_rmsnorm_quant_args p = {};
  p.rows = x.size(0);
  p.cols = x.size(1);
  p.x_stride = matrix("x", x, p.rows, p.cols, type, device);
  p.x = address(x);
  p.dtype = code_of(type);
  const at::Tensor& weight = tensor("weight", a[1]);
  const ScalarType wt = weight.scalar_type();
  TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == p.cols && (p.cols <= 1 || weight.stride(0) == 1) && weight.device() == device &&
                        (wt == type || wt == ScalarType::Float),
                    "weight must be a contiguous vector of ", p.cols, " values of ", c10::toString(type), " or Float on ", device.str());
  p.weight = address(weight);
  p.weight_dtype = code_of(wt);
  p.eps = PyFloat_AsDouble(a[2]);
  if (PyErr_Occurred()) return nullptr;
  Matrix residual, residual_out, q, scale, y;
  if (a[3] != Py_None) {
    residual.given("residual", a[3], p.rows, p.cols, type, device);
    residual_out.output("residual_out", a[4], p.rows, p.cols, p.cols, type, device);
  } else {
    TORCH_CHECK_VALUE(a[4] == Py_None, "residual_out without a residual");
  }
  q.output("q", a[5], p.rows, p.cols, ld16(p.cols), ScalarType::Float8_e4m3fn, device);
  scale.output_scales(a[6], p.rows, groups(p.cols), device);
  const int want_y = PyObject_IsTrue(a[8]);
  if (want_y < 0) return nullptr;
  if (want_y || a[7] != Py_None) y.output("y", a[7], p.rows, p.cols, p.cols, type, device);
  p.residual = residual.address, p.residual_stride = residual.row;
  p.residual_out = residual_out.address, p.residual_out_stride = residual_out.row;
  p.q = q.address, p.q_stride = q.row;
  p.scale = scale.address, p.scale_stride_row = scale.row, p.scale_stride_group = scale.col;
  p.y = y.address, p.y_stride = y.row;
  if (p.rows && p.cols) {
    if (!run(norm_entry, p, device.index())) return nullptr;
    for (const Matrix* m : {&residual_out, &q, &scale, &y}) m->written();
  }
  PyObject* r = PyTuple_New(4);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, q.release());
  PyTuple_SET_ITEM(r, 1, scale.release());
  PyTuple_SET_ITEM(r, 2, y.release());
  PyTuple_SET_ITEM(r, 3, residual_out.release());
  return r;
  END_HANDLE_TH_ERRORS
}

// (gate_up, q, scale) -> (q, scale)
PyObject* swiglu_quant(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!count("swiglu_quant", n, 3)) return nullptr;
  no_gradient(a, n);
  const at::Tensor& gate_up = tensor("gate_up", a[0]);
  on_gpu("gate_up", gate_up);
  TORCH_CHECK_VALUE(gate_up.dim() == 2 && gate_up.size(1) % 2 == 0, "gate_up must be a matrix with an even number of columns, got shape ", gate_up.sizes());
  const ScalarType type = gate_up.scalar_type();
  TORCH_CHECK_TYPE(code_of(type), "gate_up must be bfloat16, float16 or float32, got ", c10::toString(type));
  const at::Device device = gate_up.device();
  kcg_swiglu_quant_args p = {};
  p.rows = gate_up.size(0);
  p.cols = gate_up.size(1) / 2;
  p.gate_up_stride = matrix("gate_up", gate_up, p.rows, 2 * p.cols, type, device);
  p.gate_up = address(gate_up);
  p.dtype = code_of(type);
  Matrix q, scale;
  q.output("q", a[1], p.rows, p.cols, ld16(p.cols), ScalarType::Float8_e4m3fn, device);
  scale.output_scales(a[2], p.rows, groups(p.cols), device);
  p.q = q.address, p.q_stride = q.row;
  p.scale = scale.address, p.scale_stride_row = scale.row, p.scale_stride_group = scale.col;
  if (p.rows && p.cols) {
    if (!run(swiglu_entry, p, device.index())) return nullptr;
    for (const Matrix* m : {&q, &scale}) m->written();
  }
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, q.release());
  PyTuple_SET_ITEM(r, 1, scale.release());
  return r;
  END_HANDLE_TH_ERRORS
}

// (a, a_scale, b, b_scale, out, out_dtype) -> out
PyObject* matmul_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!count("matmul_fp8", n, 6)) return nullptr;
  no_gradient(a, n);
  const at::Tensor &ta = tensor("a", a[0]), &tb = tensor("b", a[2]);
  on_gpu("a", ta);
  TORCH_CHECK_VALUE(ta.dim() == 2 && tb.dim() == 2, "a and b must be matrices, got shapes ", ta.sizes(), " and ", tb.sizes());
  const at::Device device = ta.device();
  kcg_matmul_fp8_args p = {};
  p.m = ta.size(0);
  p.k = ta.size(1);
  p.n = tb.size(0);
  p.a_stride = matrix("a", ta, p.m, p.k, ScalarType::Float8_e4m3fn, device);
  p.b_stride = matrix("b", tb, p.n, p.k, ScalarType::Float8_e4m3fn, device);
  p.a = address(ta);
  p.b = address(tb);
  Matrix sa, sb, out;
  sa.given_any_strides("a_scale", a[1], p.m, groups(p.k), device);
  sb.given_any_strides("b_scale", a[3], groups(p.n), groups(p.k), device);
  ScalarType type;
  if (a[4] != Py_None) {
    type = tensor("out", a[4]).scalar_type();
  } else {
    TORCH_CHECK_TYPE(THPDtype_Check(a[5]), "out_dtype must be a torch.dtype, got ", Py_TYPE(a[5])->tp_name);
    type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  }
  TORCH_CHECK_TYPE(code_of(type), "out must be bfloat16, float16 or float32, got ", c10::toString(type));
  out.output("out", a[4], p.m, p.n, p.n, type, device);
  p.c_dtype = code_of(type);
  p.a_scale = sa.address, p.a_scale_stride_row = sa.row, p.a_scale_stride_group = sa.col;
  p.b_scale = sb.address, p.b_scale_stride_row = sb.row, p.b_scale_stride_group = sb.col;
  p.c = out.address, p.c_stride = out.row;
  if (p.m && p.n) {
    if (!run(matmul_entry, p, device.index())) return nullptr;
    out.written();
  }
  return out.release();
  END_HANDLE_TH_ERRORS
}

// weights [experts, rows, cols] with contiguous rows
void check_experts(const char* name, const at::Tensor& t, int64_t experts, int64_t rows, int64_t cols, at::Device device) {
  TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.device() == device && t.dim() == 3 && t.size(0) == experts && t.size(1) == rows && t.size(2) == cols, name,
                    " must have shape (", experts, ", ", rows, ", ", cols, ") on ", device.str(), ", got ", t.sizes(), " on ", t.device().str());
  TORCH_CHECK_VALUE(t.stride(2) == 1 || cols <= 1, name, ": the elements of a row must lie side by side, got strides ", t.strides());
}

// contiguous scales of blocks of 128 x 128 of `w`
int64_t block_scales(const char* name, PyObject* o, const at::Tensor& w, at::Device device) {
  const at::Tensor* s = o == Py_None ? nullptr : &tensor(name, o);
  const int64_t e = w.size(0), r = groups(w.size(1)), c = groups(w.size(2));
  TORCH_CHECK_VALUE(s && s->scalar_type() == ScalarType::Float && s->device() == device && s->dim() == 3 && s->size(0) == e && s->size(1) == r &&
                        s->size(2) == c && s->is_contiguous(),
                    name, " must be a contiguous torch.float32 tensor of shape (", e, ", ", r, ", ", c, ") on ", device.str());
  return address(*s);
}

// (x, logits, topk, w13, w2, w13_scale, w2_scale, renormalize, out) -> (out, ids, probs)
PyObject* moe_layer(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!count("moe_layer", n, 9)) return nullptr;
  no_gradient(a, n);
  const at::Tensor &x = tensor("x", a[0]), &logits = tensor("logits", a[1]), &w13 = tensor("w13", a[3]), &w2 = tensor("w2", a[4]);
  on_gpu("x", x);
  TORCH_CHECK_VALUE(x.dim() == 2 && logits.dim() == 2 && w13.dim() == 3, "x and logits must be matrices, w13 and w2 [experts, rows, columns]");
  const at::Device device = x.device();
  const ScalarType type = x.scalar_type(), wt = w13.scalar_type();
  kcg_moe_layer_args p = {};
  p.tokens = x.size(0);
  p.hidden = x.size(1);
  p.experts = logits.size(1);
  p.topk = PyLong_AsLongLong(a[2]);
  const int renormalize = PyObject_IsTrue(a[7]);
  if (PyErr_Occurred()) return nullptr;
  p.renormalize = renormalize;
  TORCH_CHECK_VALUE(w13.size(1) % 2 == 0, "w13 holds two weights of the same number of rows, got ", w13.size(1), " rows");
  p.inter = w13.size(1) / 2;
  p.x_stride = matrix("x", x, p.tokens, p.hidden, type, device);
  p.logits_stride = matrix("logits", logits, p.tokens, p.experts, ScalarType::Float, device);
  check_experts("w13", w13, p.experts, 2 * p.inter, p.hidden, device);
  check_experts("w2", w2, p.experts, p.hidden, p.inter, device);
  TORCH_CHECK_TYPE(w2.scalar_type() == wt && (wt == ScalarType::Float8_e4m3fn || wt == ScalarType::BFloat16) &&
                       (type == ScalarType::BFloat16 || type == ScalarType::Half),
                   "weights of ", c10::toString(wt), " and ", c10::toString(w2.scalar_type()), " with x of ", c10::toString(type),
                   ": e4m3 weights take bfloat16 or float16, bfloat16 weights bfloat16");
  if (wt == ScalarType::Float8_e4m3fn) {
    p.w13_scale = block_scales("w13_scale", a[5], w13, device);
    p.w2_scale = block_scales("w2_scale", a[6], w2, device);
    p.weight_dtype = KCG_DT_E4M3;
  } else {
    TORCH_CHECK_VALUE(a[5] == Py_None && a[6] == Py_None, "bfloat16 weights have no scales");
    p.weight_dtype = KCG_DT_BFLOAT16;
  }
  p.dtype = code_of(type);
  TORCH_CHECK(moe_workspace, "_kcg_torch is not bound to the library: call the operators through codegendemo_amd.kcg.Operators");
  p.workspace_bytes = moe_workspace(p.tokens, p.experts, p.topk, p.hidden, p.inter);
  if (p.workspace_bytes < 0) {
    raise_status((int)p.workspace_bytes);
    return nullptr;
  }
  Matrix out, ids, probs;
  out.output("out", a[8], p.tokens, p.hidden, p.hidden, type, device);
  ids.made(p.tokens, p.topk, p.topk, ScalarType::Int, device);
  probs.made(p.tokens, p.topk, p.topk, ScalarType::Float, device);
  p.x = address(x), p.logits = address(logits), p.w13 = address(w13), p.w2 = address(w2);
  p.out = out.address, p.out_stride = out.row, p.ids = ids.address, p.probs = probs.address;
  p.w13_stride_expert = w13.stride(0), p.w13_stride_row = w13.stride(1), p.w2_stride_expert = w2.stride(0), p.w2_stride_row = w2.stride(1);
  if (p.tokens) {
    // (freed to torch's allocator on return: what takes it over runs behind this call on the same stream)
    const at::Tensor workspace = at::empty_strided({p.workspace_bytes}, {1}, at::TensorOptions().dtype(ScalarType::Byte).device(device));
    p.workspace = address(workspace);
    if (!run(moe_entry, p, device.index())) return nullptr;
    out.written();
  }
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, out.release());
  PyTuple_SET_ITEM(r, 1, ids.release());
  PyTuple_SET_ITEM(r, 2, probs.release());
  return r;
  END_HANDLE_TH_ERRORS
}

#define METHOD(NAME) {#NAME, (PyCFunction)(void (*)(void))NAME, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(rmsnorm_quant), METHOD(swiglu_quant), METHOD(matmul_fp8), METHOD(moe_layer), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kcg_torch", "The operators of the 8-bit path on torch tensors.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kcg_torch(void) { return PyModule_Create(&module); }
