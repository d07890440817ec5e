// The operators over rows (zp_dropout, zp_layernorm_*, zp_add_layernorm_*) as functions on torch tensors with
// their gradients: the extension module zippel_b200._rowwise behind zippel_b200/blocks/rowwise.py.
//
// Written against torch's C++ interface, unlike the rest of this package's binding, for the time of a call: a
// layer norm of a few rows, forward and backward, takes 115 us with an autograd function in Python, of which
// the kernels are 6, and the kernels of 16384 rows of 4096 are as long as that.  Here it is 63 to 66 (around
// torch's own layer norm 68 to 71), and the forward alone 4 instead of 11.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>
#include <string>

#include "zippel_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// What a library call that failed raises: zippel_b200._lib.ZpError in a call from Python, and from the engine's
// threads what it makes of an exception's text.
struct Failed : std::exception {
  int status;
  const char *where;
  std::string text;
  Failed(int s, const char *w) : status(s), where(w) {
    text = std::string(w) + ": " + zp_status_string(s);
    if (s == ZP_ERR_CUDA) text += std::string(": ") + zp_last_cuda_error();
    text += " (status " + std::to_string(s) + ")";
  }
  const char *what() const noexcept override { return text.c_str(); }
};

void check(int status, const char *where) {
  if (status) throw Failed(status, where);
}

void *stream_of(const Tensor &x) { return c10::cuda::getCurrentCUDAStream(x.get_device()).stream(); }

// ---- arguments ------------------------------------------------------------------------------------

int type_number(at::ScalarType t) {
  return t == at::kFloat ? ZP_F32 : t == at::kHalf ? ZP_F16 : t == at::kBFloat16 ? ZP_BF16 : -1;
}

// A tracer records what goes through torch's dispatcher, which these calls do not: their results would be constants of
// the trace.
void need_no_trace(const char *what) {
  TORCH_CHECK(!at::tracer::impl::is_dispatch_enabled() &&
                  !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
              what, " leaves nothing in a trace: torch.jit.trace and make_fx cannot record it");
}

int need_rows(const Tensor &x, const char *what) {
  need_no_trace(what);
  TORCH_CHECK(x.is_cuda(), what, " needs CUDA tensors: there is no CPU path");
  const int type = type_number(x.scalar_type());
  TORCH_CHECK_TYPE(type >= 0, what, " takes float32, float16 and bfloat16, not ", x.scalar_type());
  return type;
}

// the type of weight and bias, which are checked against x (of type `type`)
int need_params(const Tensor &x, const Tensor &weight, const Tensor &bias, int type) {
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "a layer norm over the last axis of a tensor of shape ", x.sizes());
  int found = -1;
  for (const Tensor *t : {&weight, &bias}) {
    if (!t->defined()) continue;
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(-1), "weight or bias has shape ", t->sizes(), ", expected [",
                      x.size(-1), "]");
    TORCH_CHECK(t->device() == x.device(), "weight or bias is on ", t->device(), ", x on ", x.device());
    const int own = type_number(t->scalar_type());
    TORCH_CHECK_TYPE(own == type || own == ZP_F32, "weight or bias is ", t->scalar_type(), "; with x in ", x.scalar_type(),
                     " it may be that or float32");
    TORCH_CHECK_TYPE(found < 0 || own == found, "the weight is ", weight.scalar_type(), ", the bias ", bias.scalar_type());
    found = own;
  }
  return found < 0 ? type : found;
}

// ... without a look at them
int params_type(const Tensor &x, const Tensor &weight, const Tensor &bias) {
  return type_number((weight.defined() ? weight : bias.defined() ? bias : x).scalar_type());
}

// whether anything is dropped (p rounded to a multiple of 2^-16, as the library rounds it)
bool need_drop(const Tensor &x, double p, const Tensor &state) {
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "a probability is between 0 and 1: ", p);
  if (std::floor(65536.0 * p + 0.5) == 0.0) return false;
  TORCH_CHECK_VALUE(state.defined(), "dropout with p > 0 needs a state: dropout_state(device) draws one");
  TORCH_CHECK_VALUE(state.scalar_type() == at::kLong && state.dim() == 1 && state.size(0) == 2 && state.is_contiguous() &&
                        !state.is_neg(),
                    "a dropout state is two int64 one behind the other (seed, offset)");
  TORCH_CHECK(state.device() == x.device(), "the dropout state is on ", state.device(), ", x on ", x.device());
  return true;
}

// Whether autograd has to see a call: for a gradient, or to refuse tangents (forward mode).
bool recorded(std::initializer_list<const Tensor *> tensors) {
  const bool grad = at::GradMode::is_enabled();
  for (const Tensor *t : tensors)
    if (t->defined() && ((grad && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}

// ---- layout ---------------------------------------------------------------------------------------

// What the kernels read.  A wrapped tensor without memory (a functionalized one has a null address) is not one that
// is missing.
const void *address(const Tensor &t) {
  if (!t.defined() || !t.numel()) return nullptr;
  const void *p = t.const_data_ptr();
  TORCH_CHECK(p, "a tensor of shape ", t.sizes(), " has no memory of its own: it is wrapped, or zeroes that are not stored");
  return p;
}

struct Rows {                       // `t`: the tensor or a copy that the kernels can read
  Tensor t;
  int64_t rows, width, ld;
  const void *data() const { return address(t); }
};

// Whether what lies in memory is not the tensor's values: they are negated (imaginary parts of a conjugate), or zeroes
// that are not stored.  A clone has them in memory.
bool lazy(const Tensor &x) { return x.is_neg() || x._is_zerotensor(); }

// Rows that lie ld >= width elements apart are read where they are.  All others come from a copy, among them rows that
// are one row repeated (a stride of 0, as the gradient of a sum over rows has it) and rows that overlap.
Rows rows_of(const Tensor &x) {
  const int64_t w = x.dim() ? x.size(-1) : 1, rows = w ? x.numel() / w : 0;
  if (lazy(x)) return rows_of(x.clone());
  if (x.is_contiguous()) return {x, rows, w, w};
  bool fits = x.numel() && (x.stride(-1) == 1 || w == 1), found = false;
  int64_t ld = w, next = 0;
  for (int64_t i = x.dim() - 2; i >= 0 && fits; --i) {       // leading axes one row behind the other
    if (x.size(i) == 1) continue;
    if (!found) {
      found = true;
      ld = x.stride(i);
      fits = ld >= w;
    } else {
      fits = x.stride(i) == next;
    }
    next = x.stride(i) * x.size(i);
  }
  if (fits) return {x, rows, w, ld};
  return {x.contiguous(), rows, w, w};
}

// new arrays, without the dispatcher's detour (0.5 us each)
Tensor array(at::IntArrayRef sizes, at::ScalarType type, const Tensor &beside) {
  return at::detail::empty_cuda(sizes, type, beside.device(), std::nullopt);
}
Tensor like(const Tensor &x) { return array(x.sizes(), x.scalar_type(), x); }    // row behind row
Tensor lined_up(const Tensor &t) {
  return t.defined() && (!t.is_contiguous() || lazy(t)) ? t.clone(at::MemoryFormat::Contiguous) : t;
}
void *room(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
const int64_t *state_of(const Tensor &t) { return static_cast<const int64_t *>(address(t)); }

Tensor stats_for(const Tensor &x, int64_t rows) {            // mean and 1/std, one behind the other
  return array({2, rows}, at::kFloat, x);
}
const float *mean_of(const Tensor &stats) { return stats.const_data_ptr<float>(); }
const float *rstd_of(const Tensor &stats) { return mean_of(stats) + stats.size(1); }

struct ParamGrads {
  Tensor weight, bias, work;
  ParamGrads(const Tensor &w, const Tensor &b, bool want_w, bool want_b, int64_t rows) {
    if (want_w) weight = like(w);
    if (want_b) bias = like(b);
    if (!want_w && !want_b) return;
    const Tensor &t = want_w ? w : b;
    const size_t bytes = zp_rowwise_work_bytes(rows, t.size(0));
    work = array({(int64_t)bytes}, at::kByte, t);
  }
  size_t bytes() const { return work.defined() ? (size_t)work.numel() : 0; }
};

// Gradients as they are, or, where a graph of the backward is asked for, behind a node that refuses to be
// differentiated.
variable_list first_order(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "the operators over rows are differentiated once: their gradients have none", (int64_t)grads.size());
  for (Tensor &t : grads)
    if (t.defined()) t = t.detach().requires_grad_(true);
  return (*node)(std::move(grads));
}

// ---- dropout --------------------------------------------------------------------------------------

Tensor dropped(const Tensor &x, double p, const Tensor &state) {
  Tensor y = like(x);
  if (!y.numel()) return y;
  c10::cuda::CUDAGuard guard(x.device());
  const Rows r = rows_of(x);
  check(zp_dropout(r.rows, r.width, type_number(x.scalar_type()), r.data(), r.ld, p, state_of(state), y.data_ptr(), r.width,
                   stream_of(x)), "zp_dropout");
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, double p, const Tensor &state) {
    ctx->saved_data["p"] = p;
    ctx->save_for_backward({state});
    return dropped(x, p, state);
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const variable_list saved = ctx->get_saved_variables();
    return first_order({dropped(grads[0], ctx->saved_data["p"].toDouble(), saved[0]), Tensor(), Tensor()});
  }
};

Tensor dropout(const Tensor &x, double p, const Tensor &state) {
  need_rows(x, "dropout");
  if (!need_drop(x, p, state)) return x;
  return recorded({&x}) ? Dropout::apply(x, p, state) : dropped(x, p, state);
}

// ---- layer norm -----------------------------------------------------------------------------------

Tensor norm(const Rows &r, const Tensor &x, const Tensor &weight, const Tensor &bias, double eps, int ptype,
            const Tensor &stats) {
  Tensor y = like(x);
  c10::cuda::CUDAGuard guard(x.device());
  float *mean = stats.defined() ? stats.data_ptr<float>() : nullptr;
  check(zp_layernorm_forward(r.rows, r.width, type_number(x.scalar_type()), r.data(), r.ld, ptype, address(weight),
                             address(bias), (float)eps, y.data_ptr(), mean, mean ? mean + r.rows : nullptr, stream_of(x)),
        "zp_layernorm_forward");
  return y;
}

// (an input that is missing is an undefined tensor; it has no place among the inputs that want gradients)
bool wanted(AutogradContext *ctx, const Tensor &t, size_t &place) {
  return t.defined() && ctx->needs_input_grad(place++);
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &weight,
                        const std::optional<Tensor> &bias, double eps, int64_t ptype) {
    const Tensor w = lined_up(weight.value_or(Tensor())), b = lined_up(bias.value_or(Tensor()));
    const Rows r = rows_of(x);
    const Tensor stats = stats_for(x, r.rows);
    ctx->save_for_backward({r.t, w, b, stats});
    return norm(r, x, w, b, eps, (int)ptype, stats);
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
    size_t place = 0;
    const bool want_x = wanted(ctx, x, place), want_w = wanted(ctx, weight, place), want_b = wanted(ctx, bias, place);
    c10::cuda::CUDAGuard guard(x.device());
    const Rows r = rows_of(x), g = rows_of(grads[0]);
    Tensor dx = want_x ? like(x) : Tensor();
    ParamGrads params(weight, bias, want_w, want_b, r.rows);
    check(zp_layernorm_backward(r.rows, r.width, type_number(x.scalar_type()), r.data(), r.ld,
                                params_type(x, weight, bias), address(weight), mean_of(stats), rstd_of(stats), g.data(),
                                g.ld, room(dx), room(params.weight), room(params.bias), room(params.work),
                                params.bytes(), stream_of(x)), "zp_layernorm_backward");
    return first_order({dx, params.weight, params.bias, Tensor(), Tensor()});
  }
};

std::optional<Tensor> given(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

Tensor layer_norm(const Tensor &x, const Tensor &weight, const Tensor &bias, double eps) {
  const int type = need_rows(x, "layer_norm"), ptype = need_params(x, weight, bias, type);
  if (recorded({&x, &weight, &bias})) return LayerNorm::apply(x, given(weight), given(bias), eps, (int64_t)ptype);
  return norm(rows_of(x), x, lined_up(weight), lined_up(bias), eps, ptype, Tensor());
}

// ---- the join -------------------------------------------------------------------------------------

variable_list add_norm(const Tensor &x, const Tensor &residual, const Tensor &weight, const Tensor &bias, double p,
                       const Tensor &state, double eps, int ptype, const Tensor &stats) {
  Tensor y = like(x), s = like(x);
  c10::cuda::CUDAGuard guard(x.device());
  const Rows r = rows_of(x), q = rows_of(residual);
  float *mean = stats.defined() ? stats.data_ptr<float>() : nullptr;
  check(zp_add_layernorm_forward(r.rows, r.width, type_number(x.scalar_type()), r.data(), r.ld, q.data(), q.ld, p,
                                 state_of(state), ptype, address(weight), address(bias), (float)eps, s.data_ptr(),
                                 y.data_ptr(), mean, mean ? mean + r.rows : nullptr, stream_of(x)),
        "zp_add_layernorm_forward");
  return {y, s};
}

struct DropoutAddLayerNorm : torch::autograd::Function<DropoutAddLayerNorm> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &residual,
                               const std::optional<Tensor> &weight, const std::optional<Tensor> &bias, double p,
                               const std::optional<Tensor> &state, double eps, int64_t ptype) {
    const Tensor w = lined_up(weight.value_or(Tensor())), b = lined_up(bias.value_or(Tensor()));
    const Tensor st = state.value_or(Tensor());
    const Tensor stats = stats_for(x, x.numel() / x.size(-1));
    variable_list out = add_norm(x, residual, w, b, p, st, eps, (int)ptype, stats);
    ctx->saved_data["p"] = p;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({out[1], w, b, stats, st});
    return out;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &s = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3], &state = saved[4];
    variable_list out(8);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    size_t place = 0;
    const bool want_x = wanted(ctx, s, place), want_res = wanted(ctx, s, place);
    const bool want_w = wanted(ctx, weight, place), want_b = wanted(ctx, bias, place);
    c10::cuda::CUDAGuard guard(s.device());
    const Rows r = rows_of(s);
    Rows gy = {}, gs = {};
    if (grads[0].defined()) gy = rows_of(grads[0]);
    if (grads[1].defined()) gs = rows_of(grads[1]);
    // without dropout the two gradients are one, and one tensor
    Tensor dres = want_res || (want_x && !state.defined()) ? like(s) : Tensor();
    Tensor dx = want_x && state.defined() ? like(s) : Tensor();
    ParamGrads params(weight, bias, want_w, want_b, r.rows);
    check(zp_add_layernorm_backward(r.rows, r.width, type_number(s.scalar_type()), r.data(),
                                    params_type(s, weight, bias), address(weight), mean_of(stats), rstd_of(stats),
                                    address(gy.t), gy.ld, address(gs.t), gs.ld, ctx->saved_data["p"].toDouble(),
                                    state_of(state), room(dx), room(dres), room(params.weight), room(params.bias),
                                    room(params.work), params.bytes(), stream_of(s)), "zp_add_layernorm_backward");
    if (want_x) out[0] = state.defined() ? dx : dres;
    if (want_res) out[1] = dres;
    out[2] = params.weight;
    out[3] = params.bias;
    return first_order(std::move(out));
  }
};

variable_list dropout_add_layer_norm(const Tensor &x, const Tensor &residual, const Tensor &weight, const Tensor &bias,
                                     double p, Tensor state, double eps) {
  const int type = need_rows(x, "dropout_add_layer_norm"), ptype = need_params(x, weight, bias, type);
  TORCH_CHECK_VALUE(residual.sizes() == x.sizes(), "the residual has shape ", residual.sizes(), ", x ", x.sizes());
  TORCH_CHECK(residual.device() == x.device(), "the residual is on ", residual.device(), ", x on ", x.device());
  TORCH_CHECK_TYPE(residual.scalar_type() == x.scalar_type(), "the residual is ", residual.scalar_type(), ", x is ",
                   x.scalar_type());
  if (!need_drop(x, p, state)) {
    p = 0.0;
    state = Tensor();
  }
  if (recorded({&x, &residual, &weight, &bias}))
    return DropoutAddLayerNorm::apply(x, residual, given(weight), given(bias), p, given(state), eps, (int64_t)ptype);
  return add_norm(x, residual, lined_up(weight), lined_up(bias), p, state, eps, ptype, Tensor());
}

// ---- Python ---------------------------------------------------------------------------------------

Tensor tensor_arg(PyObject *o, const char *what) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, " is a tensor, not ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
Tensor tensor_or_none(PyObject *o, const char *what) { return o == Py_None ? Tensor() : tensor_arg(o, what); }
double number_arg(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

PyObject *raise(const Failed &f) {
  PyObject *module = PyImport_ImportModule("zippel_b200._lib");
  PyObject *type = module ? PyObject_GetAttrString(module, "ZpError") : nullptr;
  PyObject *error = type ? PyObject_CallFunction(type, "is", f.status, f.where) : nullptr;
  if (error) PyErr_SetObject(type, error);
  Py_XDECREF(error);
  Py_XDECREF(type);
  Py_XDECREF(module);
  return nullptr;
}

PyObject *pair(const variable_list &out) {
  PyObject *y = THPVariable_Wrap(out[0]), *s = THPVariable_Wrap(out[1]);
  PyObject *both = PyTuple_Pack(2, y, s);
  Py_DECREF(y);
  Py_DECREF(s);
  return both;
}

// CALL is worked out without the interpreter's lock, WRAP(result) with it
#define ENTRY(NAME, COUNT, ARGS, CALL, WRAP)                                          \
  PyObject *py_##NAME(PyObject *, PyObject *const *a, Py_ssize_t n) {                 \
    HANDLE_TH_ERRORS                                                                  \
    try {                                                                             \
      TORCH_CHECK_TYPE(n == COUNT, #NAME " takes " #COUNT " arguments, not ", n);     \
      ARGS;                                                                           \
      auto out = [&] {                                                                \
        pybind11::gil_scoped_release released;                                        \
        return CALL;                                                                  \
      }();                                                                            \
      return WRAP(out);                                                               \
    } catch (const Failed &f) {                                                       \
      return raise(f);                                                                \
    }                                                                                 \
    END_HANDLE_TH_ERRORS                                                              \
  }

ENTRY(layer_norm, 4,
      const Tensor x = tensor_arg(a[0], "x");
      const Tensor w = tensor_or_none(a[1], "the weight");
      const Tensor b = tensor_or_none(a[2], "the bias");
      const double eps = number_arg(a[3]),
      layer_norm(x, w, b, eps), THPVariable_Wrap)
ENTRY(dropout, 3,
      const Tensor x = tensor_arg(a[0], "x");
      const double p = number_arg(a[1]);
      const Tensor state = tensor_or_none(a[2], "the state"),
      dropout(x, p, state), THPVariable_Wrap)
ENTRY(dropout_add_layer_norm, 7,
      const Tensor x = tensor_arg(a[0], "x");
      const Tensor residual = tensor_arg(a[1], "the residual");
      const Tensor w = tensor_or_none(a[2], "the weight");
      const Tensor b = tensor_or_none(a[3], "the bias");
      const double p = number_arg(a[4]);
      const Tensor state = tensor_or_none(a[5], "the state");
      const double eps = number_arg(a[6]),
      dropout_add_layer_norm(x, residual, w, b, p, state, eps), pair)

// (rows, width, ld, whether they are a copy's) of a tensor as the functions above read it, on whatever device
PyObject *py_row_layout(PyObject *, PyObject *a) {
  HANDLE_TH_ERRORS
  const Tensor x = tensor_arg(a, "x");
  const Rows r = rows_of(x);
  return Py_BuildValue("LLLN", (long long)r.rows, (long long)r.width, (long long)r.ld, PyBool_FromLong(!r.t.is_same(x)));
  END_HANDLE_TH_ERRORS
}

template <typename F> PyCFunction fast(F *f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(f)); }
PyMethodDef methods[] = {
    {"layer_norm", fast(py_layer_norm), METH_FASTCALL, "layer_norm(x, weight, bias, eps)"},
    {"dropout", fast(py_dropout), METH_FASTCALL, "dropout(x, p, state)"},
    {"dropout_add_layer_norm", fast(py_dropout_add_layer_norm), METH_FASTCALL,
     "dropout_add_layer_norm(x, residual, weight, bias, p, state, eps)"},
    {"row_layout", py_row_layout, METH_O, "row_layout(x): (rows, width, ld, copied)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_rowwise", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__rowwise() { return PyModule_Create(&module_def); }
