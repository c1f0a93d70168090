// Host side of the operators whose call cost is their latency: reading torch tensors (addresses,
// strides, types) and filling the C ABI's structures in C++ instead of in Python.  288 tensors of an
// optimizer step cost 440 us of attribute reads in Python and 29 us here (the whole call of
// ops.adamw_step); a norm's forward 12 us and 5 us.
//
// A CPython module over torch's C++ API; it holds no state and no numerics, checks its tensors, and
// calls libunirl_hip.so.  Functions return the C ABI's status beside their tensors; the Python layer turns
// it into an exception.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/engine.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <optional>
#include <vector>

#include "../../include/unirl_hip.h"

namespace {

using at::Tensor;

// --- arguments ---------------------------------------------------------------
const Tensor& tensor_of(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor; got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
std::optional<Tensor> optional_of(PyObject* o, const char* name) {
  if (o == Py_None) return std::nullopt;
  return tensor_of(o, name);
}
int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return UNIRL_F32;
    case at::kBFloat16: return UNIRL_BF16;
    case at::kHalf: return UNIRL_F16;
    default: break;
  }
  TORCH_CHECK_TYPE(false, "unsupported dtype torch.", at::toString(t), "; expected float32, bfloat16 or float16");
}
void require_device(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " lives on ", t.device(),
              ": unirl_amd kernels run on a HIP device only (there is no CPU fallback; use the torch reference for CPU tensors)");
}
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
void expect(Py_ssize_t got, Py_ssize_t want, const char* name) {
  TORCH_CHECK_TYPE(got == want, name, " takes ", want, " arguments; got ", got);
}

// A sequence of tensors, held for the call.
struct TensorList {
  PyObject* seq = nullptr;
  const char* name;
  TensorList(PyObject* o, const char* n) : name(n) {
    if (o == Py_None) return;
    seq = PySequence_Fast(o, "a sequence of tensors is needed");
    if (!seq) throw python_error();
  }
  ~TensorList() { Py_XDECREF(seq); }
  TensorList(const TensorList&) = delete;
  TensorList& operator=(const TensorList&) = delete;
  explicit operator bool() const { return seq != nullptr; }
  int64_t size() const { return seq ? PySequence_Fast_GET_SIZE(seq) : 0; }
  const Tensor& operator[](int64_t i) const { return tensor_of(PySequence_Fast_GET_ITEM(seq, i), name); }
};

// --- norm ---------------------------------------------------------------------
// A [groups, rows, D] reading of x [..., D]: in place when its leading dimensions are at most two runs of
// equally spaced rows (per group, dimension 0 is the groups), else of a contiguous copy.  Shared gains
// leave one partial sum per group, so many short groups are copied together as well.
struct Rows {
  Tensor t;
  int64_t groups, rows, group_stride, row_stride;
};
Rows rows_of(const Tensor& x, bool per_group) {
  const int64_t dims = x.dim(), D = x.size(-1);
  Tensor t = x;
  if (!x.is_contiguous()) {
    std::array<std::array<int64_t, 2>, 2> runs{};  // size, stride
    int n = 0;
    bool fits = x.stride(-1) == 1 || D == 1;
    for (int64_t i = 0; i + 1 < dims && fits; ++i) {
      const int64_t size = x.size(i), stride = x.stride(i);
      const bool apart = per_group && i == 0;
      if (size == 1 && !apart) continue;
      if (n > 0 && !(per_group && n == 1) && runs[n - 1][1] == stride * size)
        runs[n - 1] = {runs[n - 1][0] * size, stride};
      else if (n < 2)
        runs[n++] = {size, stride};
      else
        fits = false;
    }
    if (fits && (per_group || n < 2 || runs[0][0] <= 256)) {
      if (n < 2 && per_group) {
        for (; n < 2; ++n) runs[n] = {1, 0};
      } else if (n < 2) {
        runs[1] = n ? runs[0] : std::array<int64_t, 2>{1, 0};
        runs[0] = {1, 0};
      }
      return {t, runs[0][0], runs[1][0], runs[0][1], runs[1][1]};
    }
    t = x.contiguous();
  }
  const int64_t n = t.numel() / D;
  if (per_group) {
    const int64_t G = t.size(0), R = G ? n / G : 0;
    return {t, G, R, R * D, D};
  }
  return {t, 1, n, 0, D};
}

// What a norm call reads, with the descriptor's pointers into it.
struct NormCall {
  struct unirl_norm_desc desc = {};
  Rows x;
  std::optional<Tensor> weight, bias;
  bool per_group = false;
};
bool norm_param(std::optional<Tensor>& p, const Tensor& x, const char* name) {
  if (!p) return false;
  require_device(*p, name);
  TORCH_CHECK_VALUE(p->device() == x.device(), name, " lives on ", p->device(), ", x on ", x.device());
  const int64_t D = x.size(-1);
  const bool shared = p->dim() == 1 && p->size(0) == D;
  const bool rows = p->dim() == 2 && x.dim() >= 2 && p->size(0) == x.size(0) && p->size(1) == D;
  TORCH_CHECK_VALUE(shared || rows, name, " must be [", D, "] or [groups, ", D, "]; got ", p->sizes());
  dtype_code(p->scalar_type());
  if (p->stride(-1) != 1 && D > 1) p = p->contiguous();
  return rows;
}
NormCall norm_call(const Tensor& x, std::optional<Tensor> weight, std::optional<Tensor> bias, double eps, bool rms, bool unit_offset) {
  NormCall c;
  require_device(x, "x");
  const int code = dtype_code(x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must be [..., D] with D >= 1; got ", x.sizes());
  c.weight = std::move(weight);
  c.bias = std::move(bias);
  const bool wr = norm_param(c.weight, x, "weight"), br = norm_param(c.bias, x, "bias");
  TORCH_CHECK_VALUE(!c.weight || !c.bias || (c.weight->scalar_type() == c.bias->scalar_type() && wr == br),
                    "weight and bias differ in dtype or shape");
  c.per_group = wr || br;
  c.x = rows_of(x, c.per_group);
  auto& d = c.desc;
  d.x = c.x.t.data_ptr();
  d.dtype = code;
  d.groups = c.x.groups;
  d.rows = c.x.rows;
  d.x_group_stride = c.x.group_stride;
  d.x_row_stride = c.x.row_stride;
  d.D = x.size(-1);
  d.gain = c.weight ? c.weight->data_ptr() : nullptr;
  d.bias = c.bias ? c.bias->data_ptr() : nullptr;
  d.gain_dtype = c.weight ? dtype_code(c.weight->scalar_type()) : (c.bias ? dtype_code(c.bias->scalar_type()) : UNIRL_F32);
  d.gain_group_stride = wr ? c.weight->stride(0) : 0;
  d.bias_group_stride = br ? c.bias->stride(0) : 0;
  d.gain_offset = unit_offset ? 1.0f : 0.0f;
  d.center = rms ? 0 : 1;
  d.eps = eps;
  return c;
}

struct NormOut {
  int rc = 0;
  Tensor y, mean, rstd;
};
NormOut norm_forward(const Tensor& x, std::optional<Tensor> weight, std::optional<Tensor> bias, double eps, bool rms, bool unit_offset,
                     bool want_stats) {
  NormCall c = norm_call(x, std::move(weight), std::move(bias), eps, rms, unit_offset);
  c10::hip::HIPGuard guard(x.device().index());
  NormOut o;
  o.y = at::empty(x.sizes(), x.options());
  if (want_stats) {
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    o.rstd = at::empty(lead, x.options().dtype(at::kFloat));
    if (!rms) o.mean = at::empty(lead, o.rstd.options());
    c.desc.rstd = o.rstd.data_ptr<float>();
    c.desc.mean = rms ? nullptr : o.mean.data_ptr<float>();
  }
  if (o.y.numel()) o.rc = unirl_layer_norm_fwd(&c.desc, o.y.data_ptr(), stream_of(x));
  return o;
}

struct NormGrads {
  int rc = 0;
  Tensor dx, dweight, dbias;
};
NormGrads norm_backward(const Tensor& dy, const Tensor& x, std::optional<Tensor> mean, Tensor rstd, std::optional<Tensor> weight,
                        std::optional<Tensor> bias, bool rms, bool unit_offset, bool want_dx, bool want_dweight, bool want_dbias) {
  NormCall c = norm_call(x, std::move(weight), std::move(bias), 0.0, rms, unit_offset);
  c10::hip::HIPGuard guard(x.device().index());
  TORCH_CHECK_VALUE(dy.sizes() == x.sizes(), "dy ", dy.sizes(), " != x ", x.sizes());
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  TORCH_CHECK_VALUE(rstd.sizes() == lead && (rms || (mean && mean->sizes() == lead)), "mean and rstd must be the statistics of this x");
  const auto f32 = x.options().dtype(at::kFloat);
  rstd = rstd.to(f32).contiguous();
  if (!rms) mean = mean->to(f32).contiguous();
  c.desc.rstd = rstd.data_ptr<float>();
  c.desc.mean = rms ? nullptr : mean->data_ptr<float>();
  Rows g = rows_of(dy.to(x.options()), c.per_group);
  if (g.groups != c.desc.groups || g.rows != c.desc.rows)  // cut into groups unlike x's
    g = {g.t.contiguous(), c.desc.groups, c.desc.rows, c.desc.rows * c.desc.D, c.desc.D};
  NormGrads o;
  Tensor scratch;
  if (want_dx) o.dx = at::empty(x.sizes(), x.options());
  if (want_dweight && c.weight) o.dweight = at::empty(c.weight->sizes(), c.weight->options());
  if (want_dbias && c.bias) o.dbias = at::empty(c.bias->sizes(), c.bias->options());
  const auto address = [](const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; };
  if (o.dx.defined() || o.dweight.defined() || o.dbias.defined()) {
    size_t bytes = 0;
    if (o.dweight.defined() || o.dbias.defined()) {
      bytes = unirl_layer_norm_bwd_scratch_bytes(c.desc.groups, c.desc.rows, c.desc.D);
      scratch = at::empty({(int64_t)std::max<size_t>(bytes, 16)}, x.options().dtype(at::kByte));
    }
    o.rc = unirl_layer_norm_bwd(&c.desc, g.t.data_ptr(), g.group_stride, g.row_stride, address(o.dx), address(o.dweight),
                                address(o.dbias), c.per_group, address(scratch), bytes, stream_of(x));
  }
  return o;
}

// layer_norm(x, weight, bias, eps, rms, unit_offset, want_stats) -> (status, y, mean, rstd)
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 7, "layer_norm");
  at::AutoDispatchBelowADInplaceOrView no_grad;
  const NormOut o = norm_forward(tensor_of(a[0], "x"), optional_of(a[1], "weight"), optional_of(a[2], "bias"), number(a[3]),
                                 truth(a[4]), truth(a[5]), truth(a[6]));
  return Py_BuildValue("(iNNN)", o.rc, wrap(o.y), wrap(o.mean), wrap(o.rstd));
  END_HANDLE_TH_ERRORS
}

// layer_norm_bwd(dy, x, mean, rstd, weight, bias, rms, unit_offset, want_dx, want_dweight, want_dbias)
//   -> (status, dx, dweight, dbias)
PyObject* layer_norm_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 11, "layer_norm_bwd");
  at::AutoDispatchBelowADInplaceOrView no_grad;
  const NormGrads o = norm_backward(tensor_of(a[0], "dy"), tensor_of(a[1], "x"), optional_of(a[2], "mean"), tensor_of(a[3], "rstd"),
                                    optional_of(a[4], "weight"), optional_of(a[5], "bias"), truth(a[6]), truth(a[7]), truth(a[8]),
                                    truth(a[9]), truth(a[10]));
  return Py_BuildValue("(iNNN)", o.rc, wrap(o.dx), wrap(o.dweight), wrap(o.dbias));
  END_HANDLE_TH_ERRORS
}

// The differentiable form: one node whose backward runs in the autograd engine's thread without Python.
void check(int rc, const char* what) {
  TORCH_CHECK_VALUE(rc >= 0, what, ": ", unirl_status_string(rc), " (status ", rc, ")");
  TORCH_CHECK(rc == 0, what, ": HIP error ", rc, ": ", unirl_status_string(rc));
}
// A leaf's accumulator works on the stream that was current when the first graph that still lives was
// built over the leaf.  Where that is the default stream, the engine would make it wait for work that is
// being captured, which breaks the capture and can end the process: refused while nothing is lost.
void refuse_accumulators_outside_a_capture(int8_t device) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(c10::hip::getCurrentHIPStream(device).stream(), &status) != hipSuccess ||
      status == hipStreamCaptureStatusNone)
    return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  const auto outside = c10::hip::getDefaultHIPStream(device);
  for (size_t i = 0; i < node->num_outputs(); ++i) {
    const auto& to = node->next_edge(i).function;
    if (!dynamic_cast<torch::autograd::AccumulateGrad*>(to.get()) || !node->task_should_compute_output(i)) continue;
    const auto stream = to->stream();
    TORCH_CHECK(!stream || stream->id() != outside.id() || stream->device_index() != device,
                "the norm's backward is captured while a graph built on the default stream over the same leaf is alive: "
                "release that graph (its outputs and losses) before the captured forward");
  }
}
using torch::autograd::variable_list;
constexpr int64_t kGradientGroups = 65535;  // of unirl_layer_norm_bwd with dgain or dbias per group
struct NormFunction : torch::autograd::Function<NormFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                        const std::optional<Tensor>& bias, double eps, bool rms, bool unit_offset) {
    for (const auto* p : {&weight, &bias})  // what the backward would refuse is refused here
      TORCH_CHECK_VALUE(!*p || (*p)->dim() < 2 || !(*p)->requires_grad() || (*p)->size(0) <= kGradientGroups,
                        "gains and biases per group have gradients up to the limit of ", kGradientGroups, " groups; got ",
                        (*p)->size(0));
    at::AutoDispatchBelowADInplaceOrView no_grad;
    const NormOut o = norm_forward(x, weight, bias, eps, rms, unit_offset, true);
    check(o.rc, "unirl_layer_norm_fwd");
    ctx->save_for_backward({x, weight.value_or(Tensor()), bias.value_or(Tensor()), o.mean, o.rstd});
    ctx->saved_data["rms"] = rms;
    ctx->saved_data["unit_offset"] = unit_offset;
    return o.y;
  }
  static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list dy) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &mean = saved[3];
    const auto optional = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    refuse_accumulators_outside_a_capture(x.device().index());
    const size_t bias_edge = weight.defined() ? 2 : 1;  // only the tensors that are there have an edge
    NormGrads o;
    {
      at::AutoDispatchBelowADInplaceOrView no_grad;
      o = norm_backward(dy[0], x, optional(mean), saved[4], optional(weight), optional(bias), ctx->saved_data["rms"].toBool(),
                        ctx->saved_data["unit_offset"].toBool(), ctx->needs_input_grad(0),
                        weight.defined() && ctx->needs_input_grad(1), bias.defined() && ctx->needs_input_grad(bias_edge));
    }
    check(o.rc, "unirl_layer_norm_bwd");
    variable_list grads = {o.dx, o.dweight, o.dbias};
    if (at::GradMode::is_enabled()) {  // create_graph: a second derivative, if one is taken, has to fail
      for (Tensor& g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true);
      const auto error = std::make_shared<torch::autograd::DelayedError>("the norm's backward is not differentiable", 3);
      grads = (*error)(std::move(grads));
    }
    grads.resize(6);
    return grads;
  }
};

// norm(x, weight, bias, eps, rms, unit_offset) -> y, differentiable in the first three
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 6, "norm");
  const Tensor& x = tensor_of(a[0], "x");
  const std::optional<Tensor> weight = optional_of(a[1], "weight"), bias = optional_of(a[2], "bias");
  const double eps = number(a[3]);
  const bool rms = truth(a[4]), unit_offset = truth(a[5]);
  const auto is_dual = [](const std::optional<Tensor>& t) { return t && t->_fw_grad(0).defined(); };
  TORCH_CHECK(!is_dual(x) && !is_dual(weight) && !is_dual(bias), "the norm has no forward-mode derivative");
  const auto wants = [](const std::optional<Tensor>& t) { return t && t->requires_grad(); };
  if (at::GradMode::is_enabled() && (x.requires_grad() || wants(weight) || wants(bias)))
    return wrap(NormFunction::apply(x, weight, bias, eps, rms, unit_offset));
  at::AutoDispatchBelowADInplaceOrView no_grad;
  const NormOut o = norm_forward(x, weight, bias, eps, rms, unit_offset, false);
  check(o.rc, "unirl_layer_norm_fwd");
  return wrap(o.y);
  END_HANDLE_TH_ERRORS
}

// --- lists of tensors -----------------------------------------------------------
// grad_norm(tensors) -> (status, norm)
PyObject* grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  expect(n_args, 1, "grad_norm");
  at::AutoDispatchBelowADInplaceOrView no_grad;
  const TensorList list(a[0], "grads");
  const int64_t n = list.size();
  TORCH_CHECK_VALUE(n > 0, "grad_norm needs at least one tensor");
  const at::Device device = list[0].device();
  require_device(list[0], "grads[0]");
  c10::hip::HIPGuard guard(device.index());
  std::vector<const void*> ptrs(n);
  std::vector<int64_t> numels(n);
  std::vector<int> codes(n);
  std::vector<Tensor> copies;
  for (int64_t i = 0; i < n; ++i) {
    const Tensor* t = &list[i];
    TORCH_CHECK_VALUE(t->device() == device, "grad_norm: the tensors live on different devices");
    codes[i] = dtype_code(t->scalar_type());
    if (!t->is_contiguous()) {
      copies.push_back(t->contiguous());
      t = &copies.back();
    }
    ptrs[i] = t->data_ptr();
    numels[i] = t->numel();
  }
  const auto on = at::TensorOptions().device(device);
  const Tensor out = at::empty({}, on.dtype(at::kFloat));
  // scratch of this call alone: calls on other streams, and graphs, never share it
  const int64_t bytes = (int64_t)unirl_workspace_bytes();
  const Tensor ws = at::empty({bytes}, on.dtype(at::kByte));
  const int rc = unirl_grad_norm(ptrs.data(), numels.data(), codes.data(), n, out.data_ptr<float>(), ws.data_ptr(), (size_t)bytes,
                                 stream_of(out));
  return Py_BuildValue("(iN)", rc, wrap(out));
  END_HANDLE_TH_ERRORS
}

void check_entry(const Tensor& t, const char* name, int64_t i, int64_t numel, at::ScalarType dtype, at::Device device) {
  TORCH_CHECK_VALUE(t.numel() == numel && t.scalar_type() == dtype && t.device() == device && t.is_contiguous(), name, "[", i,
                    "] must be a contiguous ", at::toString(dtype), " tensor of ", numel, " elements on ", device, "; got ",
                    at::toString(t.scalar_type()), " ", t.sizes(), " strides ", t.strides(), " on ", t.device());
}

// adamw_step(params, grads, exp_avgs, exp_avg_sqs, masters, exp_avg_scales, exp_avg_sq_scales, index_bases,
//            lr, beta1, beta2, eps, weight_decay, step, seed, grad_norm, max_norm, skip_nonfinite, control) -> status
PyObject* adamw_step(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  expect(n_args, 19, "adamw_step");
  at::AutoDispatchBelowADInplaceOrView no_grad;
  const TensorList params(a[0], "params"), grads(a[1], "grads"), ms(a[2], "exp_avgs"), vs(a[3], "exp_avg_sqs"), masters(a[4], "masters"),
      m_scales(a[5], "exp_avg_scales"), v_scales(a[6], "exp_avg_sq_scales");
  const int64_t n = params.size();
  if (n == 0) return PyLong_FromLong(UNIRL_OK);
  for (const TensorList* l : {&grads, &ms, &vs, &masters, &m_scales, &v_scales})
    TORCH_CHECK_VALUE((!*l && l != &grads && l != &ms && l != &vs) || l->size() == n, l->name, " has ", l->size(), " entries for ", n,
                      " params");
  std::vector<int64_t> bases;
  if (a[7] != Py_None) {
    PyObject* seq = PySequence_Fast(a[7], "index_bases must be a sequence");
    if (!seq) throw python_error();
    const int64_t k = PySequence_Fast_GET_SIZE(seq);
    bases.resize(k);
    for (int64_t i = 0; i < k; ++i) {
      bases[i] = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq, i));
      if (bases[i] == -1 && PyErr_Occurred()) {
        Py_DECREF(seq);
        throw python_error();
      }
    }
    Py_DECREF(seq);
    TORCH_CHECK_VALUE(k == n, "index_bases has ", k, " entries for ", n, " params");
  }
  const bool bytes = (bool)m_scales;
  const at::Device device = params[0].device();
  require_device(params[0], "params[0]");
  const at::ScalarType pt = params[0].scalar_type(), gt = grads[0].scalar_type();
  const at::ScalarType st = bytes ? at::kByte : at::kFloat;
  struct unirl_adamw_params q = {};
  q.param_dtype = dtype_code(pt);
  q.grad_dtype = dtype_code(gt);
  TORCH_CHECK_TYPE(gt == pt || gt == at::kFloat, "gradients of ", at::toString(pt), " parameters must be of that type or Float; got ",
                   at::toString(gt));
  TORCH_CHECK_VALUE(!masters || pt != at::kFloat, "masters are for 16-bit params: fp32 params hold their own values");
  q.state_bits = bytes ? 8 : 32;
  q.use_master = masters ? 1 : 0;
  q.lr = number(a[8]);
  q.beta1 = number(a[9]);
  q.beta2 = number(a[10]);
  q.eps = number(a[11]);
  q.weight_decay = number(a[12]);
  q.step = integer(a[13]);
  q.seed = (uint32_t)integer(a[14]);
  const std::optional<Tensor> norm = optional_of(a[15], "grad_norm"), control = optional_of(a[18], "control");
  q.grad_norm = norm ? norm->data_ptr<float>() : nullptr;
  q.max_norm = (float)number(a[16]);
  q.skip_nonfinite = (int)integer(a[17]);
  q.control = control ? control->data_ptr() : nullptr;

  c10::hip::HIPGuard guard(device.index());
  std::vector<struct unirl_adamw_tensor> table(n);
  std::vector<Tensor> copies;
  std::vector<void*> seen;
  seen.reserve(n);
  int64_t at_element = 0;
  for (int64_t i = 0; i < n; ++i) {
    const Tensor& p = params[i];
    const int64_t k = p.numel(), blocks = (k + 255) / 256;
    check_entry(p, "params", i, k, pt, device);
    const Tensor* g = &grads[i];
    if (!g->is_contiguous()) {
      copies.push_back(g->contiguous());
      g = &copies.back();
    }
    check_entry(*g, "grads", i, k, gt, device);
    check_entry(ms[i], "exp_avgs", i, k, st, device);
    check_entry(vs[i], "exp_avg_sqs", i, k, st, device);
    auto& t = table[i];
    t = {p.data_ptr(), g->data_ptr(), ms[i].data_ptr(), vs[i].data_ptr(), nullptr, nullptr, nullptr, k, 0};
    if (masters) {
      check_entry(masters[i], "masters", i, k, at::kFloat, device);
      t.master = masters[i].data_ptr<float>();
    }
    if (bytes) {
      check_entry(m_scales[i], "exp_avg_scales", i, blocks, at::kByte, device);
      check_entry(v_scales[i], "exp_avg_sq_scales", i, blocks, at::kByte, device);
      t.exp_avg_scale = m_scales[i].data_ptr<uint8_t>();
      t.exp_avg_sq_scale = v_scales[i].data_ptr<uint8_t>();
      t.index_base = bases.empty() ? at_element : bases[i];
      at_element += blocks * 256;
    }
    if (k) seen.push_back(t.param);
  }
  std::sort(seen.begin(), seen.end());
  TORCH_CHECK_VALUE(std::adjacent_find(seen.begin(), seen.end()) == seen.end(), "the same parameter appears more than once");
  const int rc = unirl_adamw_step(table.data(), n, &q, stream_of(params[0]));
  // written behind autograd's back: whoever saved a parameter for a backward has to notice
  for (int64_t i = 0; i < n; ++i)
    if (!params[i].is_inference()) torch::autograd::impl::bump_version(params[i]);  // inference tensors have no version
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"norm", (PyCFunction)(void (*)(void))norm, METH_FASTCALL, nullptr},
    {"layer_norm", (PyCFunction)(void (*)(void))layer_norm, METH_FASTCALL, nullptr},
    {"layer_norm_bwd", (PyCFunction)(void (*)(void))layer_norm_bwd, METH_FASTCALL, nullptr},
    {"grad_norm", (PyCFunction)(void (*)(void))grad_norm, METH_FASTCALL, nullptr},
    {"adamw_step", (PyCFunction)(void (*)(void))adamw_step, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_unirl_torch_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__unirl_torch_host(void) {
  PyObject* m = PyModule_Create(&module);
  if (m) PyModule_AddIntConstant(m, "abi_version", UNIRL_ABI_VERSION);  // the header's, not the loaded library's
  return m;
}
