// The row operators (group norm, gated feed-forward) as autograd nodes in C++, part of ss_conv/_host.
//
// A pass over a few thousand rows is bound by the host that queues it: a node written in Python costs 15 us forward and 55 to 65 us
// backward around its two library calls, a tenth of that here.  Arguments are checked here as well.
#include "ssc_host_rows.h"

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <ATen/DeviceGuard.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>

#include <memory>
#include <optional>
#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/ssconv_b200.h"

namespace {

using at::Tensor;

// The library's functions; another build of it may be put in their place (row_operators).
struct {
  decltype(&ssc_last_error) last_error = &ssc_last_error;
  decltype(&ssc_group_norm_scratch_bytes) norm_bytes = &ssc_group_norm_scratch_bytes;
  decltype(&ssc_group_norm_fwd) norm_fwd = &ssc_group_norm_fwd;
  decltype(&ssc_group_norm_bwd) norm_bwd = &ssc_group_norm_bwd;
  decltype(&ssc_gated_ff_scratch_bytes) ff_bytes = &ssc_gated_ff_scratch_bytes;
  decltype(&ssc_gated_ff_fwd) ff_fwd = &ssc_gated_ff_fwd;
  decltype(&ssc_gated_ff_bwd) ff_bwd = &ssc_gated_ff_bwd;
} library;

void check(int rc) {
  if (rc == SSC_OK) return;
  const std::string what = library.last_error();
  TORCH_CHECK_VALUE(rc != SSC_ERR_INVALID, "ssconv_b200: ", what);
  TORCH_CHECK(false, "ssconv_b200 (code ", rc, "): ", what);
}

int code_of(at::ScalarType t) { return t == at::kFloat ? SSC_PREC_FP32 : t == at::kHalf ? SSC_PREC_F16 : t == at::kBFloat16 ? SSC_PREC_BF16 : -1; }
void *stream_of(const Tensor &t) { return (void *)c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
template <class T>
T *pointer(const Tensor &t) { return t.defined() ? (T *)t.data_ptr() : nullptr; }
Tensor bytes_for(const Tensor &like, size_t n) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }
// Contiguous, and at an address the copy engine takes.
Tensor aligned(const Tensor &t) {
  const Tensor c = t.contiguous();
  return (uintptr_t)c.data_ptr() % 16 == 0 ? c : c.clone();
}
std::string shape_of(const Tensor &t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
void check_rows(const Tensor &x) {
  TORCH_CHECK(x.is_cuda(), "ssconv_b200 runs on CUDA tensors only (got a ", c10::DeviceTypeName(x.device().type(), true), " tensor)");
  TORCH_CHECK_TYPE(code_of(x.scalar_type()) >= 0, "features must be float32, float16 or bfloat16 (got ", x.scalar_type(), ")");
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(0) <= (int64_t)1 << 30, "features must be [N, C] with at most 2^30 rows (got ", shape_of(x), ")");
}
bool recorded(std::initializer_list<const Tensor *> all) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : all)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// Recording into a CUDA graph: gradients of a leaf that an earlier result of the default stream still holds on to would be added up on that
// stream, which cannot take part: the backward pass would end the process.  So the call is refused, however far behind its arguments such a
// leaf (or another part of a graph of the default stream) lies.
void recordable(std::initializer_list<const Tensor *> all, const Tensor &x) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const c10::Stream ordinary = c10::cuda::getDefaultCUDAStream(x.device().index());
  std::vector<torch::autograd::Node *> next;
  std::unordered_set<torch::autograd::Node *> seen;
  auto look = [&](torch::autograd::Node *f) {
    if (f != nullptr && seen.insert(f).second) next.push_back(f);
  };
  std::vector<std::shared_ptr<torch::autograd::Node>> leaves;       // (a leaf has its node only as long as somebody holds it)
  for (const Tensor *t : all) {
    if (!t->defined() || !t->requires_grad()) continue;
    leaves.push_back(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    look(leaves.back().get());
  }
  while (!next.empty()) {
    torch::autograd::Node *f = next.back();
    next.pop_back();
    TORCH_CHECK(!(f->stream() == ordinary), "a result computed before this recording still holds the gradient graph of the same tensors: drop it (its loss) before recording");
    for (const torch::autograd::Edge &e : f->next_edges()) look(e.function.get());
  }
}
// A tangent would be dropped without a word: the operators have no forward-mode derivative.
void no_tangents(const char *what, std::initializer_list<const Tensor *> all) {
  for (const Tensor *t : all)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what, ": forward-mode derivatives are not available");
}
void first_gradient(const char *what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": gradients of gradients are not available (create_graph)");
}

// ------------------------------------------------------------------------------------------ group norm
struct Norm {
  int64_t n_field, n_scalar, n_group, n_gate, scalar_act, gate_act;
  double eps;
};

Tensor norm_forward(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &offsets, const Tensor &table, const Tensor &status, const Norm &k,
                    at::ScalarType out_type, Tensor &stats) {
  const c10::DeviceGuard guard(x.device());
  const int64_t n = x.size(0), c = x.size(1), batch = offsets.size(0) - 1;
  const Tensor out = at::empty({n, c - k.n_gate}, x.options().dtype(out_type));
  stats = at::empty({batch, k.n_group, 2}, x.options().dtype(at::kFloat));
  const size_t bytes = library.norm_bytes((int)batch, (int)k.n_group, 0, 0);
  const Tensor scratch = bytes_for(x, bytes);
  check(library.norm_fwd(x.data_ptr(), code_of(x.scalar_type()), (int)n, (int)c, pointer<int32_t>(offsets), (int)batch, pointer<int32_t>(table), (int)k.n_field,
                         (int)k.n_scalar, (int)k.n_group, (int)k.n_gate, pointer<float>(weight), pointer<float>(bias), (float)k.eps, (int)k.scalar_act,
                         (int)k.gate_act, out.data_ptr(), code_of(out_type), pointer<float>(stats), pointer<int32_t>(status), scratch.data_ptr(), bytes,
                         stream_of(x)));
  return out;
}

// A node takes what may be absent as an optional: absent ones have no edge, the others are numbered without them.
typedef std::optional<Tensor> Maybe;
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }
// What the process keeps (channel tables, the status word) goes along as it is, not as a saved variable: those are checked for changes in place,
// and clearing the status word is one.
void keep(torch::autograd::AutogradContext *ctx, const char *name, const Tensor &t) { ctx->saved_data[name] = t; }

struct NormNode : torch::autograd::Function<NormNode> {
  static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Maybe &maybe_weight, const Maybe &maybe_bias, const Tensor &offsets,
                        const Tensor &table, const Tensor &status, const Norm &k) {
    const Tensor weight = maybe_weight.value_or(Tensor()), bias = maybe_bias.value_or(Tensor());
    Tensor stats;
    const Tensor y = norm_forward(x, weight, bias, offsets, table, status, k, x.scalar_type(), stats);
    ctx->save_for_backward({x, weight, bias, offsets, stats});
    keep(ctx, "table", table);
    keep(ctx, "status", status);
    ctx->saved_data["k"] = std::vector<int64_t>{k.n_field, k.n_scalar, k.n_group, k.n_gate, k.scalar_act, k.gate_act};
    ctx->saved_data["eps"] = k.eps;
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    first_gradient("group_norm");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &offsets = saved[3], &stats = saved[4];
    const Tensor table = ctx->saved_data["table"].toTensor(), status = ctx->saved_data["status"].toTensor();
    if (!grads[0].defined()) return torch::autograd::variable_list(7);
    const std::vector<int64_t> k = ctx->saved_data["k"].toIntVector();
    const c10::DeviceGuard guard(x.device());
    const Tensor gy = aligned(grads[0]);
    const int64_t n = x.size(0), c = x.size(1), batch = offsets.size(0) - 1;
    const Tensor gx = at::empty_like(x);
    const Tensor gw = at::empty({k[0]}, stats.options()), gb = at::empty({k[1]}, stats.options());
    const size_t bytes = library.norm_bytes((int)batch, (int)k[2], (int)k[0], (int)k[1]);
    const Tensor scratch = bytes_for(x, bytes);
    check(library.norm_bwd(x.data_ptr(), gy.data_ptr(), code_of(x.scalar_type()), (int)n, (int)c, pointer<int32_t>(offsets), (int)batch, pointer<int32_t>(table),
                           (int)k[0], (int)k[1], (int)k[2], (int)k[3], pointer<float>(weight), pointer<float>(bias), (float)ctx->saved_data["eps"].toDouble(), (int)k[4],
                           (int)k[5], pointer<float>(stats), gx.data_ptr(), pointer<float>(gw), pointer<float>(gb), pointer<int32_t>(status), scratch.data_ptr(), bytes,
                           stream_of(x)));
    const bool w = weight.defined() && ctx->needs_input_grad(1), b = bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1);
    return {gx, w ? gw : Tensor(), b ? gb : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

void check_parameter(const char *name, const Tensor &p, int64_t size, const Tensor &x) {
  if (p.defined())
    TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == size && p.device() == x.device() && p.is_floating_point(), name, " must hold ", size, " floating point values on ",
                      x.device(), " (got ", p.scalar_type(), " ", shape_of(p), " on ", p.device(), ")");
}

Tensor norm(const Tensor &features, const Tensor &weight_in, const Tensor &bias_in, const Tensor &offsets_in, const Tensor &table, const Tensor &status, const Norm &k,
            int64_t channels, at::ScalarType out_type) {
  check_rows(features);
  TORCH_CHECK_VALUE(features.size(1) == channels, "features must be [N, ", channels, "] (got ", shape_of(features), ")");
  TORCH_CHECK_VALUE(offsets_in.dim() == 1 && offsets_in.size(0) >= 2 && offsets_in.scalar_type() == at::kInt && offsets_in.device() == features.device(),
                    "offsets must be int32 [samples + 1] on ", features.device(), " (got ", offsets_in.scalar_type(), " ", shape_of(offsets_in), " on ",
                    offsets_in.device(), ")");
  check_parameter("weight", weight_in, k.n_field, features);
  check_parameter("bias", bias_in, k.n_scalar, features);
  no_tangents("group_norm", {&features, &weight_in, &bias_in});
  const c10::DeviceGuard guard(features.device());
  const Tensor x = aligned(features), offsets = offsets_in.contiguous();
  const Tensor weight = weight_in.defined() ? weight_in.to(at::kFloat).contiguous() : weight_in, bias = bias_in.defined() ? bias_in.to(at::kFloat).contiguous() : bias_in;
  if (recorded({&x, &weight, &bias})) {
    recordable({&features, &weight_in, &bias_in}, features);
    const Tensor y = NormNode::apply(x, maybe(weight), maybe(bias), offsets, table, status, k);
    return out_type == y.scalar_type() ? y : y.to(out_type);
  }
  Tensor stats;
  return norm_forward(x, weight, bias, offsets, table, status, k, out_type, stats);
}

// ------------------------------------------------------------------------------------------ gated feed-forward
Tensor ff_forward(const Tensor &x, const Tensor &w_in, const Tensor &w_out, const Tensor &b_in, const Tensor &b_out, const Tensor &residual, const Tensor &status, int64_t act) {
  const c10::DeviceGuard guard(x.device());
  const int type = code_of(x.scalar_type()), n = (int)x.size(0), c = (int)x.size(1), hidden = (int)w_out.size(1), c_out = (int)w_out.size(0);
  const Tensor out = at::empty({n, c_out}, x.options());
  const size_t bytes = library.ff_bytes(type, n, c, hidden, c_out, 0);
  const Tensor scratch = bytes_for(x, bytes);
  check(library.ff_fwd(x.data_ptr(), type, n, c, hidden, c_out, w_in.data_ptr(), w_out.data_ptr(), pointer<void>(b_in), pointer<void>(b_out), pointer<void>(residual),
                       (int)act, out.data_ptr(), pointer<int32_t>(status), scratch.data_ptr(), bytes, stream_of(x)));
  return out;
}

struct FfNode : torch::autograd::Function<FfNode> {
  static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &w_in, const Tensor &w_out, const Maybe &b_in, const Maybe &b_out,
                        const Maybe &residual, const Tensor &status, int64_t act) {
    const Tensor bias = b_in.value_or(Tensor());
    const Tensor y = ff_forward(x, w_in, w_out, bias, b_out.value_or(Tensor()), residual.value_or(Tensor()), status, act);
    ctx->save_for_backward({x, w_in, w_out, bias});
    keep(ctx, "status", status);
    ctx->saved_data["act"] = act;
    ctx->saved_data["has"] = (b_in.has_value() ? 1 : 0) | (b_out.has_value() ? 2 : 0) | (residual.has_value() ? 4 : 0);
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    first_gradient("gated_feedforward");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w_in = saved[1], &w_out = saved[2], &b_in = saved[3];
    const Tensor status = ctx->saved_data["status"].toTensor();
    torch::autograd::variable_list out(8);
    if (!grads[0].defined()) return out;
    const c10::DeviceGuard guard(x.device());
    const Tensor gy = grads[0].contiguous();
    const int type = code_of(x.scalar_type()), n = (int)x.size(0), c = (int)x.size(1), hidden = (int)w_out.size(1), c_out = (int)w_out.size(0);
    const int64_t has = ctx->saved_data["has"].toInt();
    bool any = false;
    size_t edge = 0;
    for (size_t i = 0; i < 6; ++i) {
      if (i >= 3 && !(has >> (i - 3) & 1)) continue;
      if (!ctx->needs_input_grad(edge++)) continue;
      if (i == 5) {
        out[5] = gy;
        continue;
      }
      any = true;
      out[i] = i == 0 ? at::empty_like(x) : i == 1 ? at::empty_like(w_in) : i == 2 ? at::empty_like(w_out) : i == 3 ? at::empty({2, hidden}, x.options()) : at::empty({c_out}, x.options());
    }
    if (!any) return out;
    const size_t bytes = library.ff_bytes(type, n, c, hidden, c_out, 1);
    const Tensor scratch = bytes_for(x, bytes);
    check(library.ff_bwd(x.data_ptr(), gy.data_ptr(), type, n, c, hidden, c_out, w_in.data_ptr(), w_out.data_ptr(), pointer<void>(b_in), (int)ctx->saved_data["act"].toInt(),
                         pointer<void>(out[0]), pointer<void>(out[1]), pointer<void>(out[2]), pointer<void>(out[3]), pointer<void>(out[4]), pointer<int32_t>(status),
                         scratch.data_ptr(), bytes, stream_of(x)));
    return out;
  }
};

Tensor feedforward(const Tensor &x, const Tensor &w_in, const Tensor &w_out, const Tensor &b_in, const Tensor &b_out, const Tensor &residual, const Tensor &status,
                   int64_t act) {
  check_rows(x);
  TORCH_CHECK_VALUE(w_in.dim() == 3 && w_out.dim() == 2, "features must be [N, C], weight_in [2, H, C] and weight_out [C_out, H] (got ", shape_of(x), ", ", shape_of(w_in), ", ",
                    shape_of(w_out), ")");
  const int64_t c = x.size(1), hidden = w_in.size(1), c_out = w_out.size(0);
  auto wants = [&](const char *name, const Tensor &t, std::initializer_list<int64_t> shape) {
    if (t.defined())
      TORCH_CHECK_VALUE(t.sizes() == at::IntArrayRef(shape) && t.scalar_type() == x.scalar_type() && t.device() == x.device(), name, " must be ", x.scalar_type(), " ",
                        at::IntArrayRef(shape), " on ", x.device(), " (got ", t.scalar_type(), " ", shape_of(t), " on ", t.device(), ")");
  };
  wants("weight_in", w_in, {2, hidden, c});
  wants("weight_out", w_out, {c_out, hidden});
  wants("bias_in", b_in, {2, hidden});
  wants("bias_out", b_out, {c_out});
  wants("residual", residual, {x.size(0), c_out});
  no_tangents("gated_feedforward", {&x, &w_in, &w_out, &b_in, &b_out, &residual});
  auto flat = [](const Tensor &t) { return t.defined() ? t.contiguous() : t; };
  const Tensor a = flat(x), b = flat(w_in), d = flat(w_out), e = flat(b_in), f = flat(b_out), g = flat(residual);
  if (!recorded({&a, &b, &d, &e, &f, &g})) return ff_forward(a, b, d, e, f, g, status, act);
  recordable({&x, &w_in, &w_out, &b_in, &b_out, &residual}, x);
  return FfNode::apply(a, b, d, maybe(e), maybe(f), maybe(g), status, act);
}

// ------------------------------------------------------------------------------------------ Python
bool take(PyObject *o, Tensor &t) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  t = THPVariable_Unpack(o);
  return true;
}

}  // namespace

// group_norm(x, weight, bias, offsets, table, status, (channels, n_field, n_scalar, n_group, n_gate), eps, scalar_act, gate_act, out dtype)
PyObject *ssc_py_group_norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor t[6];
  bool ok = n == 11 && PyTuple_Check(args[6]) && PyTuple_GET_SIZE(args[6]) == 5 && THPDtype_Check(args[10]);
  for (int i = 0; ok && i < 6; ++i) ok = take(args[i], t[i]);
  TORCH_CHECK_TYPE(ok && t[0].defined() && t[3].defined() && t[4].defined(), "group_norm: wrong arguments");
  int64_t v[5];
  for (int i = 0; i < 5; ++i) v[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(args[6], i));
  const Norm k = {v[1], v[2], v[3], v[4], PyLong_AsLongLong(args[8]), PyLong_AsLongLong(args[9]), PyFloat_AsDouble(args[7])};
  if (PyErr_Occurred()) throw python_error();
  const at::ScalarType out = ((THPDtype *)args[10])->scalar_type;
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    y = norm(t[0], t[1], t[2], t[3], t[4], t[5], k, v[0], out);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// gated_ff(x, w_in, w_out, b_in, b_out, residual, status, act)
PyObject *ssc_py_gated_ff(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor t[7];
  bool ok = n == 8;
  for (int i = 0; ok && i < 7; ++i) ok = take(args[i], t[i]);
  TORCH_CHECK_TYPE(ok && t[0].defined() && t[1].defined() && t[2].defined(), "gated_ff: wrong arguments");
  const int64_t act = PyLong_AsLongLong(args[7]);
  if (PyErr_Occurred()) throw python_error();
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    y = feedforward(t[0], t[1], t[2], t[3], t[4], t[5], t[6], act);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// row_operators(addresses): the functions of another build of the library, in the order of the structure above.
PyObject *ssc_py_row_operators(PyObject *, PyObject *const *args, Py_ssize_t n) {
  void *p[7];
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "row_operators: seven addresses");
    return nullptr;
  }
  for (int i = 0; i < 7; ++i) p[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred()) return nullptr;
  library.last_error = (decltype(library.last_error))p[0];
  library.norm_bytes = (decltype(library.norm_bytes))p[1];
  library.norm_fwd = (decltype(library.norm_fwd))p[2];
  library.norm_bwd = (decltype(library.norm_bwd))p[3];
  library.ff_bytes = (decltype(library.ff_bytes))p[4];
  library.ff_fwd = (decltype(library.ff_fwd))p[5];
  library.ff_bwd = (decltype(library.ff_bwd))p[6];
  Py_RETURN_NONE;
}
