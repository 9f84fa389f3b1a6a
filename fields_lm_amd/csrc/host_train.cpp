// host_train.cpp — the host side of the embedding, the gated scan, orthogonalization and the Muon step (the module of
// host.cpp). Autograd functions are C++, so that the engine's thread waits for no interpreter.
#include "host_common.h"

#include <torch/csrc/Dtype.h>
#include <torch/custom_class.h>

#include <cmath>

namespace {

using namespace host;

decltype(&fl_embedding) embedding_call = nullptr;
decltype(&fl_embedding_backward_workspace_bytes) embedding_bytes = nullptr;
decltype(&fl_embedding_backward) embedding_backward_call = nullptr;
decltype(&fl_gated_scan_workspace_bytes) scan_bytes = nullptr;
decltype(&fl_gated_scan) scan_call = nullptr;
decltype(&fl_gated_scan_backward) scan_backward_call = nullptr;
decltype(&fl_orthogonalize_check) orthogonalize_check = nullptr;
decltype(&fl_orthogonalize_workspace_bytes) orthogonalize_bytes = nullptr;
decltype(&fl_orthogonalize) orthogonalize_call = nullptr;
decltype(&fl_muon_step) muon_call = nullptr;
PyObject* stock_scan_gradients = nullptr;
int64_t scan_tile = 0;

bool kernel_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }

void check_input(const Tensor& t, const char* what) {
  check_plain(t, what);
  TORCH_CHECK_TYPE(t.layout() == at::kStrided, what, " must be dense");
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), what, " has a forward-mode derivative, which is not there");
}

void check_values(const Tensor& t, const char* what) {
  check_input(t, what);
  TORCH_CHECK_TYPE(kernel_type(t.scalar_type()), what, " must be float32 or bfloat16, got ", t.scalar_type());
}

Tensor upstream(const Tensor& g) {
  if (!g.defined()) return {};
  check_plain(g, "the upstream gradients");
  return g.resolve_neg().contiguous();
}

// ------------------------------------------------------------------ embedding

struct Rows {
  int64_t padding;  // -1: none
  double scale;
  at::ScalarType type;  // of the rows
  bool masked;          // rows of padding and of tokens outside are zeros: the transpose of the gradient
};

Tensor rows_of(const Tensor& weight, const Tensor& tokens, const Rows& r) {
  const c10::DeviceGuard guard(weight.device());
  Tensor w = weight.resolve_neg();
  if (w.stride(1) != 1 && w.size(1) > 1) w = w.contiguous();
  std::vector<int64_t> shape = tokens.sizes().vec();
  shape.push_back(w.size(1));
  const Tensor out = at::empty(shape, at::TensorOptions().dtype(r.type).device(w.device()));
  check(embedding_call(address<int64_t>(tokens), tokens.numel(), address<void>(w), dtype_code(w), w.size(0), w.size(1),
                       w.stride(0), (float)r.scale, r.masked, r.padding, address<void>(out), dtype_code(out),
                       stream_of(w)),
        "fl_embedding");
  return out;
}

Tensor weight_gradient(const Tensor& grad, const Tensor& tokens, int64_t V, int64_t D, at::ScalarType type,
                       const Rows& r) {
  const c10::DeviceGuard guard(tokens.device());
  const Tensor g = upstream(grad);
  const auto options = at::TensorOptions().device(tokens.device());
  const Tensor out = at::empty({V, D}, options.dtype(type));
  const size_t bytes = embedding_bytes(tokens.numel(), V, D);
  const Tensor ws = workspace_on(tokens.device(), bytes);
  check(embedding_backward_call(address<int64_t>(tokens), tokens.numel(), address<void>(g), dtype_code(g), V, D,
                                r.padding, (float)r.scale, address<void>(out), dtype_code(out), address<void>(ws), bytes,
                                stream_of(out)),
        "fl_embedding_backward");
  return out;
}

void save_rows(AutogradContext* ctx, const Rows& r) {
  ctx->saved_data["padding"] = r.padding;
  ctx->saved_data["scale"] = r.scale;
}

Rows saved_rows(AutogradContext* ctx, at::ScalarType type, bool masked) {
  return {ctx->saved_data["padding"].toInt(), ctx->saved_data["scale"].toDouble(), type, masked};
}

// The node that an input's gradient goes to, kept beside what is saved. (The input itself is not: its values are not
// read again, and may be written before the backward pass.)
struct Target : torch::CustomClassHolder {
  std::shared_ptr<torch::autograd::Node> node;
  explicit Target(std::shared_ptr<torch::autograd::Node> n) : node(std::move(n)) {}
};

// Both directions are linear, so that each one's derivative is the other.
struct EmbeddingGrad : torch::autograd::Function<EmbeddingGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& grad, const Tensor& tokens, int64_t V, int64_t D,
                        int64_t type, const Rows& r) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({tokens});
    save_rows(ctx, r);
    ctx->saved_data["type"] = (int64_t)grad.scalar_type();
    return weight_gradient(grad, tokens, V, D, (at::ScalarType)type, r);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads);
};

struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& tokens, const Rows& r) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({tokens});
    if (weight.requires_grad())
      ctx->saved_data["target"] = c10::IValue::make_capsule(c10::make_intrusive<Target>(node_of(weight)));
    ctx->saved_data["V"] = weight.size(0);
    ctx->saved_data["D"] = weight.size(1);
    ctx->saved_data["type"] = (int64_t)weight.scalar_type();
    save_rows(ctx, r);
    return rows_of(weight, tokens, r);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const Tensor tokens = ctx->get_saved_variables()[0];
    const int64_t V = ctx->saved_data["V"].toInt(), D = ctx->saved_data["D"].toInt();
    const int64_t type = ctx->saved_data["type"].toInt();
    const Rows r = saved_rows(ctx, grads[0].scalar_type(), true);
    const auto target = ctx->saved_data.find("target");
    if (target != ctx->saved_data.end())
      check_leaves(c10::static_intrusive_pointer_cast<Target>(target->second.toCapsule())->node, "weight's");
    out[0] = at::GradMode::is_enabled() ? EmbeddingGrad::apply(grads[0], tokens, V, D, type, r)
                                        : weight_gradient(grads[0], tokens, V, D, (at::ScalarType)type, r);
    return out;
  }
};

variable_list EmbeddingGrad::backward(AutogradContext* ctx, const variable_list& grads) {
  variable_list out(6);
  if (!grads[0].defined()) return out;
  const Tensor tokens = ctx->get_saved_variables()[0];
  const Rows r = saved_rows(ctx, (at::ScalarType)ctx->saved_data["type"].toInt(), true);
  check_plain(grads[0], "the upstream gradients");
  out[0] = at::GradMode::is_enabled() ? Embedding::apply(grads[0], tokens, r) : rows_of(grads[0], tokens, r);
  return out;
}

// ------------------------------------------------------------------ gated scan

// [B, T, C] with the channels next to each other, or [B, T]
Tensor in_rows(const Tensor& t) {
  const Tensor x = t.resolve_neg();
  return x.dim() == 3 && x.size(2) > 1 && x.stride(2) != 1 ? x.contiguous() : x;
}

struct Scanned {
  Tensor out, last, starts;
};

Scanned scan(const Tensor& gate, const Tensor& drive, const Tensor& state, bool want_last, bool want_starts) {
  const c10::DeviceGuard guard(drive.device());
  const Tensor a = in_rows(gate), u = in_rows(drive), first = state.defined() ? state.resolve_neg().contiguous() : state;
  const int64_t B = u.size(0), T = u.size(1), C = u.size(2);
  const auto fp32 = at::TensorOptions().dtype(at::kFloat).device(u.device());
  Scanned r;
  r.out = at::empty({B, T, C}, fp32.dtype(u.scalar_type()));
  if (want_last) r.last = at::empty({B, C}, fp32);
  if (want_starts) r.starts = at::empty({B, (T + scan_tile - 1) / scan_tile, C}, fp32);
  const size_t bytes = scan_bytes(B, T, C, 0);
  const Tensor ws = workspace_on(u.device(), bytes);
  check(scan_call(address<void>(a), dtype_code(a), a.dim() == 2, a.stride(0), a.stride(1), address<void>(u),
                  dtype_code(u), u.stride(0), u.stride(1), B, T, C, address<float>(first), address<float>(r.last),
                  address<float>(r.starts), address<void>(r.out), address<void>(ws), bytes, stream_of(u)),
        "fl_gated_scan");
  return r;
}

variable_list scan_gradients(const Tensor& gate, const Tensor& drive, const Tensor& starts, const Tensor& g_out,
                             const Tensor& g_last, bool want_gate, bool want_state) {
  const c10::DeviceGuard guard(drive.device());
  const Tensor a = in_rows(gate), u = in_rows(drive);
  const int64_t B = u.size(0), T = u.size(1), C = u.size(2);
  const auto fp32 = at::TensorOptions().dtype(at::kFloat).device(u.device());
  const Tensor g = upstream(g_out), k = upstream(g_last);
  variable_list r(3);
  if (want_gate) r[0] = at::empty(gate.sizes(), fp32.dtype(a.scalar_type()));
  r[1] = at::empty({B, T, C}, fp32.dtype(u.scalar_type()));
  if (want_state) r[2] = at::empty({B, C}, fp32);
  const size_t bytes = scan_bytes(B, T, C, 1);
  const Tensor ws = workspace_on(u.device(), bytes);
  check(scan_backward_call(address<void>(a), dtype_code(a), a.dim() == 2, a.stride(0), a.stride(1), address<void>(u),
                           dtype_code(u), u.stride(0), u.stride(1), B, T, C, address<float>(starts), address<void>(g),
                           address<float>(k), address<void>(r[0]), address<void>(r[1]), address<float>(r[2]),
                           address<void>(ws), bytes, stream_of(u)),
        "fl_gated_scan_backward");
  return r;
}

// The gradients in operations that can be differentiated again: the function of Python that was handed over.
variable_list stock_scan(const Tensor& gate, const Tensor& drive, const Tensor& state, const Tensor& g_out,
                         const Tensor& g_last) {
  const PyGILState_STATE gil = PyGILState_Ensure();
  const auto wrap = [](const Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); };
  PyObject* args = Py_BuildValue("(NNNNN)", wrap(gate), wrap(drive), wrap(state), wrap(g_out), wrap(g_last));
  PyObject* got = args ? PyObject_CallObject(stock_scan_gradients, args) : nullptr;
  Py_XDECREF(args);
  variable_list out(3);
  const bool fine = got && PyTuple_Check(got) && PyTuple_GET_SIZE(got) == 3;
  if (fine)
    for (int i = 0; i < 3; ++i)
      if (THPVariable_Check(PyTuple_GET_ITEM(got, i))) out[i] = THPVariable_Unpack(PyTuple_GET_ITEM(got, i));
  Py_XDECREF(got);
  if (!fine) {
    python_error e;  // carries the Python exception to whoever asked for the gradients
    e.persist();
    PyGILState_Release(gil);
    throw e;
  }
  PyGILState_Release(gil);
  return out;
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& gate, const Tensor& drive,
                               const std::optional<Tensor>& first, bool return_state) {
    const Tensor state = first ? *first : Tensor();
    const Scanned r = scan(gate, drive, state, return_state, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({gate, drive, state, r.starts});
    variable_list out = {r.out};
    if (return_state) out.push_back(r.last);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &gate = saved[0], &drive = saved[1], &state = saved[2], &starts = saved[3];
    const Tensor g = grads[0], k = grads.size() > 1 ? grads[1] : Tensor();
    variable_list out(4);
    if (!g.defined() && !k.defined()) return out;
    for (const Tensor& t : {gate, drive, state})
      if (t.defined() && t.requires_grad()) check_leaves(node_of(t), "scan's inputs'");
    const bool of_state = state.defined() && state.requires_grad();
    const variable_list r = at::GradMode::is_enabled()
                                ? stock_scan(gate, drive, state, g, k)
                                : scan_gradients(gate, drive, starts, g, k, gate.requires_grad(), of_state);
    for (int i = 0; i < (state.defined() ? 3 : 2); ++i) out[i] = r[i];
    return out;
  }
};

// ------------------------------------------------------------------ matrices

struct Matrices {
  std::vector<int64_t> rows, cols;
  explicit Matrices(const std::vector<at::IntArrayRef>& shapes, const char* what) {
    for (size_t i = 0; i < shapes.size(); ++i) {
      TORCH_CHECK_VALUE(shapes[i].size() == 2, what, " must be matrices, number ", i, " has the shape ", shapes[i]);
      rows.push_back(shapes[i][0]);
      cols.push_back(shapes[i][1]);
    }
  }
};

void check_steps(long long steps, double a, double b, double c, double eps) {
  TORCH_CHECK_VALUE(steps >= 1 && steps <= 64, "steps must be 1 to 64, got ", steps);
  TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(eps), "eps must be finite and 0 or more, got ", eps);
  TORCH_CHECK_VALUE(orthogonalize_check((int)steps, a, b, c) == FL_OK, "with the coefficients (", a, ", ", b, ", ", c,
                    ") ", steps, " steps can bring singular values, or a step's factor, past 1024");
}

}  // namespace

// embedding(tokens, weight, scale, padding index or -1, type or None) -> rows
PyObject* host_embedding(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *first, *second, *dtype;
  double scale;
  long long padding;
  if (!PyArg_ParseTuple(args, "OOdLO", &first, &second, &scale, &padding, &dtype)) return nullptr;
  TORCH_CHECK_TYPE(THPVariable_Check(first) && THPVariable_Check(second), "tokens and weight must be tensors");
  const Tensor &tokens = THPVariable_Unpack(first), &weight = THPVariable_Unpack(second);
  check_input(tokens, "tokens");
  check_values(weight, "the weight");
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong, "tokens must be int64, got ", tokens.scalar_type());
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.numel() > 0, "the weight must be [V, D], got ", weight.sizes());
  TORCH_CHECK_VALUE(std::isfinite(scale), "scale must be finite, got ", scale);
  TORCH_CHECK_VALUE(padding >= -1 && padding < weight.size(0), "padding_idx must be one of the weight's ",
                    weight.size(0), " rows, got ", padding);
  at::ScalarType type = weight.scalar_type();
  if (dtype != Py_None) {
    TORCH_CHECK_TYPE(THPDtype_Check(dtype), "dtype must be a torch.dtype");
    type = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
    TORCH_CHECK_TYPE(kernel_type(type), "dtype must be float32 or bfloat16, got ", type);
  }
  TORCH_CHECK(weight.is_cuda(), "embedding requires a ROCm (cuda) device");
  check_not_traced("embedding");
  TORCH_CHECK_VALUE(tokens.device() == weight.device(), "tokens and weight must be on one device");
  const Tensor t = tokens.resolve_neg().contiguous();
  const Rows r = {padding, scale, type, false};
  if (at::GradMode::is_enabled() && weight.requires_grad()) return THPVariable_Wrap(Embedding::apply(weight, t, r));
  return THPVariable_Wrap(rows_of(weight, t, r));
  END_HANDLE_TH_ERRORS
}

// gated_scan(gate, drive, state or None, return state) -> (all states, the last one or None)
PyObject* host_gated_scan(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *first, *second, *third;
  int return_state;
  if (!PyArg_ParseTuple(args, "OOOp", &first, &second, &third, &return_state)) return nullptr;
  TORCH_CHECK_TYPE(THPVariable_Check(first) && THPVariable_Check(second) &&
                       (third == Py_None || THPVariable_Check(third)),
                   "gate, drive and state_in must be tensors");
  const Tensor &drive = THPVariable_Unpack(second), state = third == Py_None ? Tensor() : THPVariable_Unpack(third);
  Tensor gate = THPVariable_Unpack(first);
  check_values(gate, "gate");
  check_values(drive, "drive");
  TORCH_CHECK_VALUE(drive.dim() == 3, "drive must be [B, T, C], got ", drive.sizes());
  const int64_t B = drive.size(0), T = drive.size(1), C = drive.size(2);
  const bool token = (gate.dim() == 2 || (gate.dim() == 3 && gate.size(2) == 1)) && gate.size(0) == B && gate.size(1) == T;
  TORCH_CHECK_VALUE(token || gate.sizes() == drive.sizes(), "gate must be the drive's ", drive.sizes(),
                    ", or one value a token, got ", gate.sizes());
  if (state.defined()) {
    check_input(state, "state_in");
    TORCH_CHECK_TYPE(state.scalar_type() == at::kFloat, "state_in must be float32, got ", state.scalar_type());
    TORCH_CHECK_VALUE(state.dim() == 2 && state.size(0) == B && state.size(1) == C, "state_in must be [", B, ", ", C,
                      "], got ", state.sizes());
  }
  TORCH_CHECK(drive.is_cuda(), "gated_scan requires a ROCm (cuda) device");
  check_not_traced("gated_scan");
  TORCH_CHECK_VALUE(gate.device() == drive.device() && (!state.defined() || state.device() == drive.device()),
                    "gate, drive and state_in must be on one device");
  if (gate.dim() == 3 && gate.size(2) == 1 && C != 1) gate = gate.squeeze(2);
  variable_list out;
  const bool grad = at::GradMode::is_enabled() &&
                    (gate.requires_grad() || drive.requires_grad() || (state.defined() && state.requires_grad()));
  if (drive.numel() == 0) {  // no step or no channel: nothing changes the state
    const Tensor none = (gate.dim() == 2 ? gate.unsqueeze(2) : gate).to(drive.scalar_type()) * 0;
    out = {drive + none};  // (on the graph of both)
    if (return_state)
      out.push_back(state.defined() ? state.clone()
                                    : at::zeros({B, C}, at::TensorOptions().dtype(at::kFloat).device(drive.device())));
  } else if (grad) {
    out = GatedScan::apply(gate, drive, state.defined() ? std::optional<Tensor>(state) : std::nullopt,
                           (bool)return_state);
  } else {
    const Scanned r = scan(gate, drive, state, return_state, false);
    out = {r.out};
    if (return_state) out.push_back(r.last);
  }
  PyObject* all = THPVariable_Wrap(out[0]);
  return Py_BuildValue("(NN)", all, return_state ? THPVariable_Wrap(out[1]) : Py_NewRef(Py_None));
  END_HANDLE_TH_ERRORS
}

// orthogonalize(matrices [..., M, N], steps, a, b, c, eps) -> the same shape
PyObject* host_orthogonalize(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject* first;
  long long steps;
  double a, b, c, eps;
  if (!PyArg_ParseTuple(args, "OLdddd", &first, &steps, &a, &b, &c, &eps)) return nullptr;
  TORCH_CHECK_TYPE(THPVariable_Check(first), "x must be a tensor");
  const Tensor& x = THPVariable_Unpack(first);
  check_values(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 2, "x must be [..., M, N], got ", x.sizes());
  check_steps(steps, a, b, c, eps);
  TORCH_CHECK(x.is_cuda(), "orthogonalize requires a ROCm (cuda) device");
  check_not_traced("orthogonalize");
  const c10::DeviceGuard guard(x.device());
  const Tensor in = x.detach().resolve_neg().contiguous();
  const Tensor out = at::empty(in.sizes(), in.options());
  const int64_t rows = x.size(-2), cols = x.size(-1), n = rows * cols ? x.numel() / (rows * cols) : 0;
  if (n) {
    const std::vector<int64_t> all_rows(n, rows), all_cols(n, cols);
    std::vector<void*> from(n), to(n);
    for (int64_t i = 0; i < n; ++i) {
      from[i] = static_cast<char*>(in.data_ptr()) + i * rows * cols * in.element_size();
      to[i] = static_cast<char*>(out.data_ptr()) + i * rows * cols * in.element_size();
    }
    const size_t bytes = orthogonalize_bytes(n, all_rows.data(), all_cols.data());
    const Tensor ws = workspace_on(x.device(), bytes);
    check(orthogonalize_call(n, from.data(), dtype_code(in), all_rows.data(), all_cols.data(), (int)steps, a, b, c, eps,
                             to.data(), address<void>(ws), bytes, stream_of(x)),
          "fl_orthogonalize");
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// check_steps(steps, a, b, c, eps): raises where a call would
PyObject* host_check_steps(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  long long steps;
  double a, b, c, eps;
  if (!PyArg_ParseTuple(args, "Ldddd", &steps, &a, &b, &c, &eps)) return nullptr;
  check_steps(steps, a, b, c, eps);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// muon_step(parameters, gradients, buffers, lr (a number or a tensor), momentum, nesterov, weight decay, steps, a, b, c,
// eps, whether the rate matches AdamW's update, gradient scale or None)
PyObject* host_muon_step(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *params, *grads, *buffers, *lr, *grad_scale;
  double momentum, decay, a, b, c, eps;
  int nesterov, match;
  long long steps;
  if (!PyArg_ParseTuple(args, "OOOOdpdLddddpO", &params, &grads, &buffers, &lr, &momentum, &nesterov, &decay, &steps, &a,
                        &b, &c, &eps, &match, &grad_scale))
    return nullptr;
  const Tensor& first = first_of(params, "parameters");
  const at::Device device = first.device();
  const at::ScalarType type = first.scalar_type();
  TORCH_CHECK_TYPE(kernel_type(type), "parameters must be float32 or bfloat16, got ", type);
  const auto as_long = [&](PyObject* o) {
    return (!PyList_Check(o) && !PyTuple_Check(o)) || PySequence_Fast_GET_SIZE(o) == PySequence_Fast_GET_SIZE(params);
  };
  TORCH_CHECK_VALUE(as_long(grads) && as_long(buffers), "one gradient and one momentum buffer per parameter");
  check_steps(steps, a, b, c, eps);
  TORCH_CHECK(device.is_cuda(), "muon_step requires a ROCm (cuda) device");
  check_not_traced("muon_step");
  const TensorList p(params, "parameters", device, {type});
  const int64_t n = (int64_t)p.size();
  const TensorList g(grads, "gradients", device, {type}, &p.counts, 1, true);
  const TensorList m(buffers, "momentum buffers", device, {at::kFloat}, &p.counts);
  const Matrices shapes(p.shapes, "parameters");
  for (int64_t i = 0; i < n; ++i)
    TORCH_CHECK_VALUE(p.shapes[i] == g.shapes[i], "gradient ", i, " has the shape ", g.shapes[i], ", its parameter ",
                      p.shapes[i]);
  Ranges written;
  const size_t size = type == at::kFloat ? 4 : 2;
  merge(written, ranges_of(p, size));
  merge(written, ranges_of(m, 4));
  TORCH_CHECK_VALUE(!overlap(written), "parameters or momentum buffers share memory");
  TORCH_CHECK_VALUE(!meet(written, ranges_of(g, size)), "a gradient shares memory with a parameter or a momentum buffer");
  const Tensor scale = device_value(grad_scale, "grad_scale", device);
  const Tensor lr_at = THPVariable_Check(lr) ? device_value(lr, "lr", device) : Tensor();
  const double lr_value = lr_at.defined() ? 0.0 : PyFloat_AsDouble(lr);
  if (PyErr_Occurred()) return nullptr;
  std::vector<double> rate(n);
  for (int64_t i = 0; i < n; ++i) {
    const double r = (double)shapes.rows[i], k = (double)shapes.cols[i];
    rate[i] = match ? 0.2 * std::sqrt(std::max(r, k)) : std::sqrt(std::max(1.0, k > 0 ? r / k : 1.0));
  }
  const c10::DeviceGuard guard(device);
  const size_t bytes = orthogonalize_bytes(n, shapes.rows.data(), shapes.cols.data());
  const Tensor ws = workspace_on(device, bytes);
  check(muon_call(n, p.addresses.data(), g.addresses.data(), type == at::kBFloat16 ? FL_DTYPE_BF16 : FL_DTYPE_F32,
                  reinterpret_cast<float* const*>(m.addresses.data()), shapes.rows.data(), shapes.cols.data(), lr_value,
                  address<float>(lr_at), rate.data(), momentum, nesterov, decay, (int)steps, a, b, c, eps,
                  address<float>(scale), address<void>(ws), bytes, stream_of(first)),
        "fl_muon_step");
  for (PyObject* list : {params, buffers}) count_writes(list);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// bind_train(addresses of the library's entry points, the steps of a scan's tile, the scan's differentiable gradients)
PyObject* host_bind_train(PyObject*, PyObject* args) {
  unsigned long long k[10];
  long long tile;
  PyObject* stock;
  if (!PyArg_ParseTuple(args, "KKKKKKKKKKLO", k, k + 1, k + 2, k + 3, k + 4, k + 5, k + 6, k + 7, k + 8, k + 9, &tile,
                        &stock))
    return nullptr;
  embedding_call = reinterpret_cast<decltype(embedding_call)>(k[0]);
  embedding_bytes = reinterpret_cast<decltype(embedding_bytes)>(k[1]);
  embedding_backward_call = reinterpret_cast<decltype(embedding_backward_call)>(k[2]);
  scan_bytes = reinterpret_cast<decltype(scan_bytes)>(k[3]);
  scan_call = reinterpret_cast<decltype(scan_call)>(k[4]);
  scan_backward_call = reinterpret_cast<decltype(scan_backward_call)>(k[5]);
  orthogonalize_check = reinterpret_cast<decltype(orthogonalize_check)>(k[6]);
  orthogonalize_bytes = reinterpret_cast<decltype(orthogonalize_bytes)>(k[7]);
  orthogonalize_call = reinterpret_cast<decltype(orthogonalize_call)>(k[8]);
  muon_call = reinterpret_cast<decltype(muon_call)>(k[9]);
  scan_tile = tile;
  Py_INCREF(stock);
  Py_XDECREF(stock_scan_gradients);
  stock_scan_gradients = stock;
  Py_RETURN_NONE;
}
