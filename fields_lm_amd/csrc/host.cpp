// host.cpp — the host side of calls whose cost in Python is more than their kernels': a module of CPython's and
// PyTorch's headers, no device code.
//
// token_logprobs: the whole of the call (checks, where the rows are, outputs, autograd). With a gradient it is an
// autograd function of C++, so that the engine's thread waits for no interpreter: 64 rows with entropy and five
// alternatives take 9 us a call (15.7 from Python), forward and gradient of 8 rows 49, with entropy and alternatives 67
// (110 from Python; an operator of PyTorch's own and its gradient 46).
//
// grad_norm, adamw_step: their lists of tensors are read in one pass and without a Python object per attribute. A step
// reads some twenty attributes of each of a model's hundreds of tensors: through Python's accessors that is 1.2 us a
// tensor.
//
// The calls of host_train.cpp are this module's too.
#include "host_common.h"

namespace {

using namespace host;

// The library's entry points, which the loader of the library hands over, and the stock form of the gradient.
decltype(&fl_token_logprobs_workspace_bytes) workspace_bytes = nullptr;
decltype(&fl_token_logprobs) logprobs_call = nullptr;
decltype(&fl_token_logprobs_backward) logprobs_backward_call = nullptr;
decltype(&fl_grad_norm_workspace_bytes) norm_bytes = nullptr;
decltype(&fl_grad_norm) norm_call = nullptr;
decltype(&fl_adamw_workspace_bytes) adamw_bytes = nullptr;
decltype(&fl_adamw_step) adamw_call = nullptr;
PyObject* stock_gradient = nullptr;

constexpr int64_t kMaxTop = 64, kMaxVocab = (int64_t)1 << 23, kStateBlock = 256;
constexpr double kMinTemperature = 0x1p-20, kMaxTemperature = 0x1p20;

struct Grid {
  int64_t outer, inner, stride_outer, stride_inner;
};

// The first `dims` dimensions of t as outer x inner with their strides; nothing where two do not do.
std::optional<Grid> grid_of(const Tensor& t, int64_t dims) {
  int64_t size[2] = {1, 1}, stride[2] = {0, 0};
  int n = 0;
  for (int64_t d = 0; d < dims; ++d) {
    const int64_t len = t.size(d), step = t.stride(d);
    if (len == 1) continue;
    if (n > 0 && stride[n - 1] == len * step) {  // dimensions that step as one
      size[n - 1] *= len;
      stride[n - 1] = step;
    } else if (n == 2) {
      return std::nullopt;
    } else {
      size[n] = len;
      stride[n++] = step;
    }
  }
  if (n == 2) return Grid{size[0], size[1], stride[0], stride[1]};
  return Grid{1, size[0], 0, stride[0]};
}

// Logits and tokens seen as the same outer x inner rows; what does not step like that is copied.
struct Located {
  Tensor logits, tokens;
  Grid at;
  int64_t token_outer, token_inner;
};

Located locate(const Tensor& logits, const Tensor& tokens) {
  const int64_t dims = tokens.dim(), n = tokens.numel();
  Located r = {logits, tokens, {}, 0, 0};
  if (r.logits.size(-1) > 1 && r.logits.stride(-1) != 1) r.logits = r.logits.contiguous();
  std::optional<Grid> a = grid_of(r.logits, dims), b = grid_of(r.tokens, dims);
  if (!a) {
    r.logits = r.logits.contiguous();
    a = grid_of(r.logits, dims);
  }
  if (!b) {
    r.tokens = r.tokens.contiguous();
    b = grid_of(r.tokens, dims);
  }
  if (a->outer != b->outer || a->inner != b->inner) {  // one is merged further than the other: split as the other is
    if (a->outer == 1 && a->inner == n) {
      a = Grid{b->outer, b->inner, a->stride_inner * b->inner, a->stride_inner};
    } else if (b->outer == 1 && b->inner == n) {
      b = Grid{a->outer, a->inner, b->stride_inner * a->inner, b->stride_inner};
    } else {
      r.tokens = r.tokens.contiguous();
      b = Grid{a->outer, a->inner, a->inner, 1};
    }
  }
  r.at = *a;
  r.token_outer = b->stride_outer;
  r.token_inner = b->stride_inner;
  return r;
}

struct Options {
  double temperature;
  int64_t top_k;
  bool entropy;
  int64_t ignore_index;
};

struct Results {
  Tensor logprobs, entropy, top_logprobs, top_tokens, stats;
};

Results forward(const Tensor& logits, const Tensor& tokens, const Options& o, bool want_stats) {
  const c10::DeviceGuard guard(logits.device());
  const auto fp32 = at::TensorOptions().dtype(at::kFloat).device(logits.device());
  std::vector<int64_t> shape = tokens.sizes().vec();
  Results r;
  r.logprobs = at::empty(shape, fp32);
  if (o.entropy) r.entropy = at::empty(shape, fp32);
  if (o.top_k) {
    shape.push_back(o.top_k);
    r.top_logprobs = at::empty(shape, fp32);
    r.top_tokens = at::empty(shape, fp32.dtype(at::kLong));
    shape.pop_back();
  }
  if (want_stats) {
    shape.push_back(2);
    r.stats = at::empty(shape, fp32);
  }
  const Located at = locate(logits, tokens);
  const int code = dtype_code(logits);
  const int64_t vocab = logits.size(-1);
  const size_t bytes = workspace_bytes(tokens.numel(), vocab, code, o.top_k);
  const Tensor ws = bytes ? at::empty({(int64_t)bytes}, fp32.dtype(at::kByte)) : Tensor();
  check(logprobs_call(address<void>(at.logits), code, at.at.outer, at.at.inner, vocab, at.at.stride_outer,
                      at.at.stride_inner, address<int64_t>(at.tokens), at.token_outer, at.token_inner, o.ignore_index,
                      (float)o.temperature, o.top_k, address<float>(r.logprobs), address<float>(r.entropy),
                      address<float>(r.top_logprobs), address<int64_t>(r.top_tokens), address<float>(r.stats),
                      address<void>(ws), bytes, stream_of(logits)),
        "fl_token_logprobs");
  return r;
}

Tensor backward(const Tensor& logits, const Tensor& tokens, const Tensor& stats, const Tensor& entropy,
                const Tensor& top_tokens, const Options& o, const Tensor* grads) {
  const c10::DeviceGuard guard(logits.device());
  Tensor g[3];
  for (int i = 0; i < 3; ++i) {
    if (!grads[i].defined()) continue;
    check_plain(grads[i], "the upstream gradients");
    g[i] = grads[i].resolve_neg().contiguous();
  }
  Tensor out = at::empty(logits.sizes(), at::TensorOptions().dtype(logits.scalar_type()).device(logits.device()));
  const Located at = locate(logits, tokens);
  check(logprobs_backward_call(address<void>(at.logits), dtype_code(logits), at.at.outer, at.at.inner, logits.size(-1),
                               at.at.stride_outer, at.at.stride_inner, address<int64_t>(at.tokens), at.token_outer,
                               at.token_inner, o.ignore_index, (float)o.temperature, o.top_k, address<float>(stats),
                               address<float>(entropy), address<int64_t>(top_tokens), address<float>(g[0]),
                               address<float>(g[1]), address<float>(g[2]), address<void>(out), stream_of(logits)),
        "fl_token_logprobs_backward");
  return out;
}

// The gradient in stock operations, which can be differentiated again: the function of Python that was handed over.
Tensor stock_backward(const Tensor& logits, const Tensor& tokens, const Tensor& top_tokens, const Options& o,
                      const Tensor* grads) {
  const PyGILState_STATE state = PyGILState_Ensure();
  PyObject* got = nullptr;
  const auto wrap = [](const Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); };
  PyObject* args = Py_BuildValue("(NNNdLNNN)", wrap(logits), wrap(tokens), wrap(top_tokens), o.temperature,
                                 (long long)o.ignore_index, wrap(grads[0]), wrap(grads[1]), wrap(grads[2]));
  if (args) got = PyObject_CallObject(stock_gradient, args);
  Py_XDECREF(args);
  Tensor out;
  if (got && THPVariable_Check(got)) out = THPVariable_Unpack(got);
  const bool none = got == Py_None;
  Py_XDECREF(got);
  if (!none && !out.defined()) {
    python_error e;  // carries the Python exception to whoever asked for the gradient
    e.persist();
    PyGILState_Release(state);
    throw e;
  }
  PyGILState_Release(state);
  return out;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  // the outputs that are wanted, in the order log probabilities, entropy, alternatives' log probabilities and tokens
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, double temperature,
                               int64_t top_k, bool entropy, int64_t ignore_index) {
    const Results r = ::forward(logits, tokens, {temperature, top_k, entropy, ignore_index}, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, tokens, r.stats, r.entropy, r.top_tokens});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["top_k"] = top_k;
    ctx->saved_data["ignore_index"] = ignore_index;
    variable_list out = {r.logprobs};
    if (entropy) out.push_back(r.entropy);
    if (top_k) {
      out.push_back(r.top_logprobs);
      out.push_back(r.top_tokens);
      ctx->mark_non_differentiable({r.top_tokens});
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &tokens = saved[1], &stats = saved[2], &entropy = saved[3], &top_tokens = saved[4];
    const Options o = {ctx->saved_data["temperature"].toDouble(), ctx->saved_data["top_k"].toInt(), entropy.defined(),
                       ctx->saved_data["ignore_index"].toInt()};
    Tensor g[3] = {grads[0]};
    if (o.entropy) g[1] = grads[1];
    if (o.top_k) g[2] = grads[o.entropy ? 2 : 1];
    variable_list out(6);
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return out;
    check_leaves(node_of(logits), "logits'");
    out[0] = at::GradMode::is_enabled() ? stock_backward(logits, tokens, top_tokens, o, g)
                                        : ::backward(logits, tokens, stats, entropy, top_tokens, o, g);
    return out;
  }
};

// token_logprobs(logits, tokens, temperature, top_k, entropy, ignore_index) -> (log probabilities, entropy, the
// alternatives' log probabilities, their tokens), None where not wanted
PyObject* token_logprobs(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *first, *second;
  Options o;
  long long top_k, ignore_index;
  int entropy;
  if (!PyArg_ParseTuple(args, "OOdLpL", &first, &second, &o.temperature, &top_k, &entropy, &ignore_index))
    return nullptr;
  o.top_k = top_k;
  o.entropy = entropy;
  o.ignore_index = ignore_index;
  TORCH_CHECK_TYPE(THPVariable_Check(first) && THPVariable_Check(second), "logits and tokens must be tensors");
  const Tensor &logits = THPVariable_Unpack(first), &tokens = THPVariable_Unpack(second);
  check_plain(logits, "logits");
  check_plain(tokens, "tokens");
  TORCH_CHECK_TYPE(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16,
                   "logits must be float32 or bfloat16, got ", logits.scalar_type());
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong, "tokens must be int64, got ", tokens.scalar_type());
  TORCH_CHECK_TYPE(logits.layout() == at::kStrided && tokens.layout() == at::kStrided,
                   "logits and tokens must be dense");
  TORCH_CHECK_VALUE(logits.dim() >= 1 && tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1), "tokens ",
                    tokens.sizes(), " must be the logits' rows ", logits.sizes());
  const int64_t vocab = logits.size(-1), most = std::min(kMaxTop, vocab);
  TORCH_CHECK_VALUE(vocab > 0 && vocab <= kMaxVocab, "a row must have 1 to ", kMaxVocab, " logits, got ", vocab);
  TORCH_CHECK_VALUE(o.temperature >= kMinTemperature && o.temperature <= kMaxTemperature, "temperature must be ",
                    kMinTemperature, " to ", kMaxTemperature, ", got ", o.temperature);
  TORCH_CHECK_VALUE(o.top_k >= 0 && o.top_k <= most, "top_k must be 0 to ", most, ", got ", o.top_k);
  TORCH_CHECK(logits.is_cuda(), "token_logprobs requires a ROCm (cuda) device");
  check_not_traced("token_logprobs");
  TORCH_CHECK_VALUE(tokens.device() == logits.device(), "logits and tokens must be on one device");
  TORCH_CHECK_NOT_IMPLEMENTED(!logits._fw_grad(0).defined(), "token_logprobs has no forward-mode derivative");
  const Tensor x = logits.resolve_neg(), t = tokens.resolve_neg();
  variable_list out;
  if (t.numel() == 0) {  // no rows: empty outputs, on the logits' graph
    const Tensor none = x.sum(-1, false, at::kFloat);
    out = {none};
    if (o.entropy) out.push_back(none.clone());
    if (o.top_k) {
      std::vector<int64_t> shape = none.sizes().vec();
      shape.push_back(o.top_k);
      out.push_back(none.unsqueeze(-1).expand(shape).clone());
      out.push_back(t.unsqueeze(-1).expand(shape).clone());
    }
  } else if (at::GradMode::is_enabled() && x.requires_grad()) {
    out = TokenLogprobs::apply(x, t, o.temperature, o.top_k, o.entropy, o.ignore_index);
  } else {
    const Results r = forward(x, t, o, false);
    out = {r.logprobs};
    if (o.entropy) out.push_back(r.entropy);
    if (o.top_k) out.insert(out.end(), {r.top_logprobs, r.top_tokens});
  }
  size_t i = 0;
  const auto next = [&](bool wanted) { return wanted ? THPVariable_Wrap(out[i++]) : Py_NewRef(Py_None); };
  PyObject *a = next(true), *b = next(o.entropy), *c = next(o.top_k > 0), *d = next(o.top_k > 0);
  return Py_BuildValue("(NNNN)", a, b, c, d);
  END_HANDLE_TH_ERRORS
}

// where(logits, tokens) -> (logits, tokens, outer, inner, the logits' strides, the tokens'): the rows as a call sees
// them
PyObject* where(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *first, *second;
  if (!PyArg_ParseTuple(args, "OO", &first, &second)) return nullptr;
  TORCH_CHECK_TYPE(THPVariable_Check(first) && THPVariable_Check(second), "logits and tokens must be tensors");
  const Located r = locate(THPVariable_Unpack(first), THPVariable_Unpack(second));
  return Py_BuildValue("(NNLLLLLL)", THPVariable_Wrap(r.logits), THPVariable_Wrap(r.tokens), (long long)r.at.outer,
                       (long long)r.at.inner, (long long)r.at.stride_outer, (long long)r.at.stride_inner,
                       (long long)r.token_outer, (long long)r.token_inner);
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the library's entry points, the stock gradient)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a[7];
  PyObject* stock;
  if (!PyArg_ParseTuple(args, "KKKKKKKO", a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6, &stock)) return nullptr;
  workspace_bytes = reinterpret_cast<decltype(workspace_bytes)>(a[0]);
  logprobs_call = reinterpret_cast<decltype(logprobs_call)>(a[1]);
  logprobs_backward_call = reinterpret_cast<decltype(logprobs_backward_call)>(a[2]);
  norm_bytes = reinterpret_cast<decltype(norm_bytes)>(a[3]);
  norm_call = reinterpret_cast<decltype(norm_call)>(a[4]);
  adamw_bytes = reinterpret_cast<decltype(adamw_bytes)>(a[5]);
  adamw_call = reinterpret_cast<decltype(adamw_call)>(a[6]);
  Py_INCREF(stock);
  Py_XDECREF(stock_gradient);
  stock_gradient = stock;
  Py_RETURN_NONE;
}

// grad_norm(gradients, max_norm or a negative number for none) -> (norm, scale or None)
PyObject* grad_norm(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject* list;
  double max_norm;
  if (!PyArg_ParseTuple(args, "Od", &list, &max_norm)) return nullptr;
  const at::Device device = first_of(list, "gradients").device();
  TORCH_CHECK(device.is_cuda(), "grad_norm requires a ROCm (cuda) device");
  check_not_traced("grad_norm");
  const TensorList grads(list, "gradients", device, {at::kFloat, at::kBFloat16}, nullptr, 1, true);
  const c10::DeviceGuard guard(device);
  const int64_t n = (int64_t)grads.size();
  const bool scaled = !(max_norm < 0.0);
  const Tensor out = at::empty({2}, at::TensorOptions().dtype(at::kFloat).device(device));
  const size_t bytes = norm_bytes(n, grads.counts.data());
  const Tensor ws = workspace_on(device, bytes);
  check(norm_call(n, grads.addresses.data(), grads.codes.data(), grads.counts.data(), scaled ? (float)max_norm : 0.f,
                  scaled, address<float>(out), address<void>(ws), bytes, stream_of(out)),
        "fl_grad_norm");
  PyObject* norm = THPVariable_Wrap(out.select(0, 0));
  PyObject* scale = scaled ? THPVariable_Wrap(out.select(0, 1)) : Py_NewRef(Py_None);
  return Py_BuildValue("(NN)", norm, scale);
  END_HANDLE_TH_ERRORS
}

// adamw_step(parameters, gradients, first moments, second moments, steps (a list or one tensor), lr (a number or a
// tensor), beta1, beta2, eps, weight decay, gradient scale or None, the moments' scales or None twice)
PyObject* adamw_step(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *params, *grads, *avgs, *sqs, *steps, *lr, *grad_scale, *avg_scales, *sq_scales;
  double beta1, beta2, eps, decay;
  if (!PyArg_ParseTuple(args, "OOOOOOddddOOO", &params, &grads, &avgs, &sqs, &steps, &lr, &beta1, &beta2, &eps, &decay,
                        &grad_scale, &avg_scales, &sq_scales))
    return nullptr;
  const Tensor& first = first_of(params, "parameters");
  const at::Device device = first.device();
  const at::ScalarType type = first.scalar_type();
  TORCH_CHECK_TYPE(type == at::kFloat || type == at::kBFloat16, "parameters must be float32 or bfloat16, got ", type);
  const bool eight = avg_scales != Py_None;
  const auto as_long = [&](PyObject* o) {
    return (!PyList_Check(o) && !PyTuple_Check(o)) || PySequence_Fast_GET_SIZE(o) == PySequence_Fast_GET_SIZE(params);
  };
  TORCH_CHECK_VALUE(as_long(grads) && as_long(avgs) && as_long(sqs) && as_long(steps) && as_long(avg_scales) &&
                        as_long(sq_scales),
                    "one gradient, one state of each kind and one step per parameter");
  TORCH_CHECK_VALUE(eight == (sq_scales != Py_None), "8-bit states need the scales of both moments");
  TORCH_CHECK(device.is_cuda(), "adamw_step requires a ROCm (cuda) device");
  check_not_traced("adamw_step");
  const TensorList p(params, "parameters", device, {type});
  const int64_t n = (int64_t)p.size();
  const TensorList g(grads, "gradients", device, {type}, &p.counts, 1, true);
  for (int64_t i = 0; i < n; ++i)
    TORCH_CHECK_VALUE(p.shapes[i] == g.shapes[i], "gradient ", i, " has the shape ", g.shapes[i], ", its parameter ",
                      p.shapes[i]);
  const at::ScalarType state = eight ? at::kFloat8_e4m3fn : at::kFloat;
  const TensorList m(avgs, "states", device, {state}, &p.counts), v(sqs, "states", device, {state}, &p.counts);
  Ranges written;
  written.reserve(6 * n);
  const size_t size = type == at::kFloat ? 4 : 2;
  merge(written, ranges_of(p, size));
  merge(written, ranges_of(m, eight ? 1 : 4));
  merge(written, ranges_of(v, eight ? 1 : 4));
  std::vector<void*> ms, vs;
  if (eight) {
    const TensorList m_scales(avg_scales, "scales", device, {at::kFloat}, &p.counts, kStateBlock);
    const TensorList v_scales(sq_scales, "scales", device, {at::kFloat}, &p.counts, kStateBlock);
    merge(written, ranges_of(m_scales, 4));
    merge(written, ranges_of(v_scales, 4));
    ms = m_scales.addresses;
    vs = v_scales.addresses;
  }
  std::vector<void*> step_at;
  if (THPVariable_Check(steps)) {
    const Tensor& t = THPVariable_Unpack(steps);
    check_plain(t, "steps");
    TORCH_CHECK_VALUE(t.scalar_type() == at::kLong && t.device() == device && t.dim() == 1 && t.numel() == n &&
                          t.is_contiguous() && !t.is_neg(),
                      "steps must be ", n, " contiguous int64 values on ", device);
    for (int64_t i = 0; i < n; ++i) step_at.push_back(static_cast<int64_t*>(t.data_ptr()) + i);
    const uintptr_t at = reinterpret_cast<uintptr_t>(step_at[0]);
    merge(written, {{at, at + n * 8}});
  } else {
    const std::vector<int64_t> ones(n, 1);
    const TensorList list(steps, "steps", device, {at::kLong}, &ones);
    merge(written, ranges_of(list, 8));
    step_at = list.addresses;
  }
  TORCH_CHECK_VALUE(!overlap(written), "parameters, states or step counters share memory");
  TORCH_CHECK_VALUE(!meet(written, ranges_of(g, size)),
                    "a gradient shares memory with a parameter, a state or a step counter");
  const Tensor scale = device_value(grad_scale, "grad_scale", device);
  const Tensor lr_at = THPVariable_Check(lr) ? device_value(lr, "lr", device) : Tensor();
  const double lr_value = lr_at.defined() ? 0.0 : PyFloat_AsDouble(lr);
  if (PyErr_Occurred()) return nullptr;
  const c10::DeviceGuard guard(device);
  const size_t bytes = adamw_bytes(n);
  const Tensor ws = workspace_on(device, bytes);
  check(adamw_call(n, p.addresses.data(), g.addresses.data(), type == at::kBFloat16 ? FL_DTYPE_BF16 : FL_DTYPE_F32,
                   m.addresses.data(), v.addresses.data(), eight ? reinterpret_cast<float* const*>(ms.data()) : nullptr,
                   eight ? reinterpret_cast<float* const*>(vs.data()) : nullptr, p.counts.data(),
                   reinterpret_cast<int64_t* const*>(step_at.data()), lr_value, address<float>(lr_at), beta1, beta2, eps,
                   decay, address<float>(scale), address<void>(ws), bytes, stream_of(first)),
        "fl_adamw_step");
  for (PyObject* list : {params, avgs, sqs, steps, avg_scales, sq_scales}) count_writes(list);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

}  // namespace

// the calls of host_train.cpp
PyObject* host_bind_train(PyObject*, PyObject*);
PyObject* host_embedding(PyObject*, PyObject*);
PyObject* host_gated_scan(PyObject*, PyObject*);
PyObject* host_orthogonalize(PyObject*, PyObject*);
PyObject* host_check_steps(PyObject*, PyObject*);
PyObject* host_muon_step(PyObject*, PyObject*);

namespace {

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "the library's entry points and the stock gradient"},
                         {"token_logprobs", token_logprobs, METH_VARARGS, "the call"},
                         {"where", where, METH_VARARGS, "the rows of logits and tokens"},
                         {"grad_norm", grad_norm, METH_VARARGS, "the call"},
                         {"adamw_step", adamw_step, METH_VARARGS, "the call"},
                         {"bind_train", host_bind_train, METH_VARARGS, "the entry points of the calls below"},
                         {"embedding", host_embedding, METH_VARARGS, "the call"},
                         {"gated_scan", host_gated_scan, METH_VARARGS, "the call"},
                         {"orthogonalize", host_orthogonalize, METH_VARARGS, "the call"},
                         {"check_steps", host_check_steps, METH_VARARGS, "of orthogonalization"},
                         {"muon_step", host_muon_step, METH_VARARGS, "the call"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
