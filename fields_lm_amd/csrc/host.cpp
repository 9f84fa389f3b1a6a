// host.cpp — the host side of calls whose cost in Python is more than their kernels': a module of CPython's and
// PyTorch's headers, no device code.
//
// token_logprobs: the whole of the call (checks, where the rows are, outputs, autograd). With a gradient it is an
// autograd function of C++, so that the engine's thread waits for no interpreter: 64 rows with entropy and five
// alternatives cost 15.7 us a call from Python, forward and gradient of a few rows 110 (an operator of PyTorch's own
// and its gradient: 46).
//
// Lists of tensors: what the optimizer's calls read of them, in one pass and without a Python object per attribute.
// A step reads some twenty attributes of each of a model's hundreds of tensors: through Python's accessors that is
// 1.2 us a tensor.
//
// read(tensors, device_index, dtypes, addresses, counts, codes, expected, block) -> None, or (index, what is wrong)
//   tensors: a list or tuple; dtypes: the torch dtypes taken, in the order of their codes; addresses, counts (int64)
//   and codes (int32): host addresses of arrays that hold len(tensors) words, 0 for not wanted; expected: the same of
//   the counts that the tensors must have, in blocks of `block` values (rounded up).
// same_shapes(a, b) -> the index of the first pair that differs, or -1.
// repeats(addresses, counts, n) -> whether two of the n addresses with a count that is not 0 are equal (counts 0: any).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <optional>
#include <vector>

#include "fields_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The library's entry points, which the loader of the library hands over, and the stock form of the gradient.
decltype(&fl_token_logprobs_workspace_bytes) workspace_bytes = nullptr;
decltype(&fl_token_logprobs) logprobs_call = nullptr;
decltype(&fl_token_logprobs_backward) logprobs_backward_call = nullptr;
PyObject* stock_gradient = nullptr;

constexpr int64_t kMaxTop = 64, kMaxVocab = (int64_t)1 << 23;
constexpr double kMinTemperature = 0x1p-20, kMaxTemperature = 0x1p20;

void check(int code, const char* what) {
  TORCH_CHECK_VALUE(code != FL_ERR_INVALID_ARGUMENT, what, ": invalid shape, stride or pointer");
  TORCH_CHECK_TYPE(code != FL_ERR_DTYPE, what, ": unsupported dtype");
  TORCH_CHECK(code != FL_ERR_WORKSPACE, what, ": workspace missing or too small");
  TORCH_CHECK(code < FL_ERR_HIP_BASE, what, ": HIP error ", code - FL_ERR_HIP_BASE);
  TORCH_CHECK(code == FL_OK, what, ": error code ", code);
}

int dtype_code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? FL_DTYPE_BF16 : FL_DTYPE_F32; }

void* stream_of(const Tensor& t) { return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

template <typename T>
T* address(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

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
  for (int i = 0; i < 3; ++i)
    if (grads[i].defined()) g[i] = grads[i].contiguous();
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
  if (!PyArg_ParseTuple(args, "OOdLpL", &first, &second, &o.temperature, &top_k, &entropy, &ignore_index)) return nullptr;
  o.top_k = top_k;
  o.entropy = entropy;
  o.ignore_index = ignore_index;
  TORCH_CHECK_TYPE(THPVariable_Check(first) && THPVariable_Check(second), "logits and tokens must be tensors");
  const Tensor &logits = THPVariable_Unpack(first), &tokens = THPVariable_Unpack(second);
  TORCH_CHECK_TYPE(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16,
                   "logits must be float32 or bfloat16, got ", logits.scalar_type());
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong, "tokens must be int64, got ", tokens.scalar_type());
  TORCH_CHECK_TYPE(logits.layout() == at::kStrided && tokens.layout() == at::kStrided, "logits and tokens must be dense");
  TORCH_CHECK_VALUE(logits.dim() >= 1 && tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1), "tokens ",
                    tokens.sizes(), " must be the logits' rows ", logits.sizes());
  const int64_t vocab = logits.size(-1), most = std::min(kMaxTop, vocab);
  TORCH_CHECK_VALUE(vocab > 0 && vocab <= kMaxVocab, "a row must have 1 to ", kMaxVocab, " logits, got ", vocab);
  TORCH_CHECK_VALUE(o.temperature >= kMinTemperature && o.temperature <= kMaxTemperature, "temperature must be ",
                    kMinTemperature, " to ", kMaxTemperature, ", got ", o.temperature);
  TORCH_CHECK_VALUE(o.top_k >= 0 && o.top_k <= most, "top_k must be 0 to ", most, ", got ", o.top_k);
  TORCH_CHECK(logits.is_cuda(), "token_logprobs requires a ROCm (cuda) device");
  TORCH_CHECK_VALUE(tokens.device() == logits.device(), "logits and tokens must be on one device");
  TORCH_CHECK_NOT_IMPLEMENTED(!logits._fw_grad(0).defined(), "token_logprobs has no forward-mode derivative");
  const Tensor x = logits.is_neg() ? logits.resolve_neg() : logits;
  variable_list out;
  if (tokens.numel() == 0) {  // no rows: empty outputs, on the logits' graph
    const Tensor none = x.sum(-1, false, at::kFloat);
    out = {none};
    if (o.entropy) out.push_back(none.clone());
    if (o.top_k) {
      std::vector<int64_t> shape = none.sizes().vec();
      shape.push_back(o.top_k);
      out.push_back(none.unsqueeze(-1).expand(shape).clone());
      out.push_back(tokens.unsqueeze(-1).expand(shape).clone());
    }
  } else if (at::GradMode::is_enabled() && x.requires_grad()) {
    out = TokenLogprobs::apply(x, tokens, o.temperature, o.top_k, o.entropy, o.ignore_index);
  } else {
    const Results r = forward(x, tokens, o, false);
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

// where(logits, tokens) -> (logits, tokens, outer, inner, the logits' strides, the tokens'): the rows as a call sees them
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

// bind(addresses of the library's three entry points, the stock gradient)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a, b, c;
  PyObject* stock;
  if (!PyArg_ParseTuple(args, "KKKO", &a, &b, &c, &stock)) return nullptr;
  workspace_bytes = reinterpret_cast<decltype(workspace_bytes)>(a);
  logprobs_call = reinterpret_cast<decltype(logprobs_call)>(b);
  logprobs_backward_call = reinterpret_cast<decltype(logprobs_backward_call)>(c);
  Py_INCREF(stock);
  Py_XDECREF(stock_gradient);
  stock_gradient = stock;
  Py_RETURN_NONE;
}

// Items of a list or tuple, borrowed.
struct Items {
  PyObject** at = nullptr;
  Py_ssize_t n = 0;
  bool of(PyObject* o) {
    if (!PyList_Check(o) && !PyTuple_Check(o)) {
      PyErr_SetString(PyExc_TypeError, "a list or tuple is wanted");
      return false;
    }
    at = PySequence_Fast_ITEMS(o);
    n = PySequence_Fast_GET_SIZE(o);
    return true;
  }
};

PyObject* wrong(Py_ssize_t i, const char* what) { return Py_BuildValue("(ns)", i, what); }

PyObject* read(PyObject*, PyObject* args) {
  PyObject *list, *types;
  long long device, addresses, counts, codes, expected, block;
  Items items, taken;
  if (!PyArg_ParseTuple(args, "OLOLLLLL", &list, &device, &types, &addresses, &counts, &codes, &expected,
                        &block) || !items.of(list) ||
      !taken.of(types))
    return nullptr;
  at::ScalarType wanted[8];
  if (block < 1) return PyErr_Format(PyExc_ValueError, "a block has 1 value or more");
  if (taken.n > 8) return PyErr_Format(PyExc_ValueError, "at most 8 types");
  for (Py_ssize_t k = 0; k < taken.n; ++k) {
    if (!THPDtype_Check(taken.at[k])) return PyErr_Format(PyExc_TypeError, "a dtype is wanted");
    wanted[k] = reinterpret_cast<THPDtype*>(taken.at[k])->scalar_type;
  }
  try {
    for (Py_ssize_t i = 0; i < items.n; ++i) {
      if (!THPVariable_Check(items.at[i])) return wrong(i, "tensor");
      const Tensor& t = THPVariable_Unpack(items.at[i]);
      Py_ssize_t code = 0;
      while (code < taken.n && wanted[code] != t.scalar_type()) ++code;
      if (code == taken.n) return wrong(i, "dtype");
      if (t.layout() != at::kStrided || t.is_neg()) return wrong(i, "layout");
      if (!t.device().is_cuda() || t.device().index() != device) return wrong(i, "device");
      if (!t.is_contiguous()) return wrong(i, "contiguous");
      if (expected && t.numel() != (reinterpret_cast<const int64_t*>(expected)[i] + block - 1) / block) return wrong(i, "count");
      if (addresses) reinterpret_cast<int64_t*>(addresses)[i] = reinterpret_cast<int64_t>(t.data_ptr());
      if (counts) reinterpret_cast<int64_t*>(counts)[i] = t.numel();
      if (codes) reinterpret_cast<int32_t*>(codes)[i] = (int32_t)code;
    }
  } catch (const std::exception& e) {  // a tensor without memory of its own (a wrapper of some transform)
    return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
  }
  Py_RETURN_NONE;
}

PyObject* same_shapes(PyObject*, PyObject* args) {
  PyObject *first, *second;
  Items a, b;
  if (!PyArg_ParseTuple(args, "OO", &first, &second) || !a.of(first) || !b.of(second)) return nullptr;
  try {
    for (Py_ssize_t i = 0; i < a.n; ++i) {
      if (i >= b.n || !THPVariable_Check(a.at[i]) || !THPVariable_Check(b.at[i]) ||
          THPVariable_Unpack(a.at[i]).sizes() != THPVariable_Unpack(b.at[i]).sizes())
        return PyLong_FromSsize_t(i);
    }
  } catch (const std::exception& e) {
    return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
  }
  return PyLong_FromSsize_t(a.n == b.n ? -1 : a.n);
}

PyObject* repeats(PyObject*, PyObject* args) {
  long long addresses, counts, n;
  if (!PyArg_ParseTuple(args, "LLL", &addresses, &counts, &n)) return nullptr;
  try {
    std::vector<int64_t> at;
    for (long long i = 0; i < n; ++i)
      if (!counts || reinterpret_cast<const int64_t*>(counts)[i]) at.push_back(reinterpret_cast<const int64_t*>(addresses)[i]);
    std::sort(at.begin(), at.end());
    return PyBool_FromLong(std::adjacent_find(at.begin(), at.end()) != at.end());
  } catch (const std::exception& e) {
    return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
  }
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "the library's entry points and the stock gradient"},
                         {"token_logprobs", token_logprobs, METH_VARARGS, "the call"},
                         {"where", where, METH_VARARGS, "the rows of logits and tokens"},
                         {"read", read, METH_VARARGS, "addresses, counts and types of a list of tensors"},
                         {"same_shapes", same_shapes, METH_VARARGS, "first pair of unequal shapes"},
                         {"repeats", repeats, METH_VARARGS, "whether an address occurs twice"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
