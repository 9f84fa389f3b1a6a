// host_common.h — what the sources of the host module _host.so share: checks, addresses, lists of tensors.
#ifndef FL_HOST_COMMON_H_
#define FL_HOST_COMMON_H_

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <memory>
#include <optional>
#include <unordered_set>
#include <utility>
#include <vector>

#include "fields_amd.h"

namespace host {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline void check(int code, const char* what) {
  TORCH_CHECK_VALUE(code != FL_ERR_INVALID_ARGUMENT, what, ": invalid shape, stride or pointer");
  TORCH_CHECK_TYPE(code != FL_ERR_DTYPE, what, ": unsupported dtype");
  TORCH_CHECK(code != FL_ERR_WORKSPACE, what, ": workspace missing or too small");
  TORCH_CHECK(code < FL_ERR_HIP_BASE, what, ": HIP error ", code - FL_ERR_HIP_BASE);
  TORCH_CHECK(code == FL_OK, what, ": error code ", code);
}

// a trace would keep the results of its example as constants
inline void check_not_traced(const char* what) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " reads addresses and cannot be traced");
}

// A tensor that dispatches to Python (a fake one, say) has no memory of its own behind its address.
inline void check_plain(const Tensor& t, const char* what) {
  TORCH_CHECK_TYPE(!t.key_set().has(c10::DispatchKey::Python), what, " must be plain tensors");
}

inline int dtype_code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? FL_DTYPE_BF16 : FL_DTYPE_F32; }

inline void* stream_of(const Tensor& t) { return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

template <typename T>
T* address(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

// where an input's gradient goes
inline std::shared_ptr<torch::autograd::Node> node_of(const Tensor& input) {
  return input.grad_fn() ? input.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(input);
}

// A captured backward adds into an input's leaves on the streams that their eager graphs, where one still lives,
// were made on. The default stream cannot join a capture, which ends in an error that the engine does not survive.
inline void check_leaves(const std::shared_ptr<torch::autograd::Node>& from, const char* whose) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  std::vector<std::shared_ptr<torch::autograd::Node>> todo = {from};
  std::unordered_set<torch::autograd::Node*> seen;
  while (!todo.empty()) {
    const std::shared_ptr<torch::autograd::Node> node = todo.back();
    todo.pop_back();
    if (!node || !seen.insert(node.get()).second) continue;
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(node.get())) {
      const std::optional<c10::Stream> stream = node->stream();
      TORCH_CHECK(!stream || stream->id() != 0, "the ", whose,
                  " leaves hold an autograd graph made on the default stream: drop it (its outputs) before a backward "
                  "pass is captured");
    }
    for (const auto& edge : node->next_edges()) todo.push_back(edge.function);
  }
}

// A Python list or tuple of tensors: contiguous, of one of `types` (their places are the type codes), on `device`, with
// the counts of values that are expected. Gradients of other strides are copied.
struct TensorList {
  std::vector<void*> addresses;
  std::vector<int64_t> counts;
  std::vector<int> codes;
  std::vector<Tensor> kept;  // copies that have to live until the launch
  std::vector<at::IntArrayRef> shapes;

  TensorList(PyObject* list, const char* what, at::Device device, std::initializer_list<at::ScalarType> types,
             const std::vector<int64_t>* expected = nullptr, int64_t block = 1, bool copy = false) {
    TORCH_CHECK_TYPE(PyList_Check(list) || PyTuple_Check(list), what, " must be a list or tuple of tensors");
    PyObject** items = PySequence_Fast_ITEMS(list);
    const size_t n = (size_t)PySequence_Fast_GET_SIZE(list);
    addresses.reserve(n);
    counts.reserve(n);
    codes.reserve(n);
    shapes.reserve(n);
    for (size_t i = 0; i < n; ++i) {
      TORCH_CHECK_TYPE(THPVariable_Check(items[i]), what, ": number ", i, " is no tensor");
      const Tensor& t = THPVariable_Unpack(items[i]);
      check_plain(t, what);
      const auto at = std::find(types.begin(), types.end(), t.scalar_type());
      TORCH_CHECK_TYPE(at != types.end(), what, " must be ", *types.begin(),
                       types.size() > 1 ? " or another type of the list" : "",
                       ", number ", i, " is ", t.scalar_type());
      TORCH_CHECK_TYPE(t.layout() == at::kStrided, what, " must be dense, number ", i, " is ", t.layout());
      TORCH_CHECK_VALUE(t.device() == device, what, " must be on ", device, ", number ", i, " is on ", t.device());
      const int64_t count = t.numel();
      TORCH_CHECK_VALUE(!expected || count == ((*expected)[i] + block - 1) / block, what, ": number ", i, " has ",
                        count,
                        " values, ", ((*expected)[i] + block - 1) / block, " are wanted");
      const bool plain = t.is_contiguous() && !t.is_neg();
      TORCH_CHECK_VALUE(plain || copy, what, " must be contiguous, number ", i, " is not");
      if (!plain) kept.push_back(t.detach().resolve_neg().contiguous());
      addresses.push_back((plain ? t : kept.back()).data_ptr());
      counts.push_back(count);
      codes.push_back((int)(at - types.begin()));
      shapes.push_back(t.sizes());
    }
  }
  size_t size() const { return addresses.size(); }
};

typedef std::vector<std::pair<uintptr_t, uintptr_t>> Ranges;  // of addresses, [first, last + 1), in their order

inline Ranges ranges_of(const TensorList& list, size_t size) {
  Ranges r;
  r.reserve(list.size());
  for (size_t i = 0; i < list.size(); ++i) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(list.addresses[i]);
    if (list.counts[i]) r.emplace_back(at, at + list.counts[i] * size);
  }
  if (!std::is_sorted(r.begin(), r.end())) std::sort(r.begin(), r.end());
  return r;
}

// Lists that lie in one buffer each come in order and apart, and need no sorting of all ranges anew; states allocated
// parameter by parameter lie between each other and are merged (host time of a step of 240 tensors with 8-bit states:
// 53 us in one buffer a kind, 75 as AdamW makes them).
inline void merge(Ranges& to, const Ranges& r) {
  if (r.empty()) return;
  const bool ahead = !to.empty() && r.back() < to.front(), behind = to.empty() || to.back() < r.front();
  const auto middle = to.insert(ahead ? to.begin() : to.end(), r.begin(), r.end());
  if (!ahead && !behind) std::inplace_merge(to.begin(), middle, to.end());
}

inline bool overlap(const Ranges& r) {
  for (size_t i = 1; i < r.size(); ++i)
    if (r[i].first < r[i - 1].second) return true;
  return false;
}

// whether one of a, which are apart, and one of b share an address
inline bool meet(const Ranges& a, const Ranges& b) {
  for (size_t i = 0, j = 0; i < a.size() && j < b.size();) {
    if (a[i].second <= b[j].first) ++i;
    else if (b[j].second <= a[i].first) ++j;
    else return true;
  }
  return false;
}

// the first tensor of a list or tuple, whose device the others are to be on
inline const Tensor& first_of(PyObject* list, const char* what) {
  TORCH_CHECK_TYPE(PyList_Check(list) || PyTuple_Check(list), what, " must be a list or tuple of tensors");
  TORCH_CHECK_VALUE(PySequence_Fast_GET_SIZE(list) > 0, "no ", what);
  PyObject* first = PySequence_Fast_ITEMS(list)[0];
  TORCH_CHECK_TYPE(THPVariable_Check(first), what, ": number 0 is no tensor");
  return THPVariable_Unpack(first);
}

// one fp32 value on the device (a copy where its memory holds the negative), or none
inline Tensor device_value(PyObject* o, const char* what, at::Device device) {
  if (o == Py_None) return {};
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must be a tensor");
  const Tensor& t = THPVariable_Unpack(o);
  check_plain(t, what);
  TORCH_CHECK_VALUE(t.numel() == 1 && t.scalar_type() == at::kFloat && t.device() == device, what,
                    " must be one float32 value on ", device);
  TORCH_CHECK_VALUE(t.data_ptr(), what, " has no memory");  // (an address of 0 stands for no value)
  return t.is_neg() ? t.detach().resolve_neg() : t;
}

inline Tensor workspace_on(at::Device device, size_t bytes) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 1)}, at::TensorOptions().dtype(at::kByte).device(device));
}

// Tensors (one, a list or tuple, or None) that were written in place: what autograd saved of them is stale.
inline void count_writes(PyObject* o) {
  const auto count = [](PyObject* item) {
    const Tensor& t = THPVariable_Unpack(item);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  };
  if (o == Py_None) return;
  if (THPVariable_Check(o)) return count(o);
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(o); ++i) count(PySequence_Fast_ITEMS(o)[i]);
}

}  // namespace host

#endif  // FL_HOST_COMMON_H_
