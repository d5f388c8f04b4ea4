// What the operators of the `supa` namespace share: checks of arguments, calls
// through the dispatcher, and whether tensors share memory.
#pragma once

#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <algorithm>
#include <optional>

#include "common.h"

namespace supa {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = std::optional<at::Tensor>;

inline bool is_float16_or_32(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
inline bool given(const OptTensor& t) { return t.has_value() && t->defined(); }
inline OptTensor maybe(const at::Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
inline const void* ptr(const OptTensor& t) { return given(t) ? t->data_ptr() : nullptr; }

// Values of forward-mode differentiation would be dropped without a word.
inline void check_no_tangent(const char* op, std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), op,
                                ": no forward-mode derivative");
}
inline const at::Tensor& tensor(const OptTensor& t) {
  static const at::Tensor none;
  return given(t) ? *t : none;
}

// The operator of this schema name, called through the dispatcher.
template <typename F> c10::TypedOperatorHandle<F> find_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<F>();
}

// Meta tensors stand for supa ones.
inline bool is_supa(const at::Tensor& t) { return t.device().type() == kSupa || t.is_meta(); }
inline at::Tensor empty_beside(const at::Tensor& t, c10::IntArrayRef sizes, at::ScalarType dtype) {
  return t.is_meta() ? at::empty(sizes, t.options().dtype(dtype)) : empty_supa(sizes, dtype, t.device().index());
}

inline void check_on(const char* op, const char* name, const at::Tensor& t, const at::Tensor& like) {
  TORCH_CHECK(t.device() == like.device(), op, ": ", name, " is on ", t.device(), ", expected ", like.device());
}

inline OptTensor contiguous(const OptTensor& t) { return given(t) ? OptTensor(t->contiguous()) : std::nullopt; }

// A step through memory, in bytes, and how often the one and the other tensor take it.
struct Step {
  int64_t stride, one, other;
};
using Steps = c10::SmallVector<Step, 8>;

// The steps of a tensor and, if there is one, of another, from long to short; a
// step that both take is one step, one that a tensor takes in two dims is two.
inline Steps steps_of(const at::Tensor& one, const at::Tensor& other = {}) {
  Steps steps;
  const auto add = [&](const at::Tensor& t, int64_t Step::* times) {
    for (int64_t i = 0; i < t.dim(); ++i) {
      if (t.size(i) == 1) continue;
      const int64_t stride = t.stride(i) * (int64_t)t.element_size();
      auto at = std::find_if(steps.begin(), steps.end(), [&](const Step& s) { return s.stride == stride && s.*times == 0; });
      if (at == steps.end()) at = steps.insert(at, {stride, 0, 0});
      (*at).*times = t.size(i) - 1;
    }
  };
  add(one, &Step::one);
  if (other.defined()) add(other, &Step::other);
  std::sort(steps.begin(), steps.end(), [](const Step& a, const Step& b) { return a.stride > b.stride; });
  return steps;
}

// Whether blocks of `block` bytes, one at every combination of the first n steps
// (the one tensor's), keep apart: each step goes past all that the smaller ones reach.
inline bool apart(const Steps& steps, size_t n, int64_t block) {
  for (size_t i = n; i-- > 0;) {
    if (steps[i].stride < block) return false;
    block += steps[i].one * steps[i].stride;
  }
  return true;
}

// Whether two tensors share no memory, of any types and shapes: over their smaller
// steps (or none, or all) each fills a block, the other's beside the one's, and
// their larger steps, which both may take, lead from one such pair of blocks to the
// next (q and k of a packed projection, token by token or sample by sample; the
// columns of a matrix).
inline bool beside(const at::Tensor& a, const at::Tensor& b) {
  const bool ordered = a.data_ptr() <= b.data_ptr();
  const at::Tensor &one = ordered ? a : b, &other = ordered ? b : a;
  const int64_t distance = static_cast<const char*>(other.data_ptr()) - static_cast<const char*>(one.data_ptr());
  const Steps steps = steps_of(one, other);
  int64_t first = (int64_t)one.element_size(), second = (int64_t)other.element_size();  // the blocks' bytes
  for (size_t outer = steps.size();; --outer) {
    // the other's first block lies so many steps ahead, and `gap` behind the one's block there
    int64_t gap = distance;
    Steps joint(steps.begin(), steps.begin() + outer);
    for (Step& s : joint) {
      if (s.stride == 0) return false;
      const int64_t ahead = gap / s.stride;
      gap -= ahead * s.stride;
      s.one = std::max(s.one, s.other + ahead);
    }
    if (first <= gap && apart(joint, outer, gap + second)) return true;
    if (outer == 0) return false;
    first += steps[outer - 1].one * steps[outer - 1].stride;
    second += steps[outer - 1].other * steps[outer - 1].stride;
  }
}

// A tensor that was written has a new version, in inference mode too (where autograd's
// kernels are left out, this key's are not).
inline void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace supa
