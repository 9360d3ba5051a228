// operator_calls.h — what the calls of the decoder's and the experts' operators look at in their tensors.
#pragma once

#include "rxmet_torch.h"

#include <ATen/TensorSubclassLikeUtils.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <optional>

#include "rxmet_qdq.h"

namespace rxmet_torch {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// rxmet_last_error of the librxmet.so that rxmet_lib.py has loaded (bind_decoder()).
inline const char *(*last_error)(void) = nullptr;

inline void check(int rc, const char *what) {
  if (rc != 0)
    throw LibraryError(std::string(what) + " failed (" + std::to_string(rc) + "): " + last_error());
}

inline int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return RXMET_QDQ_F32;
    case at::kHalf: return RXMET_QDQ_F16;
    case at::kBFloat16: return RXMET_QDQ_BF16;
    default: return -1;
  }
}

inline bool plain(const Tensor &t) {
  return t.is_cuda() && !at::isTensorSubclassLike(t) && !torch::jit::tracer::isTracing();
}

inline bool is(const Tensor &t, at::ScalarType type, const Tensor &like) {
  return t.scalar_type() == type && plain(t) && t.device() == like.device();
}

// Whether forward-mode differentiation goes through t: a tangent that no kernel gives must not go missing.
inline bool dual(const Tensor &t) { return t._fw_grad(/*level=*/0).defined(); }

// t as rows with a dense last axis; false where that takes a copy.
inline bool as_rows(const Tensor &t, int64_t &rows, int64_t &cols, int64_t &stride) {
  if (t.dim() < 1) return false;
  cols = t.size(-1);
  if (cols < 1) return false;
  if (t.is_contiguous()) {
    rows = t.numel() / cols;
    stride = cols;
    return true;
  }
  if (t.dim() != 2 || t.stride(1) != 1) return false;
  rows = t.size(0);
  stride = t.stride(0);
  return true;
}

inline bool vector_of(const Tensor &t, int64_t n) {
  return t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}

inline const void *ptr(const OptTensor &t) { return t ? t->const_data_ptr() : nullptr; }

}  // namespace rxmet_torch
