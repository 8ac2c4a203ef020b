// What the sources of the torch binding share: type codes, output allocation, status and tangent checks.
#pragma once

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>

#include <optional>

#include "ifa4.h"

namespace ifa4_torch {

inline int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return IFA4_BF16;
    case at::kHalf: return IFA4_FP16;
    case at::kFloat: return IFA4_FP32;
    default: return -1;
  }
}

// Uninitialised tensors on q's GPU from the caching allocator, without a dispatcher
// round per tensor (the output, the LSE and the workspace of a call: 9.4 -> 8.4 us
// of host time for a short prompt).  Where deterministic algorithms are on, through
// at::empty, which fills them: rows no sequence covers come back as it leaves them.
inline at::Tensor empty_on(const at::Tensor& q, at::IntArrayRef sizes, at::ScalarType dtype) {
  if (at::globalContext().deterministicAlgorithms())
    return at::empty(sizes, q.options().dtype(dtype).memory_format(at::MemoryFormat::Contiguous));
  return at::Tensor(at::detail::empty_cuda(sizes, dtype, q.device(), std::nullopt));
}

inline void check_status(int32_t st, const char* what) {
  TORCH_CHECK(st == IFA4_OK, "inkling_fa4.", what, ": ", ifa4_status_str(st));
}

// A tangent (forward-mode differentiation) is refused: below autograd it would vanish.
inline bool has_tangent(const at::Tensor& t) {
  return t.defined() && t._fw_grad(/*level=*/0).defined();
}
inline bool has_tangent(const std::optional<at::Tensor>& t) {
  return t.has_value() && has_tangent(*t);
}
template <typename... T>
void check_no_tangent(const char* op, const T&... inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(inputs) || ...), "inkling_fa4.", op,
                              ": no forward-mode derivative");
}

}  // namespace ifa4_torch
