// Helpers shared by the flagos:: op files.
#pragma once

#include <ATen/core/dispatch/Dispatcher.h>

#include "tensor_utils.h"

namespace flb200::aten {

inline int FloatCode(const at::Tensor& t, const char* op) {
  const int c = B200Dtype(t.scalar_type());
  TORCH_CHECK(c == FL_B200_F32 || c == FL_B200_BF16 || c == FL_B200_F16, op,
              ": float32, bfloat16 or float16 expected, got ", t.scalar_type());
  return c;
}

inline void SameDevice(const at::Tensor& a, const at::Tensor& b, const char* op) {
  TORCH_CHECK(a.device() == b.device(), op, ": tensors on ", a.device(), " and ", b.device());
}

inline RowsView Rows(const at::Tensor& x, at::Tensor& keep) {
  auto r = AsRows(x);
  if (r) {
    keep = x;
    return *r;
  }
  keep = x.contiguous();
  return *AsRows(keep);
}

// The handle of the op `name` with signature Fn, looked up once at each place
// that names it: the lambda, and so its static, is that place's own, and ops
// of one signature do not share a handle.
#define FLB_OP(Fn, name)                                                                                   \
  ([]() -> const c10::TypedOperatorHandle<Fn>& {                                                           \
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Fn>();           \
    return op;                                                                                             \
  }())
// There is no forward-mode formula: a tangent would be dropped unseen.
inline void NoTangent(const at::Tensor& t, const char* op) {
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), op, ": forward-mode derivatives are not there");
}

}  // namespace flb200::aten
