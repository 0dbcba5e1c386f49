// Gradient clipping, also called from Python without the dispatcher: turning
// two lists of 128 tensors into its arguments took half of a call's 43 us.
#pragma once

#include <ATen/ATen.h>

namespace flb200::aten {

at::Tensor GradNorm(at::TensorList grads, double norm_type);
at::Tensor ClipGradsOut(at::TensorList grads, double max_norm, double norm_type, at::TensorList out);

}  // namespace flb200::aten
