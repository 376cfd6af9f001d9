// Helpers that the torch binding's files share.
#pragma once

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include "../../include/maxsim_amd.h"

namespace maxsim_torch {

inline void check_status(int rc) {
  TORCH_CHECK(rc == MAXSIM_OK, "maxsim_amd: ", maxsim_amd_last_error());
}

inline void* current_stream(const at::Tensor& t) {
  return reinterpret_cast<void*>(
      c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream());
}

inline at::TensorOptions f32_opts(const at::Tensor& t) {
  return at::TensorOptions().dtype(at::kFloat).device(t.device());
}
inline at::TensorOptions i32_opts(const at::Tensor& t) {
  return at::TensorOptions().dtype(at::kInt).device(t.device());
}

}  // namespace maxsim_torch
