// Helpers that the torch binding's files share.
#pragma once

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <chrono>

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

// Whether `stream` is being captured into a graph (or cannot tell).
inline bool capturing(hipStream_t stream) {
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  const hipError_t asked = hipStreamIsCapturing(stream, &capture);
  if (asked != hipSuccess) (void)hipGetLastError();
  return asked != hipSuccess || capture != hipStreamCaptureStatusNone;
}

// Waits until a kernel queued on `stream` has set bit 0 of the word of pinned
// memory at `w`, and returns the word.  Polls it, and the stream every 100 ms
// (a query puts a marker into it), so that an error there, or a stream that
// ended without the word, ends the wait.
inline int64_t wait_for_word(const int64_t* w, hipStream_t stream, const char* what) {
  constexpr std::chrono::milliseconds kLook{100};
  auto look = std::chrono::steady_clock::now() + kLook;
  bool drained = false;
  for (int64_t spins = 1;; ++spins) {
    const int64_t v = __atomic_load_n(w, __ATOMIC_ACQUIRE);
    if (v & 1) return v;
    TORCH_CHECK(!drained, "maxsim_amd: ", what, " did not report");
    if (spins % 4096 == 0 && std::chrono::steady_clock::now() >= look) {
      look = std::chrono::steady_clock::now() + kLook;
      const hipError_t e = hipStreamQuery(stream);
      if (e == hipErrorNotReady) {
        (void)hipGetLastError();
      } else {
        TORCH_CHECK(e == hipSuccess, "maxsim_amd: HIP error: ", hipGetErrorString(e));
        drained = true;  // one more look
      }
    } else {
      __builtin_ia32_pause();
    }
  }
}

}  // namespace maxsim_torch
