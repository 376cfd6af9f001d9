// The norm of many gradients together, the factor that clips them to a limit,
// and clipping in place.
//
//   norm = sqrt(sum_i |g_i|^2),  factor = min(1, max_norm / (norm + eps)), 1 for 0 / 0
//
// Memory-bound: every gradient is read once (and written once where it is
// clipped).  A launch takes up to kTensors tensors by their addresses in its
// arguments and cuts each into chunks, one per workgroup, that finds its
// tensor as adamw_kernel does.  Squares are added in 64 bits: no gradient is
// too large or too small for them, and their order matters to no digit that
// is kept.  Each chunk's sum is stored, and one workgroup adds them up: no
// atomics, the same bits every time, and nothing to clear before a call.
#include <algorithm>
#include <cmath>

#include "maxsim_host.h"
#include "maxsim_rows.h"
#include "../../include/maxsim_amd_encoder.h"

namespace maxsim {

constexpr int kGradThreads = 256;
// A workgroup's share: 16-byte loads that a thread has in flight.  One turn of
// them (two: 64.5 us against 62.3 for 91 M fp32 gradients, multiplying them 134
// against 127, launches of either kind in a row; where the norm has just read
// them the multiplying takes 107), and shorter ones where there are few bytes,
// for more CUs (100000 bf16 gradients: the squares 3.5 us against 5.4, clipping
// 3.1 against 5.3).
template <int UNROLL_> struct Share {
  static constexpr int UNROLL = UNROLL_;
  static constexpr int64_t bytes = (int64_t)kGradThreads * 16 * UNROLL_;
};
using Large = Share<8>;
using Small = Share<2>;
constexpr int64_t kSmallBytes = 8 << 20;  // of all tensors together
constexpr int64_t kGradMaxChunks = UINT32_MAX / kGradThreads;  // of a launch: threads in 32 bits
constexpr int kJoinThreads = 1024;

struct GradArgs {
  static constexpr int kTensors = (4096 - 128) / 20;
  void* p[kTensors];
  uint64_t n[kTensors];      // 4 * elements + type
  uint32_t first[kTensors];  // number of the tensor's first chunk
  int count;
  double* sums;         // of the launch's chunks
  const float* factor;  // clipping in place
};
static_assert(sizeof(GradArgs) <= 4096, "kernel arguments");

// The last tensor that starts at or before this chunk.
__device__ __forceinline__ int tensor_of(const GradArgs& a, uint32_t chunk) {
  const int lane = threadIdx.x & 63;
  int k = -1;
#pragma unroll
  for (int i = 0; i < GradArgs::kTensors; i += 64)
    k += __popcll(__ballot(i + lane < a.count && a.first[min(i + lane, a.count - 1)] <= chunk));
  return k;
}

// Sum over the workgroup in every thread, lanes and then waves in one order.
template <int THREADS>
__device__ __forceinline__ double block_sum(double s) {
  __shared__ double waves[THREADS / 64];
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
  __syncthreads();
  s = waves[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) s += waves[w];
  return s;
}

// Squares of elements [at, end) of p, added up by thread t of THREADS.
template <typename T, int UNROLL, int THREADS>
__device__ __forceinline__ double squares(const void* p, int64_t at, int64_t end, int t) {
  constexpr int V = kVec<T>;
  const auto* g = static_cast<const typename T::storage*>(p);
  double s[2] = {0.0, 0.0};
  int64_t i = at + t * V;
  constexpr int64_t step = THREADS * V;
  for (; i + (UNROLL - 1) * step + V <= end; i += UNROLL * step) {
    Chunk<T> c[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) c[u] = load_any<Chunk<T>>(g + i + u * step);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float f[V];
      unpack<T>(c[u], f);
#pragma unroll
      for (int e = 0; e < V; ++e) s[e & 1] = fma((double)f[e], (double)f[e], s[e & 1]);
    }
  }
  for (; i < end; i += step) {
    if (i + V <= end) {
      float f[V];
      unpack<T>(load_any<Chunk<T>>(g + i), f);
#pragma unroll
      for (int e = 0; e < V; ++e) s[e & 1] = fma((double)f[e], (double)f[e], s[e & 1]);
    } else {
      for (int64_t e = i; e < end; ++e) {
        const double d = to_float<T>(g[e]);
        s[0] = fma(d, d, s[0]);
      }
    }
  }
  return s[0] + s[1];
}

// Those of a chunk of S::bytes.
template <typename S, int UNROLL, int THREADS>
__device__ __forceinline__ double chunk_squares(const GradArgs& a, uint32_t chunk, int t) {
  const int k = tensor_of(a, chunk);
  const int64_t n = (int64_t)(a.n[k] >> 2);
  const int type = (int)(a.n[k] & 3);
  const int64_t each = S::bytes / (type == MAXSIM_FLOAT32 ? 4 : 2);
  const int64_t at = (int64_t)(chunk - a.first[k]) * each, end = min(at + each, n);
  if (type == MAXSIM_FLOAT32) return squares<F32, UNROLL, THREADS>(a.p[k], at, end, t);
  if (type == MAXSIM_FLOAT16) return squares<F16, UNROLL, THREADS>(a.p[k], at, end, t);
  return squares<BF16, UNROLL, THREADS>(a.p[k], at, end, t);
}

template <typename S>
__global__ __launch_bounds__(kGradThreads) void grad_squares_kernel(GradArgs a) {
  const double s =
      block_sum<kGradThreads>(chunk_squares<S, S::UNROLL, kGradThreads>(a, blockIdx.x, threadIdx.x));
  if (threadIdx.x == 0) a.sums[blockIdx.x] = s;
}

__device__ __forceinline__ float clip_factor(double norm, double max_norm, double eps) {
  // gradients of zeros are within a limit of 0 too
  const double f = norm + eps == 0.0 ? 1.0 : max_norm / (norm + eps);
  return f > 1.0 ? 1.0f : (float)f;  // NaN stays
}
__device__ __forceinline__ void write_norm(double s, double max_norm, double eps, float* norm,
                                           float* factor) {
  if (threadIdx.x != 0) return;
  const double root = sqrt(s);
  *norm = (float)root;
  if (factor) *factor = clip_factor(root, max_norm, eps);
}

__global__ __launch_bounds__(kJoinThreads) void grad_norm_kernel(const double* __restrict__ sums,
                                                                 int64_t count, double max_norm,
                                                                 double eps, float* norm,
                                                                 float* factor) {
  double s = 0.0;
  constexpr int U = 8;
  for (int64_t i = threadIdx.x; i < count; i += kJoinThreads * U) {
    double v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = sums[min(i + u * kJoinThreads, count - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) s += i + u * kJoinThreads < count ? v[u] : 0.0;
  }
  write_norm(block_sum<kJoinThreads>(s), max_norm, eps, norm, factor);
}

// The norm of so few chunks in one launch of one workgroup, a wave a chunk.
constexpr uint32_t kFewChunks = 64;
__global__ __launch_bounds__(kJoinThreads) void grad_few_kernel(GradArgs a, uint32_t chunks,
                                                                double max_norm, double eps,
                                                                float* norm, float* factor) {
  double s = 0.0;
  for (uint32_t c = threadIdx.x >> 6; c < chunks; c += kJoinThreads / 64)
    s += chunk_squares<Small, Small::bytes / 1024, 64>(a, c, threadIdx.x & 63);
  write_norm(block_sum<kJoinThreads>(s), max_norm, eps, norm, factor);
}

template <typename T, int UNROLL>
__device__ __forceinline__ void scale_chunk(void* p, int64_t at, int64_t end, float factor) {
  constexpr int V = kVec<T>;
  auto* g = static_cast<typename T::storage*>(p);
  constexpr int64_t step = kGradThreads * V;
  int64_t i = at + threadIdx.x * V;
  auto scaled = [&](const Chunk<T>& c) {
    float f[V];
    unpack<T>(c, f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] *= factor;
    return pack<T>(f);
  };
  for (; i + (UNROLL - 1) * step + V <= end; i += UNROLL * step) {
    Chunk<T> c[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) c[u] = load_any<Chunk<T>>(g + i + u * step);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) store_any(g + i + u * step, scaled(c[u]));
  }
  for (; i < end; i += step) {
    if (i + V <= end) {
      store_any(g + i, scaled(load_any<Chunk<T>>(g + i)));
    } else {
      for (int64_t e = i; e < end; ++e) g[e] = from_float<T>(to_float<T>(g[e]) * factor);
    }
  }
}

template <typename S>
__global__ __launch_bounds__(kGradThreads) void grad_scale_kernel(GradArgs a) {
  const float factor = *a.factor;
  if (factor == 1.0f) return;  // every element stays what it is
  const int k = tensor_of(a, blockIdx.x);
  const int64_t n = (int64_t)(a.n[k] >> 2);
  const int type = (int)(a.n[k] & 3);
  const int64_t each = S::bytes / (type == MAXSIM_FLOAT32 ? 4 : 2);
  const int64_t at = (int64_t)(blockIdx.x - a.first[k]) * each, end = min(at + each, n);
  if (type == MAXSIM_FLOAT32) scale_chunk<F32, S::UNROLL>(a.p[k], at, end, factor);
  else if (type == MAXSIM_FLOAT16) scale_chunk<F16, S::UNROLL>(a.p[k], at, end, factor);
  else scale_chunk<BF16, S::UNROLL>(a.p[k], at, end, factor);
}

static int64_t grad_chunks(const maxsim_grad_tensor& t, int64_t bytes) {
  const int64_t each = bytes / (t.dtype == MAXSIM_FLOAT32 ? 4 : 2);
  return t.numel / each + (t.numel % each != 0);
}

// Bytes of a workgroup's share.
static int64_t grad_share(const maxsim_grad_tensor* tensors, int64_t count) {
  int64_t bytes = 0;
  for (int64_t i = 0; i < count && bytes <= kSmallBytes; ++i)
    bytes += std::min(tensors[i].numel, kSmallBytes) * (tensors[i].dtype == MAXSIM_FLOAT32 ? 4 : 2);
  return bytes <= kSmallBytes ? Small::bytes : Large::bytes;
}

static int check_grads(const maxsim_grad_tensor* tensors, int64_t count) {
  if (count < 0 || (count > 0 && !tensors)) return fail(MAXSIM_ERR_INVALID, "no tensors");
  for (int64_t i = 0; i < count; ++i) {
    if (int e = check_dtype(tensors[i].dtype)) return e;
    if (tensors[i].numel < 0) return fail(MAXSIM_ERR_INVALID, "negative size");
    if (tensors[i].numel > 0 && !tensors[i].grad)
      return fail(MAXSIM_ERR_INVALID, "null pointer argument");
    if (grad_chunks(tensors[i], Large::bytes) > kGradMaxChunks)
      return fail(MAXSIM_ERR_UNSUPPORTED, "tensor too large for one launch");
  }
  return MAXSIM_OK;
}

// Calls launch(arguments, chunks) for as many tensors as an argument list holds.
template <typename F>
static int for_grads(const maxsim_grad_tensor* tensors, int64_t count, int64_t share, F&& launch) {
  GradArgs a{};
  uint32_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    const maxsim_grad_tensor& t = tensors[i];
    if (t.numel == 0) continue;
    const uint32_t more = (uint32_t)grad_chunks(t, share);
    if (a.count == GradArgs::kTensors || (uint64_t)chunks + more > (uint64_t)kGradMaxChunks) {
      if (int e = launch(a, chunks)) return e;
      a.count = 0, chunks = 0;
    }
    const int k = a.count++;
    a.p[k] = t.grad, a.n[k] = (uint64_t)t.numel * 4 + (uint64_t)t.dtype, a.first[k] = chunks;
    chunks += more;
  }
  return a.count > 0 ? launch(a, chunks) : MAXSIM_OK;
}

// The norm and (or NULL) the factor, and clipping in place.
static int run_norm(const maxsim_grad_tensor* tensors, int64_t count, double max_norm, double eps,
                    float* norm, float* factor, bool clip, void* workspace, size_t workspace_bytes,
                    hipStream_t stream) {
  if (int e = check_grads(tensors, count)) return e;
  if (!norm) return fail(MAXSIM_ERR_INVALID, "null pointer argument");
  if (factor && (!(max_norm >= 0.0) || !(eps >= 0.0)))
    return fail(MAXSIM_ERR_INVALID, "max_norm and eps must be >= 0");
  const int64_t share = grad_share(tensors, count);
  int64_t all = 0, full = 0;  // sums, and tensors that have any
  for (int64_t i = 0; i < count; ++i) {
    all += grad_chunks(tensors[i], share);
    full += tensors[i].numel > 0;
  }
  if (all > 0 && (!workspace || workspace_bytes < (size_t)all * sizeof(double)))
    return fail(MAXSIM_ERR_INVALID, "workspace too small: %zu bytes, %zu needed", workspace_bytes,
                (size_t)all * sizeof(double));
  double* sums = static_cast<double*>(workspace);
  // few enough for one launch (100000 fp32 gradients of four tensors: 6.9 us a
  // call against 10.4)
  const bool few = share == Small::bytes && all > 0 && all <= kFewChunks &&
                   full <= GradArgs::kTensors;
  int64_t at = 0;
  int rc = for_grads(tensors, count, share, [&](GradArgs& a, uint32_t chunks) -> int {
    a.sums = sums + at;
    at += chunks;
    if (few)
      hipLaunchKernelGGL(grad_few_kernel, dim3(1), dim3(kJoinThreads), 0, stream, a, chunks, max_norm,
                         eps, norm, factor);
    else if (share == Small::bytes)
      hipLaunchKernelGGL(grad_squares_kernel<Small>, dim3(chunks), dim3(kGradThreads), 0, stream, a);
    else
      hipLaunchKernelGGL(grad_squares_kernel<Large>, dim3(chunks), dim3(kGradThreads), 0, stream, a);
    return check_launch("grad_squares_kernel");
  });
  if (rc == MAXSIM_OK && !few) {
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kJoinThreads), 0, stream, sums, all, max_norm,
                       eps, norm, factor);
    rc = check_launch("grad_norm_kernel");
  }
  if (rc != MAXSIM_OK || !clip) return rc;
  return for_grads(tensors, count, share, [&](GradArgs& a, uint32_t chunks) {
    a.factor = factor;
    if (share == Small::bytes)
      hipLaunchKernelGGL(grad_scale_kernel<Small>, dim3(chunks), dim3(kGradThreads), 0, stream, a);
    else
      hipLaunchKernelGGL(grad_scale_kernel<Large>, dim3(chunks), dim3(kGradThreads), 0, stream, a);
    return check_launch("grad_scale_kernel");
  });
}

}  // namespace maxsim

using namespace maxsim;

extern "C" {

size_t maxsim_amd_grad_norm_workspace_size(const maxsim_grad_tensor* tensors, int64_t count) {
  if (check_grads(tensors, count) != MAXSIM_OK) return 0;
  const int64_t share = grad_share(tensors, count);
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) chunks += grad_chunks(tensors[i], share);
  return (size_t)chunks * sizeof(double);
}

int maxsim_amd_grad_norm(const maxsim_grad_tensor* tensors, int64_t count, double max_norm,
                         double eps, float* norm, float* factor, void* workspace,
                         size_t workspace_bytes, void* stream) {
  clear_error();
  return run_norm(tensors, count, max_norm, eps, norm, factor, false, workspace, workspace_bytes,
                  static_cast<hipStream_t>(stream));
}

int maxsim_amd_clip_grads(const maxsim_grad_tensor* tensors, int64_t count, double max_norm,
                          double eps, float* norm, float* factor, void* workspace,
                          size_t workspace_bytes, void* stream) {
  clear_error();
  if (!factor) return fail(MAXSIM_ERR_INVALID, "null pointer argument");
  return run_norm(tensors, count, max_norm, eps, norm, factor, true, workspace, workspace_bytes,
                  static_cast<hipStream_t>(stream));
}

}  // extern "C"
