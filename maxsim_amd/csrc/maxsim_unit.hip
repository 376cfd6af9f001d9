// Token embeddings of unit length, padded or packed on the way, forward and
// backward, and the offsets of packed sequences.
//
//   y  = x / max(|x|, eps)
//   dx = (dy - y <y, dy>) / |x| where |x| > eps, dy / eps below
//
// x is [sequences, length, dim]; with `lengths`, the tokens behind a
// sequence's length are not read: y and dx are 0 there, or y has no row for
// them (packed: sequence s starts at row offsets[s]).
//
// Memory-bound: each row is read once into one group of lanes
// (maxsim_rows.h).  The backward takes |x| from x again instead of reading
// the rounded y and a saved norm: the same bytes, and nothing is saved.  Sums
// are fp32, y and dx are rounded once, to nearest even.
#include <algorithm>

#include "maxsim_host.h"
#include "maxsim_rows.h"
#include "../../include/maxsim_amd_training.h"

namespace maxsim {

struct UnitRows {
  const void* x;
  const void* dy;  // backward only
  int64_t x_seq, x_row, dy_seq, dy_row;  // strides in elements (dy: padded only)
  int64_t rows;                          // sequences * length
  int length, dim;
  const int32_t* lengths;  // NULL: every token is real
  const int32_t* offsets;  // NULL: padded
  int64_t packed_rows;
  float eps;
  void* out;  // y or dx
};

// Where row r of the padded layout is, and whether it is a real token.
struct Place {
  int64_t seq;
  int t;
  bool real;
  int64_t packed;
};
__device__ __forceinline__ Place place_of(const UnitRows& a, int64_t r) {
  Place p;
  p.seq = r / a.length;
  p.t = (int)(r - p.seq * a.length);
  p.real = !a.lengths || p.t < a.lengths[p.seq];
  p.packed = 0;
  if (a.offsets) {
    p.packed = (int64_t)a.offsets[p.seq] + p.t;
    p.real = p.real && p.packed >= 0 && p.packed < a.packed_rows;
  }
  return p;
}

template <typename T, int G, int K, bool BACKWARD>
__global__ __launch_bounds__(row_threads(G)) void unit_rows_kernel(UnitRows a) {
  using S = typename T::storage;
  constexpr int V = kVec<T>, GROUPS = row_threads(G) / G;
  constexpr int SUMS = BACKWARD ? 2 : 1;
  __shared__ float part[2][G > 64 ? SUMS * G / 64 : 1];
  const int j = threadIdx.x % G, group = threadIdx.x / G;
  const int dim = a.dim;
  const S* x = static_cast<const S*>(a.x);
  const S* dy = static_cast<const S*>(a.dy);
  S* out = static_cast<S*>(a.out);

  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group;
  uint4 next_x[K], next_d[K];
  Place next;
  auto load = [&](int64_t r) {
    next.real = false;
    if (r < a.rows) next = place_of(a, r);
    const S* xr = x + next.seq * a.x_seq + next.t * a.x_row;
    const S* dr = !BACKWARD ? nullptr
                  : a.offsets ? dy + next.packed * dim
                              : dy + next.seq * a.dy_seq + next.t * a.dy_row;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      next_x[k] = next.real ? load_chunk<T>(xr, (j + k * G) * V, dim) : make_uint4(0, 0, 0, 0);
      if constexpr (BACKWARD)
        next_d[k] = next.real ? load_chunk<T>(dr, (j + k * G) * V, dim) : make_uint4(0, 0, 0, 0);
    }
  };
  next.seq = 0, next.t = 0, next.packed = 0;
  load(row);
  int turn = 0;
  // the workgroup's groups stay together: the reductions need every lane
  for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < a.rows; base += step, row += step) {
    float f[K][V], d[K][V];
    const Place at = next;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      unpack16<T>(next_x[k], f[k]);
      if constexpr (BACKWARD) unpack16<T>(next_d[k], d[k]);
    }
    load(row + step);
    float sums[SUMS] = {};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        sums[0] += f[k][e] * f[k][e];
        if constexpr (BACKWARD) sums[1] += f[k][e] * d[k][e];
      }
    group_sums<G>(sums, part[turn]);
    turn ^= 1;
    if (row >= a.rows) continue;
    const float norm = sqrtf(sums[0]);
    const float inv = 1.0f / fmaxf(norm, a.eps);
    if constexpr (BACKWARD) {
      // y <y, dy> / |x| = x <x, dy> / |x|^3; a NaN norm stays NaN
      const float along = norm <= a.eps ? 0.0f : sums[1] * inv * inv;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < V; ++e)
          f[k][e] = at.real ? (d[k][e] - f[k][e] * along) * inv : 0.0f;
        store_chunk<T>(out + row * dim, (j + k * G) * V, dim, f[k]);
      }
    } else {
      if (a.offsets && !at.real) continue;
      const float scale = norm != norm ? norm : inv;
      S* to = out + (a.offsets ? at.packed : row) * dim;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[k][e] = at.real ? f[k][e] * scale : 0.0f;
        store_chunk<T>(to, (j + k * G) * V, dim, f[k]);
      }
    }
  }
}

// offsets[s] = sum of the lengths before s, each clamped to [0, max_len];
// offsets[n] the total.  One workgroup: a batch has few thousand sequences,
// and a thread's share is added in registers between two passes over them.
constexpr int kScanThreads = 1024;
__global__ __launch_bounds__(kScanThreads) void length_offsets_kernel(
    const int32_t* __restrict__ lengths, int64_t n, int32_t max_len, int32_t* __restrict__ clamped,
    int32_t* __restrict__ offsets) {
  __shared__ int32_t part[kScanThreads];
  __shared__ int32_t carried;
  const int t = threadIdx.x;
  if (t == 0) carried = 0;
  __syncthreads();
  for (int64_t base = 0; base < n; base += kScanThreads) {
    const int64_t i = base + t;
    const int32_t len = i < n ? min(max(lengths[i], 0), max_len) : 0;
    part[t] = len;
    __syncthreads();
    for (int off = 1; off < kScanThreads; off <<= 1) {
      const int32_t before = t >= off ? part[t - off] : 0;
      __syncthreads();
      part[t] += before;
      __syncthreads();
    }
    const int32_t start = carried;
    if (i < n) {
      clamped[i] = len;
      offsets[i] = start + part[t] - len;
      if (i == n - 1) offsets[n] = start + part[t];
    }
    __syncthreads();
    if (t == kScanThreads - 1) carried = start + part[t];
    __syncthreads();
  }
  if (n == 0 && t == 0) offsets[0] = 0;
}

template <bool BACKWARD>
static int run_unit_rows(maxsim_dtype dtype, const UnitRows& a, void* stream) {
  auto go = [&](auto t) {
    using T = decltype(t);
    with_shape<T>(a.dim, [&](auto s) {
      constexpr int G = decltype(s)::G, K = decltype(s)::K, threads = row_threads(G);
      const int64_t need = (a.rows + threads / G - 1) / (threads / G);
      const int64_t blocks = std::min<int64_t>(need, (int64_t)device_cus() * (2048 / threads));
      hipLaunchKernelGGL((unit_rows_kernel<T, G, K, BACKWARD>), dim3((unsigned)blocks),
                         dim3(threads), 0, static_cast<hipStream_t>(stream), a);
    });
  };
  if (dtype == MAXSIM_FLOAT32) go(F32{});
  else if (dtype == MAXSIM_FLOAT16) go(F16{});
  else go(BF16{});
  return check_launch("unit_rows_kernel");
}

static int check_unit_rows(maxsim_dtype dtype, int64_t sequences, int64_t length, int64_t dim,
                           const int32_t* lengths, const int32_t* offsets, int64_t packed_rows,
                           float eps) {
  if (int e = check_dtype(dtype)) return e;
  if (int e = check_dim(dim)) return e;
  if (sequences < 0 || length < 0 || packed_rows < 0)
    return fail(MAXSIM_ERR_INVALID, "negative size");
  if (length > INT32_MAX) return fail(MAXSIM_ERR_UNSUPPORTED, "length exceeds 2^31 - 1");
  if (!(eps > 0.0f)) return fail(MAXSIM_ERR_INVALID, "eps must be > 0");
  if (sequences > 0 && offsets && !lengths)
    return fail(MAXSIM_ERR_INVALID, "offsets without lengths");
  return MAXSIM_OK;
}

}  // namespace maxsim

using namespace maxsim;

extern "C" {

int maxsim_amd_unit_rows_forward(maxsim_dtype dtype, const void* x, int64_t sequences,
                                 int64_t length, int64_t dim, int64_t x_seq_stride,
                                 int64_t x_row_stride, const int32_t* lengths,
                                 const int32_t* offsets, int64_t packed_rows, float eps, void* y,
                                 void* stream) {
  clear_error();
  if (int e = check_unit_rows(dtype, sequences, length, dim, lengths, offsets, packed_rows, eps))
    return e;
  if (x_seq_stride < 0 || x_row_stride < 0) return fail(MAXSIM_ERR_INVALID, "negative stride");
  if (sequences == 0 || length == 0 || (offsets && packed_rows == 0)) return MAXSIM_OK;
  if (!x || !y) return fail(MAXSIM_ERR_INVALID, "null pointer argument");
  const UnitRows a{x,           nullptr, x_seq_stride, x_row_stride, 0,           0,
                   sequences * length, (int)length, (int)dim, lengths, offsets, packed_rows, eps, y};
  return run_unit_rows<false>(dtype, a, stream);
}

int maxsim_amd_unit_rows_backward(maxsim_dtype dtype, const void* dy, int64_t dy_seq_stride,
                                  int64_t dy_row_stride, const void* x, int64_t sequences,
                                  int64_t length, int64_t dim, int64_t x_seq_stride,
                                  int64_t x_row_stride, const int32_t* lengths,
                                  const int32_t* offsets, int64_t packed_rows, float eps, void* dx,
                                  void* stream) {
  clear_error();
  if (int e = check_unit_rows(dtype, sequences, length, dim, lengths, offsets, packed_rows, eps))
    return e;
  if (x_seq_stride < 0 || x_row_stride < 0 || dy_seq_stride < 0 || dy_row_stride < 0)
    return fail(MAXSIM_ERR_INVALID, "negative stride");
  if (sequences == 0 || length == 0) return MAXSIM_OK;
  if (!x || !dx || (!dy && !(offsets && packed_rows == 0)))
    return fail(MAXSIM_ERR_INVALID, "null pointer argument");
  const UnitRows a{x,       dy,          x_seq_stride, x_row_stride, dy_seq_stride, dy_row_stride,
                   sequences * length, (int)length, (int)dim, lengths, offsets, packed_rows, eps, dx};
  return run_unit_rows<true>(dtype, a, stream);
}

int maxsim_amd_length_offsets(const int32_t* lengths, int64_t sequences, int64_t max_len,
                              int32_t* clamped, int32_t* offsets, void* stream) {
  clear_error();
  if (sequences < 0 || max_len < 0) return fail(MAXSIM_ERR_INVALID, "negative size");
  if (max_len > 0 && sequences > INT32_MAX / max_len)
    return fail(MAXSIM_ERR_UNSUPPORTED, "more than 2^31 - 1 padded rows: offsets are int32");
  if (!offsets || (sequences > 0 && (!lengths || !clamped)))
    return fail(MAXSIM_ERR_INVALID, "null pointer argument");
  hipLaunchKernelGGL(length_offsets_kernel, dim3(1), dim3(kScanThreads), 0,
                     static_cast<hipStream_t>(stream), lengths, sequences, (int32_t)max_len,
                     clamped, offsets);
  return check_launch("length_offsets_kernel");
}

}  // extern "C"
