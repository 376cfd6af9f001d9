// Layer norm over the last axis, forward and backward.
//
//   mu = mean(x), s = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) s
//   y  = xh w + b
//   g  = dy w
//   dx = s (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Memory-bound: the forward reads and writes each element once, the backward
// reads x and dy and writes dx, at under 20 operations per element.  A row
// stays in the registers of one group of lanes (maxsim_rows.h), so the mean
// and then the squared distances from it are taken from the one read: no
// difference of large sums.  Statistics, sums and the weights' gradients are
// fp32; y, dx, dw and db are rounded once, to nearest even.
#include <algorithm>

#include "maxsim_host.h"
#include "maxsim_rows.h"
#include "../../include/maxsim_amd_training.h"

namespace maxsim {

struct LnForward {
  const void* x;
  int64_t rows, stride;  // stride: elements from row to row of x
  int dim;
  const void* weight;
  const void* bias;
  float eps;
  void* y;
  float* mean;  // both or neither
  float* rstd;
};

// Workgroups that take the rows in turn, each group of lanes with its weights
// in registers for all its rows and the next row's loads in flight.
template <typename T, typename W, int G, int K>
__global__ __launch_bounds__(row_threads(G)) void ln_forward_kernel(LnForward a) {
  using S = typename T::storage;
  constexpr int V = kVec<T>, GROUPS = row_threads(G) / G;
  __shared__ float part[2][G > 64 ? G / 64 : 1];
  const int j = threadIdx.x % G, group = threadIdx.x / G;
  const int dim = a.dim;
  const S* x = static_cast<const S*>(a.x);
  S* y = static_cast<S*>(a.y);
  const float inv_dim = 1.0f / (float)dim;
  const bool whole = dim == G * K * V;

  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group;
  Chunk<T> next[K] = {};
  if (row < a.rows) {
#pragma unroll
    for (int k = 0; k < K; ++k) next[k] = load_chunk<T, takes_short(G)>(x + row * a.stride, (j + k * G) * V, dim);
  }
  float w[K][V], b[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load_param<W, V>(a.weight, (j + k * G) * V, dim, 1.0f, w[k]);
    load_param<W, V>(a.bias, (j + k * G) * V, dim, 0.0f, b[k]);
  }
  // the workgroup's groups stay together: the reductions need every lane
  for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < a.rows; base += step, row += step) {
    float f[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!whole) place_chunk<T, takes_short(G)>(next[k], (j + k * G) * V, dim);
      unpack<T>(next[k], f[k]);
    }
    if (row + step < a.rows) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        next[k] = load_chunk<T, takes_short(G)>(x + (row + step) * a.stride, (j + k * G) * V, dim);
    }
    float sum[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) sum[0] += f[k][e];
    group_sums<G>(sum, part[0]);
    const float mean = sum[0] * inv_dim;
    float sq[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[k][e] -= mean;
        sq[0] += (j + k * G) * V + e < dim ? f[k][e] * f[k][e] : 0.0f;
      }
    group_sums<G>(sq, part[1]);
    const float rstd = 1.0f / sqrtf(sq[0] * inv_dim + a.eps);
    if (row < a.rows) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[k][e] = f[k][e] * rstd * w[k][e] + b[k][e];
        store_chunk<T>(y + row * dim, (j + k * G) * V, dim, f[k]);
      }
      if (a.mean && j == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
      }
    }
  }
}

struct LnBackward {
  const void* dy;
  const void* x;
  int64_t rows, dy_stride, x_stride;
  int dim;
  const float* mean;
  const float* rstd;
  const void* weight;
  void* dx;        // NULL: not wanted
  float* partial;  // [gridDim.x][2][dim] sums of dy xh and dy; NULL: not wanted
};

// The rows in turn as in the forward; each lane adds up its columns' share of
// dw and db over its rows, the workgroup joins its groups' (in one order) and
// writes one partial row, which ln_weight_grad_kernel adds up.  Chunks of 16
// bytes cost 16-bit rows 200 registers, two waves per SIMD, and still win
// (294912 x 768 bf16 235 us = 5.8 TB/s, in chunks of 8 bytes 255).
template <typename T, typename W, int G, int K>
__global__ __launch_bounds__(row_threads(G)) void ln_backward_kernel(LnBackward a) {
  using S = typename T::storage;
  constexpr int V = kVec<T>, GROUPS = row_threads(G) / G;
  constexpr int COLS = G * K * V;
  // lanes of 1024 threads have 128 registers, too few for the next row and the
  // weights besides: both are loaded where they are used (10000 x 8192 fp32 185
  // us, with them kept 190)
  constexpr bool AHEAD = G < 1024;
  __shared__ float part[2][G > 64 ? 2 * G / 64 : 1];
  __shared__ alignas(16) float cols[G < 256 ? row_threads(G) / 64 : 1][G < 256 ? COLS : 4];
  const int j = threadIdx.x % G, group = threadIdx.x / G;
  const int dim = a.dim;
  const S* x = static_cast<const S*>(a.x);
  const S* dy = static_cast<const S*>(a.dy);
  S* dx = static_cast<S*>(a.dx);
  const float inv_dim = 1.0f / (float)dim;
  const bool whole = dim == G * K * V;

  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group;
  Chunk<T> next_x[K] = {}, next_d[K] = {};
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto load = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      next_x[k] = load_chunk<T, takes_short(G)>(x + r * a.x_stride, (j + k * G) * V, dim);
      next_d[k] = load_chunk<T, takes_short(G)>(dy + r * a.dy_stride, (j + k * G) * V, dim);
    }
    next_mean = a.mean[r];
    next_rstd = a.rstd[r];
  };
  if (AHEAD && row < a.rows) load(row);
  float w[AHEAD ? K : 1][V], dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if constexpr (AHEAD) load_param<W, V>(a.weight, (j + k * G) * V, dim, 1.0f, w[k]);
#pragma unroll
    for (int e = 0; e < V; ++e) dw[k][e] = db[k][e] = 0.0f;
  }
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < a.rows; base += step, row += step) {
    float f[K][V], d[K][V];
    if constexpr (!AHEAD) {
      asm volatile("" ::: "memory");  // the weights are not kept over the rows
      load(row);
    }
    const float mean = next_mean, rstd = next_rstd;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!whole) {
        place_chunk<T, takes_short(G)>(next_x[k], (j + k * G) * V, dim);
        place_chunk<T, takes_short(G)>(next_d[k], (j + k * G) * V, dim);
      }
      unpack<T>(next_x[k], f[k]);
      unpack<T>(next_d[k], d[k]);
    }
    const bool here = row < a.rows;
    if (AHEAD && row + step < a.rows) load(row + step);
    float sums[2] = {0.0f, 0.0f};
    // past the row's end dy and w are 0; a group without a row adds nothing
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float(&wk)[V] = w[AHEAD ? k : 0];
      if constexpr (!AHEAD) load_param<W, V>(a.weight, (j + k * G) * V, dim, 1.0f, wk);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[k][e] = (f[k][e] - mean) * rstd;
        if (here) {
          dw[k][e] += d[k][e] * f[k][e];
          db[k][e] += d[k][e];
        }
        d[k][e] *= wk[e];
        sums[0] += d[k][e];
        sums[1] += d[k][e] * f[k][e];
      }
    }
    if (dx) {
      group_sums<G>(sums, part[turn]);
      turn ^= 1;
      if (here) {
        const float c1 = sums[0] * inv_dim, c2 = sums[1] * inv_dim;
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
          for (int e = 0; e < V; ++e) f[k][e] = rstd * (d[k][e] - c1 - f[k][e] * c2);
          store_chunk<T>(dx + row * dim, (j + k * G) * V, dim, f[k]);
        }
      }
    }
  }
  if (!a.partial) return;
  float* out = a.partial + (int64_t)blockIdx.x * 2 * dim;
  auto write = [&](float (&v)[K][V], float* to) {
    if constexpr (G < 256) {
      // a wave's groups in registers, the waves in LDS
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[k][e] = groups_sum<G>(v[k][e]);
        if ((threadIdx.x & 63) < G) {
#pragma unroll
          for (int e = 0; e < V; ++e) cols[threadIdx.x >> 6][(j + k * G) * V + e] = v[k][e];
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < dim; c += row_threads(G)) {
        float sum = cols[0][c];
#pragma unroll
        for (int wave = 1; wave < row_threads(G) / 64; ++wave) sum += cols[wave][c];
        to[c] = sum;
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (j + k * G) * V;
        if (c + V <= dim) {
          __builtin_memcpy(to + c, v[k], sizeof v[k]);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (c + e < dim) to[c + e] = v[k][e];
        }
      }
    }
  };
  write(dw, out);
  write(db, out + dim);
}

// dw and db from the partial rows: a workgroup takes 32 columns of one of the
// two, and each 32 of its threads every 32nd partial row, joined in LDS in one
// order.
constexpr int kGradCols = 32, kGradSlices = 32;
template <typename W>
__global__ __launch_bounds__(kGradCols * kGradSlices) void ln_weight_grad_kernel(
    const float* __restrict__ partial, int count, int dim, void* dweight, void* dbias) {
  __shared__ float part[kGradSlices][kGradCols + 1];
  const int col = threadIdx.x % kGradCols, slice = threadIdx.x / kGradCols;
  const int c = blockIdx.x * kGradCols + col, which = blockIdx.y;
  float s = 0.0f;
  if (c < dim) {
    const float* p = partial + (int64_t)which * dim + c;
    // eight rows asked for at a time, also at the end
    for (int i = slice; i < count; i += 8 * kGradSlices) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = p[(int64_t)min(i + u * kGradSlices, count - 1) * 2 * dim];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += i + u * kGradSlices < count ? v[u] : 0.0f;
    }
  }
  part[slice][col] = s;
  __syncthreads();
  // a wave takes two columns: each half adds one's 32 slices
  const int row = threadIdx.x & 31, column = threadIdx.x >> 5;
  s = lanes_sum<32>(part[row][column]);
  const int at = blockIdx.x * kGradCols + column;
  auto* out = static_cast<typename W::storage*>(which ? dbias : dweight);
  if (row == 0 && at < dim && out) out[at] = from_float<W>(s);
}

template <typename F>
static void with_types(maxsim_dtype t, maxsim_dtype w, F&& f) {
  if (t == MAXSIM_FLOAT32) f(F32{}, F32{});
  else if (t == MAXSIM_FLOAT16 && w == MAXSIM_FLOAT16) f(F16{}, F16{});
  else if (t == MAXSIM_FLOAT16) f(F16{}, F32{});
  else if (w == MAXSIM_BFLOAT16) f(BF16{}, BF16{});
  else f(BF16{}, F32{});
}

static int check_layer_norm(maxsim_dtype dtype, maxsim_dtype weight_dtype, int64_t rows,
                            int64_t dim) {
  if (int e = check_dtype(dtype)) return e;
  if (int e = check_dtype(weight_dtype)) return e;
  if (weight_dtype != dtype && weight_dtype != MAXSIM_FLOAT32)
    return fail(MAXSIM_ERR_INVALID, "weight_dtype must be the rows' dtype or float32");
  if (rows < 0) return fail(MAXSIM_ERR_INVALID, "negative size");
  return check_dim(dim);
}

// Workgroups take their rows in turn, with this turn's and the next's rows
// asked for; how many there are per CU sets how much is in flight.  Past 32 KB
// per CU (forward, one array) and 48 KB (backward, two) more only gets into
// each other's way in the memory: 294912 x 768 bf16 backward 235 / 254 us with
// 48 / 72 KB, 65000 x 1024 76 / 82, 100000 x 768 fp32 161 / 177 with 48 / 96.
constexpr int64_t kForwardInFlight = 32 << 10, kBackwardInFlight = 48 << 10;
static int workgroups_for(int64_t in_flight, int64_t bytes_each) {
  return (int)((in_flight + bytes_each - 1) / bytes_each);
}

// Workgroups of the backward, at most kMaxPartials (what the workspace holds
// partial rows for) and with at least kLeastTurns turns each where there are
// more turns than CUs: a workgroup costs a partial row of 8 dim bytes, written
// and read again.  Four is no sharp optimum: 18433 x 301 fp32 takes 17.7 us
// with four and 19.0 with eight, 2049 x 2560 bf16 15.9 and 16.9, 16000 x 768
// 18.8 with either, and 4000 x 2048 is better with eight, 16.4 and 15.2.  How
// evenly the turns divide, which this rule does not look at, counts as much.
constexpr int64_t kMaxPartials = 1024;
constexpr int64_t kLeastTurns = 4;
static int64_t backward_blocks(int64_t turns, int64_t cus, int64_t per_cu) {
  return std::min<int64_t>({turns, cus * per_cu, kMaxPartials,
                            std::max<int64_t>(cus, turns / kLeastTurns)});
}

template <typename F>
static void with_backward(maxsim_dtype dtype, maxsim_dtype weight_dtype, int64_t dim, F&& f) {
  with_types(dtype, weight_dtype, [&](auto t, auto w) {
    with_shape<kVec<decltype(t)>>(dim, [&](auto s) { f(t, w, s); });
  });
}

}  // namespace maxsim

using namespace maxsim;

extern "C" {

int maxsim_amd_layer_norm_forward(maxsim_dtype dtype, maxsim_dtype weight_dtype, const void* x,
                                  int64_t rows, int64_t dim, int64_t row_stride,
                                  const void* weight, const void* bias, float eps, void* y,
                                  float* mean, float* rstd, void* stream) {
  clear_error();
  if (int e = check_layer_norm(dtype, weight_dtype, rows, dim)) return e;
  if (!(eps >= 0.0f)) return fail(MAXSIM_ERR_INVALID, "eps must be >= 0");
  if (row_stride < 0) return fail(MAXSIM_ERR_INVALID, "negative row stride");
  if (rows == 0) return MAXSIM_OK;
  if (!x || !y || !mean != !rstd) return fail(MAXSIM_ERR_INVALID, "null pointer argument");
  const LnForward a{x, rows, row_stride, (int)dim, weight, bias, eps, y, mean, rstd};
  with_types(dtype, weight_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    with_shape<kVec<T>>(dim, [&](auto s) {
      constexpr int G = decltype(s)::G, K = decltype(s)::K, threads = row_threads(G);
      const auto kernel = ln_forward_kernel<T, decltype(w), G, K>;
      static std::atomic<int> resident[kMaxDevices];
      const int64_t turns = (rows + threads / G - 1) / (threads / G);
      // rows wider than a wave: two at least, one to run at the other's barriers
      // (10000 x 8192 bf16: 64 us against 78 with one)
      const int per_cu = std::min<int>(
          resident_per_cu(reinterpret_cast<const void*>(kernel), threads, 0, resident),
          std::max(G > 64 ? 2 : 1,
                   workgroups_for(kForwardInFlight, 2 * (threads / G) * dim * T::bytes)));
      const int64_t blocks = std::min<int64_t>(turns, (int64_t)device_cus() * per_cu);
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0,
                         static_cast<hipStream_t>(stream), a);
    });
  });
  return check_launch("ln_forward_kernel");
}

size_t maxsim_amd_layer_norm_backward_workspace_size(maxsim_dtype dtype, int64_t rows,
                                                     int64_t dim) {
  if (rows <= 0 || dim <= 0 || dim > MAXSIM_AMD_MAX_DIM) return 0;
  int64_t turns = 0;
  with_backward(dtype, dtype, dim, [&](auto, auto, auto s) {
    constexpr int groups = row_threads(decltype(s)::G) / decltype(s)::G;
    turns = (rows + groups - 1) / groups;
  });
  return (size_t)std::min(turns, kMaxPartials) * 2 * dim * sizeof(float);
}

int maxsim_amd_layer_norm_backward(maxsim_dtype dtype, maxsim_dtype weight_dtype, const void* dy,
                                   int64_t dy_stride, const void* x, int64_t x_stride,
                                   const float* mean, const float* rstd, const void* weight,
                                   int64_t rows, int64_t dim, void* dx, void* dweight,
                                   void* dbias, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  clear_error();
  if (int e = check_layer_norm(dtype, weight_dtype, rows, dim)) return e;
  if (dy_stride < 0 || x_stride < 0) return fail(MAXSIM_ERR_INVALID, "negative row stride");
  if (rows > 0 && (!dy || !x || !mean || !rstd))
    return fail(MAXSIM_ERR_INVALID, "null pointer argument");
  const bool weights = dweight || dbias;
  if (!dx && !weights) return MAXSIM_OK;
  if (weights && rows > 0 &&
      (!workspace ||
       workspace_bytes < maxsim_amd_layer_norm_backward_workspace_size(dtype, rows, dim)))
    return fail(MAXSIM_ERR_INVALID,
                "the weights' gradients need a workspace of "
                "maxsim_amd_layer_norm_backward_workspace_size() bytes");
  float* partial = weights ? static_cast<float*>(workspace) : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  int64_t blocks = 0;
  if (rows > 0) {
    const LnBackward a{dy, x, rows, dy_stride, x_stride, (int)dim, mean, rstd, weight, dx, partial};
    with_backward(dtype, weight_dtype, dim, [&](auto t, auto w, auto s) {
      constexpr int G = decltype(s)::G, threads = row_threads(G);
      const auto kernel = ln_backward_kernel<decltype(t), decltype(w), G, decltype(s)::K>;
      static std::atomic<int> resident[kMaxDevices];
      const int per_cu = std::min<int>(
          resident_per_cu(reinterpret_cast<const void*>(kernel), threads, 0, resident),
          workgroups_for(kBackwardInFlight, 4 * (threads / G) * dim * decltype(t)::bytes));
      blocks = backward_blocks((rows + threads / G - 1) / (threads / G), device_cus(), per_cu);
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, st, a);
    });
    if (int e = check_launch("ln_backward_kernel")) return e;
  }
  if (!weights) return MAXSIM_OK;
  with_types(dtype, weight_dtype, [&](auto, auto w) {
    hipLaunchKernelGGL((ln_weight_grad_kernel<decltype(w)>), dim3((unsigned)((dim + kGradCols - 1) / kGradCols), 2),
                       dim3(kGradCols * kGradSlices), 0, st, partial, (int)blocks, (int)dim, dweight,
                       dbias);
  });
  return check_launch("ln_weight_grad_kernel");
}

}  // extern "C"
