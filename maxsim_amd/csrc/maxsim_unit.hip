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
// are fp32, y and dx are rounded once, to nearest even.  A row whose squares
// leave fp32 (longer than 2^63, or shorter than 2^-45 beside an eps that is
// too) is moved to where they do not, by a power of two: rescale_row.
#include <algorithm>
#include <cfloat>

#include "maxsim_host.h"
#include "maxsim_rows.h"
#include "../../include/maxsim_amd_training.h"

namespace maxsim {

struct UnitRows {
  const void* x;
  const void* dy;  // backward only
  int64_t x_seq, x_row, dy_seq, dy_row;  // strides in elements (dy: padded only)
  int64_t sequences, rows;               // rows: sequences * length
  int64_t begin;                         // first row of this launch
  int length, dim;
  const void* lengths;  // int32, or int64; NULL: every token is real
  int lengths64;
  const int32_t* offsets;  // NULL: padded
  int64_t packed_rows;
  float eps;
  float least;  // squares' sums below it are not trusted
  void* out;    // y or dx
};

// Sums of squares, and products, above this may have passed fp32's largest
// number on the way or be about to.
constexpr float kMostSquares = 0x1p126f;
// fp16's squares stay far from both.
template <typename T> constexpr bool kWideRange = true;
template <> constexpr bool kWideRange<F16> = false;
// Sums of squares below this have lost part of themselves to fp32's smallest
// one.  No loss where eps is larger than their root: the quotient is by eps.
constexpr float kLeastSquares = 0x1p-90f, kLeastRoot = 0x1p-45f;
static float least_squares(float eps) { return eps < kLeastRoot ? kLeastSquares : 0.0f; }

// Where a row of the padded layout is, and whether it is a real token.
struct Place {
  int64_t seq;
  int t;
  bool real;
  int64_t packed;
};

// Both words of an int64 length, the one of an int32 twice: no branch that a
// load would wait at.
__device__ __forceinline__ int64_t length_of(const UnitRows& a, int64_t seq) {
  const int is64 = a.lengths64 ? 1 : 0;
  const int32_t* l = static_cast<const int32_t*>(a.lengths) + (seq << is64);
  const int32_t lo = l[0], hi = l[is64];
  return is64 ? (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo) : lo;
}

// The words as they are in memory: the numbers unpacked from them before are
// not kept for those after.
template <typename T, int K>
__device__ __forceinline__ void keep_packed(Chunk<T> (&c)[K]) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (uint32_t& w : c[k].w) asm("" : "+v"(w));
}

// For a row x with its dy and eps: all three times 2^-e, with e the exponent
// of the larger of eps and x's largest element.  That changes neither
// x / max(|x|, eps) nor dx, and the squares are then of numbers around 1.
// Numbers that are not finite stay as they are.
template <typename T, int G, int K, bool BACKWARD>
__device__ void rescale_row(Chunk<T> (&x)[K], Chunk<T> (&dy)[K], float& eps, bool far,
                            uint32_t* part) {
  constexpr int V = kVec<T>;
  uint32_t big = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float f[V];
    unpack<T>(x[k], f);
#pragma unroll
    for (int e = 0; e < V; ++e) big = max(big, __float_as_uint(f[e]) & 0x7fffffffu);
  }
  big = group_max<G>(big, part);
  keep_packed(x);
  if (!far || big >= 0x7f800000u) return;
  const int shift = 127 - (int)(max(big, __float_as_uint(eps)) >> 23);
  eps = __builtin_amdgcn_ldexpf(eps, shift);
  auto move = [&](Chunk<T>& c) {
    float f[V];
    unpack<T>(c, f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = __builtin_amdgcn_ldexpf(f[e], shift);
    c = pack<T>(f);
  };
#pragma unroll
  for (int k = 0; k < K; ++k) {
    move(x[k]);
    if constexpr (BACKWARD) move(dy[k]);
  }
}

// Workgroup b takes the rows from begin + b * GROUPS * U on, each group of lanes U of
// them, GROUPS apart: the lengths of all U are asked for together, then the
// rows themselves, so that a wave waits for two loads in a row however many
// rows it has (a loop over rows that looked one ahead waited for both in every
// turn: 38 + 72 us for the forward and backward of 512 x 1024 x 128 packed
// in bf16, against 29 + 51).
template <typename T, int G, int K, int U, bool BACKWARD>
__global__ __launch_bounds__(row_threads(G)) void unit_rows_kernel(UnitRows a) {
  using S = typename T::storage;
  constexpr int V = kVec<T>, GROUPS = row_threads(G) / G;
  constexpr int SUMS = BACKWARD ? 2 * U : U;
  __shared__ float part[G > 64 ? SUMS * G / 64 : 1];
  const int j = threadIdx.x % G, group = threadIdx.x / G;
  const int dim = a.dim;
  const S* x = static_cast<const S*>(a.x);
  const S* dy = static_cast<const S*>(a.dy);
  S* out = static_cast<S*>(a.out);

  // the workgroup's first row by one division, its others by what they are past it
  const int64_t row0 = a.begin + (int64_t)blockIdx.x * GROUPS * U;
  const uint32_t length = (uint32_t)a.length;
  const int64_t seq0 = row0 >> 32 ? row0 / length : (int64_t)((uint32_t)row0 / length);
  const uint32_t t0 = (uint32_t)(row0 - seq0 * length);
  Place at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t past = t0 + (uint32_t)(u * GROUPS + group);  // length < 2^31
    const uint32_t more = past < length ? 0 : past / length;
    at[u].seq = seq0 + more;
    at[u].t = (int)(past - more * length);
    at[u].real = row0 + u * GROUPS + group < a.rows;
    at[u].packed = 0;
  }
  if (a.lengths) {
    int64_t len[U];
    int32_t off[U];
    const int64_t last = a.sequences - 1;
    if (length >= (uint32_t)(GROUPS * U)) {
      // rows of two sequences at most: loads that are the workgroup's own
      const int64_t seq1 = min(seq0 + 1, last);
      const int64_t len0 = length_of(a, seq0), len1 = length_of(a, seq1);
      const int32_t off0 = a.offsets ? a.offsets[seq0] : 0, off1 = a.offsets ? a.offsets[seq1] : 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        len[u] = at[u].seq == seq0 ? len0 : len1;
        off[u] = at[u].seq == seq0 ? off0 : off1;
      }
    } else {
      // all loads before the first use
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t seq = min(at[u].seq, last);
        len[u] = length_of(a, seq);
        off[u] = a.offsets ? a.offsets[seq] : 0;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      at[u].real = at[u].real && at[u].t < len[u];
      if (a.offsets) {
        at[u].packed = (int64_t)off[u] + at[u].t;
        at[u].real = at[u].real && at[u].packed >= 0 && at[u].packed < a.packed_rows;
      }
    }
  }
  Chunk<T> raw[U][K], raw_d[BACKWARD ? U : 1][K];
  auto load = [&] {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const S* xr = x + at[u].seq * a.x_seq + at[u].t * a.x_row;
        raw[u][k] = at[u].real ? load_pieces<T>(xr, (j + k * G) * V, dim) : Chunk<T>{};
        if constexpr (BACKWARD) {
          const S* dr = a.offsets ? dy + at[u].packed * dim
                                  : dy + at[u].seq * a.dy_seq + at[u].t * a.dy_row;
          raw_d[u][k] = at[u].real ? load_pieces<T>(dr, (j + k * G) * V, dim) : Chunk<T>{};
        }
      }
  };
  float sums[SUMS];
  auto add_up = [&] {
#pragma unroll
    for (int i = 0; i < SUMS; ++i) sums[i] = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float f[V], d[V];
        unpack<T>(raw[u][k], f);
        if constexpr (BACKWARD) unpack<T>(raw_d[u][k], d);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          sums[u] += f[e] * f[e];
          if constexpr (BACKWARD) sums[U + u] += f[e] * d[e];
        }
      }
    group_sums<G>(sums, part);
  };
  bool far[U];  // the sums are not to be trusted
  // Writes the rows whose far is `which`.
  auto finish = [&](bool which, auto eps_of) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + u * GROUPS + group;
      const bool real = at[u].real;
      if (row >= a.rows || far[u] != which || (!BACKWARD && a.offsets && !real)) continue;
      const float norm = sqrtf(sums[u]), eps = eps_of(u);
      float scale = 1.0f / fmaxf(norm, eps), along = 0.0f;
      if constexpr (BACKWARD) {
        // y <y, dy> / |x| = x <x, dy> / |x|^3; a NaN norm stays NaN
        if (!(norm <= eps)) along = sums[U + u] * scale * scale;
      } else {
        if (norm != norm) scale = norm;
      }
      S* to = out + (!BACKWARD && a.offsets ? at[u].packed : row) * dim;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float f[V], d[V];
        unpack<T>(raw[u][k], f);
        if constexpr (BACKWARD) unpack<T>(raw_d[u][k], d);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if constexpr (BACKWARD) f[e] = d[e] - f[e] * along;
          f[e] = real ? f[e] * scale : 0.0f;
        }
        store_chunk<T>(to, (j + k * G) * V, dim, f);
      }
    }
  };
  load();
  add_up();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    bool near = sums[u] >= a.least && sums[u] < kMostSquares;
    if constexpr (BACKWARD) near = near && fabsf(sums[U + u]) < kMostSquares;
    far[u] = kWideRange<T> && at[u].real && !near;
  }
  finish(false, [&](int) { return a.eps; });
  if constexpr (kWideRange<T>) {
    // The far ones from their loads on again: nothing is held or waited for
    // above for their sake.  A wave's rows go through it together, and a
    // workgroup's where it has one row: the sums, and so the answer, are the
    // same in all its threads.
    bool any = false;
#pragma unroll
    for (int u = 0; u < U; ++u) any |= far[u];
    if (__ballot(any) == 0) return;
    load();
    float eps[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      eps[u] = a.eps;
      rescale_row<T, G, K, BACKWARD>(raw[u], raw_d[BACKWARD ? u : 0], eps[u], far[u],
                                     reinterpret_cast<uint32_t*>(part));
    }
    add_up();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      keep_packed(raw[u]);
      if constexpr (BACKWARD) keep_packed(raw_d[u]);
    }
    finish(true, [&](int u) { return eps[u]; });
  }
}

// offsets[s] = sum of the lengths before s, each clamped to [0, max_len];
// offsets[n] the total, which also goes to `total` (pinned host memory, if
// given) as 2 * total + 1.  One workgroup: a batch has a few thousand
// sequences.  A thread takes eight in a row, the waves are joined by their
// lanes' prefix sums and one barrier (n = 512: 3 us, most of it the launch and
// the load).
constexpr int kScanThreads = 1024, kScanWaves = kScanThreads / 64, kScanRun = 8;
template <typename L>
__global__ __launch_bounds__(kScanThreads) void length_offsets_kernel(
    const L* __restrict__ lengths, int64_t n, int32_t max_len, int32_t* __restrict__ clamped,
    int32_t* __restrict__ offsets, uint64_t* total) {
  __shared__ int32_t waves[2][kScanWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int32_t before = 0;  // sum of the passes before this one
  int turn = 0;
  for (int64_t base = 0; base < n; base += kScanThreads * kScanRun, turn ^= 1) {
    const int64_t i0 = base + threadIdx.x * kScanRun;
    int32_t len[kScanRun], mine = 0;
#pragma unroll
    for (int e = 0; e < kScanRun; ++e) {
      const L v = i0 + e < n ? lengths[i0 + e] : (L)0;
      len[e] = (int32_t)min(max(v, (L)0), (L)max_len);
      mine += len[e];
    }
    int32_t upto = mine;  // this thread's and those of the lanes before it
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int32_t v = __shfl_up(upto, off, 64);
      if (lane >= off) upto += v;
    }
    if (lane == 63) waves[turn][wave] = upto;
    __syncthreads();
    int32_t at = before + upto - mine;
#pragma unroll
    for (int w = 0; w < kScanWaves; ++w) {
      before += waves[turn][w];
      if (w < wave) at += waves[turn][w];
    }
#pragma unroll
    for (int e = 0; e < kScanRun; ++e)
      if (i0 + e < n) {
        clamped[i0 + e] = len[e];
        offsets[i0 + e] = at;
        at += len[e];
      }
  }
  if (threadIdx.x == 0) {
    offsets[n] = before;
    if (total)
      __hip_atomic_store(total, 2ull * (uint64_t)before + 1, __ATOMIC_RELEASE,
                         __HIP_MEMORY_SCOPE_SYSTEM);
  }
}

template <bool BACKWARD>
static int run_unit_rows(maxsim_dtype dtype, const UnitRows& a, void* stream) {
  int rc = MAXSIM_OK;
  auto launch = [&](auto t, auto s, auto rows) {
    using T = decltype(t);
    constexpr int G = decltype(s)::G, K = decltype(s)::K, U = decltype(rows)::value;
    constexpr int threads = row_threads(G), each = threads / G * U;
    constexpr int64_t most = UINT32_MAX / threads;  // a launch's threads fit 32 bits
    UnitRows part = a;
    for (; part.begin < a.rows && rc == MAXSIM_OK; part.begin += most * each) {
      const int64_t blocks = std::min<int64_t>((a.rows - part.begin + each - 1) / each, most);
      hipLaunchKernelGGL((unit_rows_kernel<T, G, K, U, BACKWARD>), dim3((unsigned)blocks),
                         dim3(threads), 0, static_cast<hipStream_t>(stream), part);
      rc = check_launch("unit_rows_kernel");
    }
  };
  // Rows per group: more where each waits for its sequence's length first
  // (32000 x 300 x 128 f16, forward: 673 us with four against 705 with two;
  // 1.2 M rows of 96 bf16 without lengths: 82 us with two against 95 with
  // four), one where a row is several chunks (1000 x 300 x 128 fp32: 25.7 us
  // against 26.8 with two).  The backward has two rows in flight for one.
  constexpr int both = BACKWARD ? 2 : 1;
  auto go = [&](auto t) {
    with_shape<kVec<decltype(t)>>(a.dim, [&](auto s) {
      if constexpr (decltype(s)::K > 1) launch(t, s, std::integral_constant<int, 1>{});
      else if (a.lengths) launch(t, s, std::integral_constant<int, 4 / both>{});
      else launch(t, s, std::integral_constant<int, 2 / both>{});
    });
  };
  if (dtype == MAXSIM_FLOAT32) go(F32{});
  else if (dtype == MAXSIM_FLOAT16) go(F16{});
  else go(BF16{});
  return rc;
}

static int check_unit_rows(maxsim_dtype dtype, int64_t sequences, int64_t length, int64_t dim,
                           const void* lengths, const int32_t* offsets, int64_t packed_rows,
                           float eps) {
  if (int e = check_dtype(dtype)) return e;
  if (int e = check_dim(dim)) return e;
  if (sequences < 0 || length < 0 || packed_rows < 0)
    return fail(MAXSIM_ERR_INVALID, "negative size");
  if (length > INT32_MAX) return fail(MAXSIM_ERR_UNSUPPORTED, "length exceeds 2^31 - 1");
  // 1 / eps has to be a number too
  if (!(eps >= FLT_MIN)) return fail(MAXSIM_ERR_INVALID, "eps must be at least 2^-126");
  if (sequences > 0 && offsets && !lengths)
    return fail(MAXSIM_ERR_INVALID, "offsets without lengths");
  return MAXSIM_OK;
}

}  // namespace maxsim

using namespace maxsim;

extern "C" {

int maxsim_amd_unit_rows_forward(maxsim_dtype dtype, const void* x, int64_t sequences,
                                 int64_t length, int64_t dim, int64_t x_seq_stride,
                                 int64_t x_row_stride, const void* lengths, int lengths64,
                                 const int32_t* offsets, int64_t packed_rows, float eps, void* y,
                                 void* stream) {
  clear_error();
  if (int e = check_unit_rows(dtype, sequences, length, dim, lengths, offsets, packed_rows, eps))
    return e;
  if (x_seq_stride < 0 || x_row_stride < 0) return fail(MAXSIM_ERR_INVALID, "negative stride");
  if (sequences == 0 || length == 0 || (offsets && packed_rows == 0)) return MAXSIM_OK;
  if (!x || !y) return fail(MAXSIM_ERR_INVALID, "null pointer argument");
  const UnitRows a{x,           nullptr, x_seq_stride, x_row_stride, 0,           0,
                   sequences, sequences * length, 0, (int)length, (int)dim, lengths,
                   lengths64, offsets, packed_rows, eps, least_squares(eps), y};
  return run_unit_rows<false>(dtype, a, stream);
}

int maxsim_amd_unit_rows_backward(maxsim_dtype dtype, const void* dy, int64_t dy_seq_stride,
                                  int64_t dy_row_stride, const void* x, int64_t sequences,
                                  int64_t length, int64_t dim, int64_t x_seq_stride,
                                  int64_t x_row_stride, const void* lengths, int lengths64,
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
                   sequences, sequences * length, 0, (int)length, (int)dim, lengths,
                   lengths64, offsets, packed_rows, eps, least_squares(eps), dx};
  return run_unit_rows<true>(dtype, a, stream);
}

int maxsim_amd_length_offsets(const void* lengths, int lengths64, int64_t sequences,
                              int64_t max_len, int32_t* clamped, int32_t* offsets,
                              uint64_t* total, void* stream) {
  clear_error();
  if (sequences < 0 || max_len < 0) return fail(MAXSIM_ERR_INVALID, "negative size");
  if (max_len > 0 && sequences > INT32_MAX / max_len)
    return fail(MAXSIM_ERR_UNSUPPORTED, "more than 2^31 - 1 padded rows: offsets are int32");
  if (!offsets || (sequences > 0 && (!lengths || !clamped)))
    return fail(MAXSIM_ERR_INVALID, "null pointer argument");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int32_t most = (int32_t)std::min<int64_t>(max_len, INT32_MAX);
  if (lengths64)
    hipLaunchKernelGGL(length_offsets_kernel<int64_t>, dim3(1), dim3(kScanThreads), 0, st,
                       static_cast<const int64_t*>(lengths), sequences, most, clamped, offsets,
                       total);
  else
    hipLaunchKernelGGL(length_offsets_kernel<int32_t>, dim3(1), dim3(kScanThreads), 0, st,
                       static_cast<const int32_t*>(lengths), sequences, most, clamped, offsets,
                       total);
  return check_launch("length_offsets_kernel");
}

}  // extern "C"
