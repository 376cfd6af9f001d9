// Token ids looked up in an embedding table, and the table's gradient.
//
//   y[t] = scale * weight[id_t]          dweight[v] = scale * sum over id_t = v of dy[t]
//
// Memory-bound, both ways: two operations per element at most.
//
// The gradient adds up rows that lie anywhere in dy, many of them for a
// frequent token and none for most others of a large table.  Floating-point
// atomics would do that in an order of their own every time, and one by one
// for a frequent token; here the tokens are sorted by row first, stably, so
// that every order is decided by the ids alone:
//   embed_sort_kernel  a workgroup for each value of the row's low bits (rows
//                      of one frequency lie side by side in a vocabulary, and
//                      part ways in their low bits) reads all ids, keeps its
//                      own in order and sorts them by the high bits; it also
//                      writes the zeros of its rows that no token has;
//   embed_sum_kernel   groups of lanes add up `window` sorted tokens each, a
//                      run of one row in registers, and write the finished rows;
//                      a run of up to kShortRun tokens that crosses into the
//                      next window is finished by the group it began with, of
//                      a longer one each group leaves its part in the workspace;
//   embed_join_kernel  adds those parts.
#include <algorithm>

#include "maxsim_host.h"
#include "maxsim_rows.h"
#include "../../include/maxsim_amd_encoder.h"

namespace maxsim {

// ---- forward -----------------------------------------------------------------

struct EmbedArgs {
  const void* weight;
  int64_t w_row;  // stride in elements
  int64_t vocab;
  int dim;
  const void* ids;
  int ids64;
  int64_t sequences, tokens;  // tokens: sequences * length
  int64_t begin;              // first token of this launch
  uint32_t length;
  const void* lengths;  // int32, or int64; NULL: every token is real
  int lengths64;
  int64_t padding;  // its row gets no gradient; -1: none
  float scale;
  void* y;
  int32_t* rows;  // NULL: not wanted
};

// Value i of an array of int32 or int64: both words of one, the other's twice.
__device__ __forceinline__ int64_t load_index(const void* p, int is64, int64_t i) {
  is64 = is64 ? 1 : 0;
  const int32_t* l = static_cast<const int32_t*>(p) + (i << is64);
  const int32_t lo = l[0], hi = l[is64];
  return is64 ? (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo) : lo;
}

// N elements of a row of type W from e0 on, those past dim as zero.
template <typename W, int N> struct Piece { Chunk<W> c[N / kVec<W>]; };
template <typename W, int N>
__device__ __forceinline__ Piece<W, N> load_piece(const typename W::storage* row, int e0, int dim) {
  Piece<W, N> p;
#pragma unroll
  for (int c = 0; c < N / kVec<W>; ++c) p.c[c] = load_pieces<W>(row, e0 + c * kVec<W>, dim);
  return p;
}
template <typename W, int N>
__device__ __forceinline__ void unpack_piece(const Piece<W, N>& p, float (&f)[N]) {
  constexpr int v = kVec<W>;
#pragma unroll
  for (int c = 0; c < N / v; ++c) {
    float part[v];
    unpack<W>(p.c[c], part);
#pragma unroll
    for (int e = 0; e < v; ++e) f[c * v + e] = part[e];
  }
}
template <typename W, int N>
__device__ __forceinline__ void store_piece(typename W::storage* row, int e0, int dim,
                                            const float (&f)[N]) {
  constexpr int v = kVec<W>;
#pragma unroll
  for (int c = 0; c < N / v; ++c) {
    float part[v];
#pragma unroll
    for (int e = 0; e < v; ++e) part[e] = f[c * v + e];
    store_chunk<W>(row, e0 + c * v, dim, part);
  }
}

// A group of G lanes looks up U tokens, GROUPS apart: their ids (and lengths)
// are asked for together, then their rows.
template <typename W, typename T, int G, int K, int U>
__global__ __launch_bounds__(row_threads(G)) void embed_kernel(EmbedArgs a) {
  constexpr int V = kVec<T>, GROUPS = row_threads(G) / G;
  const int j = threadIdx.x % G, group = threadIdx.x / G;
  const int dim = a.dim;
  const int64_t token0 = a.begin + (int64_t)blockIdx.x * GROUPS * U + group;
  bool real[U], known[U];
  int64_t id[U];
#pragma unroll
  for (int u = 0; u < U; ++u) real[u] = token0 + u * GROUPS < a.tokens;
  if (a.lengths) {
    // the first token's sequence by one division, the others' by what they are past it
    const int64_t seq0 = token0 >> 32 ? token0 / a.length
                                      : (int64_t)((uint32_t)token0 / a.length);
    const uint32_t t0 = (uint32_t)(token0 - seq0 * a.length);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t past = t0 + (uint32_t)(u * GROUPS);  // length < 2^31
      const uint32_t more = past < a.length ? 0 : past / a.length;
      const int64_t seq = min(seq0 + more, a.sequences - 1);
      const int64_t len = load_index(a.lengths, a.lengths64, seq);
      real[u] = real[u] && (int64_t)(past - more * a.length) < len;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    id[u] = real[u] ? load_index(a.ids, a.ids64, token0 + u * GROUPS) : -1;
  Piece<W, V> raw[U][K];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    known[u] = id[u] >= 0 && id[u] < a.vocab;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const auto* row = static_cast<const typename W::storage*>(a.weight) + id[u] * a.w_row;
      raw[u][k] = known[u] ? load_piece<W, V>(row, (j + k * G) * V, dim) : Piece<W, V>{};
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t token = token0 + u * GROUPS;
    if (token >= a.tokens) continue;
    if (a.rows && j == 0) a.rows[token] = known[u] && id[u] != a.padding ? (int32_t)id[u] : -1;
    auto* to = static_cast<typename T::storage*>(a.y) + token * dim;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float f[V];
      unpack_piece<W, V>(raw[u][k], f);
#pragma unroll
      for (int e = 0; e < V; ++e)
        f[e] = known[u] ? f[e] * a.scale : real[u] ? __builtin_nanf("") : 0.0f;
      store_chunk<T>(to, (j + k * G) * V, dim, f);
    }
  }
}

// ---- backward: the sort ------------------------------------------------------

// A token of dy and its row of the table.
struct Entry { uint32_t row, token; };

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kBucketBits = 8;   // low bits of a row: at most a workgroup per CU
constexpr int kDigitBits = 9;    // high bits of a row that one pass sorts by
constexpr int kListSize = 192;   // a wave's entries that LDS holds
constexpr int kKeysInFlight = 4; // loads of four ids per lane

struct SortArgs {
  const int32_t* rows;
  uint32_t tokens, vocab;
  int bucket_bits, high_bits, passes;
  Entry *sorted, *other;  // [tokens]
  uint32_t* total;        // entries in all
  void* dweight;
  int64_t row_bytes;
  int element;  // bytes of one
};

// Lanes before this one that are set in `mask`.
__device__ __forceinline__ uint32_t set_before(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// One stable pass: entries [from, to) of a wave, in the waves' order, to
// out[...] by bits [shift, shift + bits) of their rows.
template <typename Source>
__device__ __forceinline__ void sort_pass(Source in, uint32_t from, uint32_t to, int shift,
                                          int bits, uint32_t (&counts)[kSortWaves][1 << kDigitBits],
                                          uint32_t (&part)[kSortWaves], Entry* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t digits = 1u << bits, mask = digits - 1;
  for (uint32_t i = threadIdx.x; i < kSortWaves * digits; i += kSortThreads)
    counts[i >> bits][i & mask] = 0;
  __syncthreads();
  for (uint32_t i = from + lane; i < to; i += 64)
    atomicAdd(&counts[wave][(in(i).row >> shift) & mask], 1u);
  __syncthreads();
  // where each wave's entries of a digit start: thread d has digit d
  static_assert((1 << kDigitBits) <= kSortThreads, "a digit per thread");
  uint32_t mine = 0;
  if (threadIdx.x < digits)
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = counts[w][threadIdx.x];
      counts[w][threadIdx.x] = mine;
      mine += c;
    }
  uint32_t upto = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t v = __shfl_up(upto, off, 64);
    if (lane >= off) upto += v;
  }
  if (lane == 63) part[wave] = upto;
  __syncthreads();
  uint32_t base = upto - mine;
  for (int w = 0; w < wave; ++w) base += part[w];
  if (threadIdx.x < digits)
    for (int w = 0; w < kSortWaves; ++w) counts[w][threadIdx.x] += base;
  __syncthreads();
  for (uint32_t i0 = from; i0 < to; i0 += 64) {
    const uint32_t i = i0 + lane;
    const bool has = i < to;
    const Entry e = has ? in(i) : Entry{};
    const uint32_t d = (e.row >> shift) & mask;
    uint64_t same = __ballot(has);
    for (int b = 0; b < bits; ++b) {
      const uint64_t ones = __ballot((d >> b) & 1);
      same &= (d >> b) & 1 ? ones : ~ones;
    }
    if (has) {
      volatile uint32_t* at = &counts[wave][d];
      const uint32_t start = *at, rank = set_before(same);
      out[start + rank] = e;
      if (rank == 0) *at = start + (uint32_t)__popcll(same);
    }
  }
  __syncthreads();
}

__device__ __forceinline__ void zero_row(char* row, int64_t bytes, int element) {
  const int lane = threadIdx.x & 63;
  int64_t i = lane * 16;
  for (; i + 16 <= bytes; i += 64 * 16) store_any(row + i, make_uint4(0, 0, 0, 0));
  for (; i < bytes; i += element) {  // the lane that met the row's end
    if (element == 4) store_any(row + i, 0u);
    else store_any(row + i, (uint16_t)0);
  }
}

__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(SortArgs a) {
  __shared__ Entry list[kSortWaves][kListSize];
  __shared__ uint32_t counts[kSortWaves][1 << kDigitBits];
  __shared__ uint32_t part[kSortWaves], found[kSortWaves], less[kSortWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t bucket = blockIdx.x, low = (1u << a.bucket_bits) - 1;

  // the wave's share of the ids, a multiple of what its lanes take at a time
  constexpr uint32_t kTurn = 64 * 4 * kKeysInFlight;
  const uint32_t share = ((a.tokens + kSortWaves - 1) / kSortWaves + kTurn - 1) / kTurn * kTurn;
  const uint64_t begin = (uint64_t)wave * share;
  const uint64_t end = min(begin + share, (uint64_t)a.tokens);

  // Calls keep(entry, number among the wave's own) for the bucket's ids in
  // order; returns their number and adds to `fewer` those of lower buckets.
  auto scan = [&](uint32_t& fewer, auto keep) {
    uint32_t mine = 0;
    for (uint64_t i0 = begin; i0 < end; i0 += kTurn) {
      uint32_t key[kKeysInFlight][4];
#pragma unroll
      for (int u = 0; u < kKeysInFlight; ++u) {
        const uint64_t i = i0 + u * 256 + lane * 4;
        if (i + 4 <= a.tokens) {
          const uint4 q = load_any<uint4>(a.rows + i);
          key[u][0] = q.x, key[u][1] = q.y, key[u][2] = q.z, key[u][3] = q.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) key[u][e] = i + e < a.tokens ? (uint32_t)a.rows[i + e] : ~0u;
        }
      }
#pragma unroll
      for (int u = 0; u < kKeysInFlight; ++u) {
        uint64_t own[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t d = key[u][e] & low;
          const uint64_t valid = __ballot(key[u][e] < a.vocab);
          own[e] = __ballot(d == bucket) & valid;
          fewer += (uint32_t)__popcll(__ballot(d < bucket) & valid);
        }
        if ((own[0] | own[1] | own[2] | own[3]) == 0) continue;
        uint32_t at = mine;
#pragma unroll
        for (int e = 0; e < 4; ++e) at += set_before(own[e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (own[e] >> lane & 1)
            keep(Entry{key[u][e], (uint32_t)(i0 + u * 256 + lane * 4 + e)}, at++);
          mine += (uint32_t)__popcll(own[e]);
        }
      }
    }
    return mine;
  };
  uint32_t fewer = 0;
  const uint32_t own = scan(fewer, [&](Entry e, uint32_t at) {
    if (at < kListSize) list[wave][at] = e;
  });
  if (lane == 0) found[wave] = own, less[wave] = fewer;
  __syncthreads();
  uint32_t start = 0, count = 0, before = 0, most = 0;
  for (int w = 0; w < kSortWaves; ++w) {
    start += less[w];
    before += w < wave ? found[w] : 0;
    count += found[w];
    most = max(most, found[w]);
  }
  if (bucket == low && threadIdx.x == 0) *a.total = start + count;

  // The passes end in `sorted`; the first reads LDS, or the buffer that it
  // does not write where a wave's own are more than LDS holds.
  const bool in_lds = most <= kListSize;
  Entry* to = (a.passes & 1 ? a.sorted : a.other) + start;
  Entry* from = (a.passes & 1 ? a.other : a.sorted) + start;
  if (!in_lds) {
    uint32_t unused = 0;
    scan(unused, [&](Entry e, uint32_t at) { from[before + at] = e; });
    __syncthreads();
  }
  const uint32_t each = (count + kSortWaves - 1) / kSortWaves;
  const uint32_t lo = min((uint32_t)wave * each, count), hi = min(lo + each, count);
  for (int p = 0; p < a.passes; ++p) {
    const int shift = a.bucket_bits + p * kDigitBits;
    const int bits = min(a.high_bits - p * kDigitBits, kDigitBits);
    if (p == 0 && in_lds)
      sort_pass([&](uint32_t i) { return list[wave][i]; }, 0, own, shift, bits, counts, part, to);
    else
      sort_pass([&](uint32_t i) { return from[i]; }, lo, hi, shift, bits, counts, part, to);
    Entry* const t = to;
    to = from, from = t;
  }

  // Zeros for the rows without a token, by a bit for each of the bucket's rows.
  constexpr uint32_t kBits = kSortWaves * (1 << kDigitBits) * 32;
  uint32_t* has = &counts[0][0];
  const uint64_t rows = (uint64_t)1 << a.high_bits;  // that the bucket may have
  for (uint64_t r0 = 0; r0 < rows; r0 += kBits) {
    const uint32_t n = (uint32_t)min(rows - r0, (uint64_t)kBits);
    for (uint32_t i = threadIdx.x; i < (n + 31) / 32; i += kSortThreads) has[i] = 0;
    __syncthreads();
    auto mark = [&](uint32_t row) {
      const uint64_t r = (row >> a.bucket_bits) - r0;
      if (r < n) atomicOr(&has[r / 32], 1u << (r & 31));
    };
    if (in_lds)
      for (uint32_t i = lane; i < own; i += 64) mark(list[wave][i].row);
    else
      for (uint32_t i = lo + lane; i < hi; i += 64) mark(from[i].row);
    __syncthreads();
    for (uint32_t r = wave; r < n; r += kSortWaves) {
      const uint64_t v = ((r0 + r) << a.bucket_bits) + bucket;
      if (v >= a.vocab) break;
      if (!(has[r / 32] >> (r & 31) & 1))
        zero_row(static_cast<char*>(a.dweight) + v * a.row_bytes, a.row_bytes, a.element);
    }
    __syncthreads();
  }
}

// ---- backward: the sums ------------------------------------------------------

constexpr int kShortRun = 64;

struct SumArgs {
  const void* dy;
  int64_t dy_row;  // stride in elements
  int dim;
  const Entry* sorted;
  const uint32_t* total;
  uint32_t window;
  float scale;
  void* dweight;
  float* parts;     // [windows][2][part_dim]: of a run from before, of one that goes on
  int part_dim;
  uint32_t* begins;  // [windows] whether a long run begins here and goes on
};

template <typename T, typename W, int G, int K, int U>
__global__ __launch_bounds__(row_threads(G)) void embed_sum_kernel(SumArgs a) {
  using S = typename T::storage;
  constexpr int V = kVec<T>, GROUPS = row_threads(G) / G;
  constexpr bool SHORT = takes_short(G);
  constexpr int L = G < 64 ? G : 64;  // lanes that look at entries together
  const int j = threadIdx.x % G, group = threadIdx.x / G;
  const int dim = a.dim;
  const uint32_t total = *a.total;
  const uint32_t window = blockIdx.x * GROUPS + group;
  const uint64_t begin = (uint64_t)window * a.window;
  if (begin >= total) return;
  const uint32_t i0 = (uint32_t)begin, i1 = (uint32_t)min(begin + a.window, (uint64_t)total);
  const Entry* __restrict__ sorted = a.sorted;

  // Entries of `row` among the kShortRun from `at` on, or before it.
  auto count = [&](uint32_t row, int64_t at, int step) {
    uint32_t n = 0;
    const int shift = (threadIdx.x & 63) / L * L;
#pragma unroll
    for (int t = 0; t < kShortRun; t += L) {
      const int64_t i = at + (int64_t)step * (t + (int)(threadIdx.x % L));
      const bool same = i >= 0 && i < total && sorted[i].row == row;
      const uint64_t all = __ballot(same) >> shift;
      n += (uint32_t)__popcll(L == 64 ? all : all & (((uint64_t)1 << L) - 1));
    }
    return n;
  };
  auto is_long = [&](uint32_t row, uint32_t first) {
    const uint64_t i = (uint64_t)first + kShortRun;
    return i < total && sorted[i].row == row;
  };
  uint32_t at = i0, stop = i1;
  bool joins = false, goes_on = false;  // the first run is a long one's next part; so is the last's
  if (i0 > 0) {
    const uint32_t row = sorted[i0].row, back = count(row, (int64_t)i0 - 1, -1);
    if (back == kShortRun || (back > 0 && is_long(row, i0 - back))) joins = true;
    else if (back > 0) at = i0 + count(row, i0, 1);  // whose group has it
  }
  if (at < i1 && i1 < total) {
    const uint32_t row = sorted[i1 - 1].row;
    if (sorted[i1].row == row) {
      const uint32_t back = count(row, (int64_t)i1 - 1, -1);
      if (back == kShortRun || is_long(row, i1 - back)) goes_on = true;
      else stop = i1 + count(row, i1, 1);
    }
  }

  float acc[K][V];
  auto clear = [&] {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[k][e] = 0.0f;
  };
  auto write_row = [&](uint32_t row) {
    auto* to = static_cast<typename W::storage*>(a.dweight) + (int64_t)row * dim;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int e = 0; e < V; ++e) acc[k][e] *= a.scale;
      store_piece<W, V>(to, (j + k * G) * V, dim, acc[k]);
    }
  };
  auto write_part = [&](int which) {
    float* to = a.parts + ((int64_t)window * 2 + which) * a.part_dim;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int e0 = (j + k * G) * V;
#pragma unroll
      for (int e = 0; e < V; e += 4)
        if (e0 + e < a.part_dim)
          store_any(to + e0 + e, make_float4(acc[k][e], acc[k][e + 1], acc[k][e + 2], acc[k][e + 3]));
    }
  };
  clear();
  uint32_t row = at < stop ? sorted[at].row : 0;
  bool part = joins;
  Entry next[U];
#pragma unroll
  for (int u = 0; u < U; ++u) next[u] = sorted[min(at + u, stop - 1)];
  for (uint32_t i = at; i < stop; i += U) {
    Chunk<T> raw[U][K];
    Entry now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      now[u] = next[u];
      const S* from = static_cast<const S*>(a.dy) + (int64_t)now[u].token * a.dy_row;
#pragma unroll
      for (int k = 0; k < K; ++k) raw[u][k] = load_chunk<T, SHORT>(from, (j + k * G) * V, dim);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = sorted[min(i + U + u, stop - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= stop) break;
      if (now[u].row != row) {
        if (part) write_part(0);
        else write_row(row);
        part = false;
        row = now[u].row;
        clear();
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float f[V];
        place_chunk<T, SHORT>(raw[u][k], (j + k * G) * V, dim);
        unpack<T>(raw[u][k], f);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[k][e] += f[e];
      }
    }
  }
  if (at < stop) {
    if (part) write_part(0);
    else if (goes_on) write_part(1);
    else write_row(row);
  }
  if (j == 0) a.begins[window] = goes_on && !part;
}

constexpr int kPartThreads = 256, kPartUnroll = 8;

// A workgroup for each window: adds up the parts of the long run that begins
// in it and goes on, if there is one.
template <typename W>
__global__ __launch_bounds__(kPartThreads) void embed_join_kernel(SumArgs a) {
  const uint32_t total = *a.total, window = blockIdx.x;
  const uint64_t begin = (uint64_t)window * a.window;
  if (begin >= total || !a.begins[window]) return;
  const uint32_t row = a.sorted[begin + a.window - 1].row;
  // the windows after it that the run reaches into
  uint32_t more = 0;
  for (;;) {
    const uint64_t i = begin + (uint64_t)(more + 1 + (threadIdx.x & 63)) * a.window;
    const uint64_t same = __ballot(i < total && a.sorted[min(i, (uint64_t)total - 1)].row == row);
    more += (uint32_t)__popcll(same);
    if (~same) break;
  }
  auto* out = static_cast<typename W::storage*>(a.dweight) + (int64_t)row * a.dim;
  for (int e0 = threadIdx.x * 4; e0 < a.dim; e0 += kPartThreads * 4) {
    const float* p = a.parts + (int64_t)window * 2 * a.part_dim + e0;
    float4 s = load_any<float4>(p + a.part_dim);
    for (uint32_t w = 1; w <= more; w += kPartUnroll) {
      float4 v[kPartUnroll];
#pragma unroll
      for (int u = 0; u < kPartUnroll; ++u)
        v[u] = load_any<float4>(p + (int64_t)min(w + u, more) * 2 * a.part_dim);
#pragma unroll
      for (int u = 0; u < kPartUnroll; ++u)
        if (w + u <= more) s.x += v[u].x, s.y += v[u].y, s.z += v[u].z, s.w += v[u].w;
    }
    const float f[4] = {s.x * a.scale, s.y * a.scale, s.z * a.scale, s.w * a.scale};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e0 + e < a.dim) out[e0 + e] = from_float<W>(f[e]);
  }
}

// ---- sizes -------------------------------------------------------------------

static int bits_of(uint64_t n) {  // that numbers below n have
  int b = 0;
  while (((uint64_t)1 << b) < n) ++b;
  return b;
}

// Tokens of a window: enough windows to fill the chip, long enough that few
// runs cross into the next, and no more than 2^20 of them (a launch's threads
// fit 32 bits).
static uint32_t window_of(int64_t tokens) {
  const int64_t most = std::max<int64_t>(128, (tokens >> 20) + 1);
  return (uint32_t)std::min<int64_t>(std::max<int64_t>(tokens / 2048, 8), most);
}

struct EmbedLayout {
  int64_t windows;
  int part_dim;
  size_t sorted, other, begins, parts, bytes;  // offsets, and all
};
static EmbedLayout embed_layout(int64_t tokens, int64_t dim) {
  EmbedLayout l;
  const int64_t window = window_of(tokens);
  l.windows = (tokens + window - 1) / window;
  l.part_dim = (int)((dim + 7) / 8 * 8);
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  l.sorted = 256;  // the total first
  l.other = l.sorted + up((size_t)tokens * sizeof(Entry));
  l.begins = l.other + up((size_t)tokens * sizeof(Entry));
  l.parts = l.begins + up((size_t)l.windows * sizeof(uint32_t));
  l.bytes = l.parts + (size_t)l.windows * 2 * l.part_dim * sizeof(float);
  return l;
}

static int check_embed(maxsim_dtype weight_dtype, maxsim_dtype dtype, int64_t vocab, int64_t dim) {
  if (int e = check_dtype(dtype)) return e;
  if (int e = check_dtype(weight_dtype)) return e;
  if (weight_dtype != dtype && weight_dtype != MAXSIM_FLOAT32)
    return fail(MAXSIM_ERR_INVALID, "weight_dtype must be dtype or float32");
  if (int e = check_dim(dim)) return e;
  if (vocab < 0) return fail(MAXSIM_ERR_INVALID, "negative size");
  if (vocab > INT32_MAX) return fail(MAXSIM_ERR_UNSUPPORTED, "more than 2^31 - 1 rows of the table");
  return MAXSIM_OK;
}

// Calls f(weight type, type).
template <typename F>
static int with_embed_types(maxsim_dtype weight_dtype, maxsim_dtype dtype, F&& f) {
  const bool wide = weight_dtype == MAXSIM_FLOAT32;
  if (dtype == MAXSIM_FLOAT32) return f(F32{}, F32{});
  if (dtype == MAXSIM_FLOAT16) return wide ? f(F32{}, F16{}) : f(F16{}, F16{});
  return wide ? f(F32{}, BF16{}) : f(BF16{}, BF16{});
}

}  // namespace maxsim

using namespace maxsim;

extern "C" {

int maxsim_amd_embed_forward(maxsim_dtype weight_dtype, maxsim_dtype dtype, const void* weight,
                             int64_t vocab, int64_t dim, int64_t weight_stride, const void* ids,
                             int ids64, int64_t sequences, int64_t length, const void* lengths,
                             int lengths64, float scale, int64_t padding_idx, void* y,
                             int32_t* rows, void* stream) {
  clear_error();
  if (int e = check_embed(weight_dtype, dtype, vocab, dim)) return e;
  if (sequences < 0 || length < 0) return fail(MAXSIM_ERR_INVALID, "negative size");
  if (weight_stride < 0) return fail(MAXSIM_ERR_INVALID, "negative stride");
  if (length > INT32_MAX) return fail(MAXSIM_ERR_UNSUPPORTED, "length exceeds 2^31 - 1");
  if (sequences == 0 || length == 0) return MAXSIM_OK;
  if (rows && sequences > INT32_MAX / length)
    return fail(MAXSIM_ERR_UNSUPPORTED, "a gradient of more than 2^31 - 1 tokens");
  if (!ids || !y || (vocab > 0 && !weight))
    return fail(MAXSIM_ERR_INVALID, "null pointer argument");
  const EmbedArgs all{weight, weight_stride, vocab, (int)dim, ids, ids64, sequences,
                      sequences * length, 0, (uint32_t)length, lengths, lengths64,
                      padding_idx < 0 ? -1 : padding_idx, scale, y, rows};
  return with_embed_types(weight_dtype, dtype, [&](auto w, auto t) {
    using W = decltype(w);
    using T = decltype(t);
    int rc = MAXSIM_OK;
    with_shape<kVec<T>>(dim, [&](auto s) {
      constexpr int G = decltype(s)::G, K = decltype(s)::K, U = K > 1 ? 1 : 2;
      constexpr int threads = row_threads(G), each = threads / G * U;
      constexpr int64_t most = UINT32_MAX / threads;  // a launch's threads fit 32 bits
      EmbedArgs a = all;
      for (; a.begin < a.tokens && rc == MAXSIM_OK; a.begin += most * each) {
        const int64_t blocks = std::min<int64_t>((a.tokens - a.begin + each - 1) / each, most);
        hipLaunchKernelGGL((embed_kernel<W, T, G, K, U>), dim3((unsigned)blocks), dim3(threads), 0,
                           static_cast<hipStream_t>(stream), a);
        rc = check_launch("embed_kernel");
      }
    });
    return rc;
  });
}

size_t maxsim_amd_embed_backward_workspace_size(maxsim_dtype dtype, int64_t tokens, int64_t vocab,
                                                int64_t dim) {
  if (check_embed(dtype, dtype, vocab, dim) != MAXSIM_OK || tokens < 0 || tokens > INT32_MAX)
    return 0;
  return embed_layout(tokens, dim).bytes;
}

int maxsim_amd_embed_backward(maxsim_dtype weight_dtype, maxsim_dtype dtype, const void* dy,
                              int64_t dy_stride, const int32_t* rows, int64_t tokens,
                              int64_t vocab, int64_t dim, float scale, void* dweight,
                              void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (int e = check_embed(weight_dtype, dtype, vocab, dim)) return e;
  if (tokens < 0) return fail(MAXSIM_ERR_INVALID, "negative size");
  if (dy_stride < 0) return fail(MAXSIM_ERR_INVALID, "negative stride");
  if (tokens > INT32_MAX)
    return fail(MAXSIM_ERR_UNSUPPORTED, "a gradient of more than 2^31 - 1 tokens");
  if (vocab == 0) return MAXSIM_OK;
  if (!dweight || (tokens > 0 && (!dy || !rows)))
    return fail(MAXSIM_ERR_INVALID, "null pointer argument");
  const EmbedLayout l = embed_layout(tokens, dim);
  if (!workspace || workspace_bytes < l.bytes)
    return fail(MAXSIM_ERR_INVALID, "workspace too small: %zu bytes, %zu needed", workspace_bytes,
                l.bytes);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  uint32_t* total = reinterpret_cast<uint32_t*>(ws);
  Entry* sorted = reinterpret_cast<Entry*>(ws + l.sorted);
  const int bits = bits_of((uint64_t)vocab), bucket_bits = std::min(bits, kBucketBits);
  const int high_bits = bits - bucket_bits;
  const int element = weight_dtype == MAXSIM_FLOAT32 ? 4 : 2;
  const SortArgs sort{rows, (uint32_t)tokens, (uint32_t)vocab, bucket_bits, high_bits,
                      std::max((high_bits + kDigitBits - 1) / kDigitBits, 1), sorted,
                      reinterpret_cast<Entry*>(ws + l.other), total, dweight, dim * element,
                      element};
  hipLaunchKernelGGL(embed_sort_kernel, dim3(1u << bucket_bits), dim3(kSortThreads), 0, st, sort);
  if (int e = check_launch("embed_sort_kernel")) return e;
  if (tokens == 0) return MAXSIM_OK;
  const SumArgs sum{dy, dy_stride, (int)dim, sorted, total, window_of(tokens), scale, dweight,
                    reinterpret_cast<float*>(ws + l.parts), l.part_dim,
                    reinterpret_cast<uint32_t*>(ws + l.begins)};
  return with_embed_types(weight_dtype, dtype, [&](auto w, auto t) {
    using W = decltype(w);
    using T = decltype(t);
    int rc = MAXSIM_OK;
    with_shape<kVec<T>>(dim, [&](auto s) {
      constexpr int G = decltype(s)::G, K = decltype(s)::K;
      constexpr int U = K >= 3 ? 4 : 8;
      constexpr int threads = row_threads(G), groups = threads / G;
      hipLaunchKernelGGL((embed_sum_kernel<T, W, G, K, U>),
                         dim3((unsigned)((l.windows + groups - 1) / groups)), dim3(threads), 0, st,
                         sum);
      rc = check_launch("embed_sum_kernel");
    });
    if (rc != MAXSIM_OK) return rc;
    hipLaunchKernelGGL(embed_join_kernel<W>, dim3((unsigned)l.windows), dim3(kPartThreads), 0, st,
                       sum);
    return check_launch("embed_join_kernel");
  });
}

}  // extern "C"
