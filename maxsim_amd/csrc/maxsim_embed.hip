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
// that the ids alone decide every order:
//   embed_few_kernel   few tokens: one launch does all of it in LDS;
//   embed_count_kernel, embed_place_kernel   a pass of the sort of many;
//   embed_sum_kernel   groups of lanes add up `window` sorted tokens each, a
//                      run of one row in registers, and write the finished rows;
//                      a run of up to short_run tokens that crosses into the
//                      next window is finished by the group it began with, of
//                      a longer one each group leaves its part in the workspace;
//                      more workgroups write the rows without a token;
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

// ---- backward: shared parts --------------------------------------------------

// A token of dy and its row of the table.
struct Entry { uint32_t row, token; };
constexpr uint32_t kNoRow = ~0u;

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;

// Lanes before this one that are set in `mask`.
__device__ __forceinline__ uint32_t set_before(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Lanes among `has` with this lane's d, a number of `bits` bits.
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int bits, uint64_t has) {
  for (int b = 0; b < bits; ++b) {
    const uint64_t ones = __ballot(d >> b & 1);
    has &= d >> b & 1 ? ones : ~ones;
  }
  return has;
}

// Sum over the lanes up to this one.
__device__ __forceinline__ uint32_t sum_upto(uint32_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t below = __shfl_up(v, off, 64);
    if (lane >= off) v += below;
  }
  return v;
}

// Sum over the threads before this one, of kSortThreads.
__device__ __forceinline__ uint32_t sum_before(uint32_t v, uint32_t (&waves)[kSortWaves]) {
  const int wave = threadIdx.x >> 6;
  const uint32_t upto = sum_upto(v);
  if ((threadIdx.x & 63) == 63) waves[wave] = upto;
  __syncthreads();
  uint32_t s = upto - v;
  for (int w = 0; w < wave; ++w) s += waves[w];
  return s;
}

// The rows of the table that some workgroups look after: those without a token
// become 0.
struct ZeroArgs {
  void* dweight;
  int64_t row_bytes;
  uint32_t vocab, rows;  // rows: of a workgroup, up to kZeroRows
  int element;           // bytes of one
};
constexpr int kZeroRows = 4096;
constexpr int64_t kZeroBytes = 65536;  // of a workgroup, where that is a row or more

__device__ __forceinline__ void zero_row(char* row, int64_t bytes, int element) {
  const int lane = threadIdx.x & 63;
  int64_t i = lane * 16;
  for (; i + 16 <= bytes; i += 64 * 16) store_any(row + i, make_uint4(0, 0, 0, 0));
  for (; i < bytes; i += element) {  // the lane that met the row's end
    if (element == 4) store_any(row + i, 0u);
    else store_any(row + i, (uint16_t)0);
  }
}

// Rows from `first` on whose bit is not set in `has`, a row per wave.
__device__ __forceinline__ void zero_rows(const ZeroArgs& a, uint32_t first, const uint32_t* has) {
  const uint32_t n = min(a.rows, a.vocab - first);
  for (uint32_t r = threadIdx.x >> 6; r < n; r += blockDim.x >> 6)
    if (!(has[r / 32] >> (r & 31) & 1))
      zero_row(static_cast<char*>(a.dweight) + ((int64_t)first + r) * a.row_bytes, a.row_bytes,
               a.element);
}

// ---- backward: few tokens, in one launch ---------------------------------------

// One workgroup for each value of a row's low bits reads all the ids, keeps its
// own in order, sorts them in LDS by the high bits and adds up their rows of
// dy; more workgroups write the rows without a token.  An entry is a number:
// the high bits above a token's kTokenBits, so that order of rows and then of
// tokens is the order of the numbers.
constexpr int kTokenBits = 12, kFewTokens = 1 << kTokenBits;
constexpr int kBucketBits = 8;   // low bits of a row: a workgroup per CU
constexpr int kFewVocabBits = 32 - kTokenBits + kBucketBits;
constexpr int kFewDigitBits = 8; // high bits that a pass sorts by
constexpr int kWaveIds = kFewTokens / kSortWaves;
static_assert(kWaveIds == 64 * 4, "four ids per lane");

struct FewArgs {
  const int32_t* rows;
  const void* dy;
  int64_t dy_row;  // stride in elements
  uint32_t tokens;
  int dim, bucket_bits, high_bits;
  uint32_t buckets;
  float scale;
  ZeroArgs zero;
};

// Four ids in a row; past the end there is no row.
__device__ __forceinline__ void load_rows(const int32_t* rows, uint32_t i, uint32_t n,
                                          uint32_t (&key)[4]) {
  if (i + 4 <= n) {
    const uint4 q = load_any<uint4>(rows + i);
    key[0] = q.x, key[1] = q.y, key[2] = q.z, key[3] = q.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) key[e] = i + e < n ? (uint32_t)rows[i + e] : kNoRow;
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(kSortThreads) void embed_few_kernel(FewArgs a) {
  using S = typename T::storage;
  constexpr int V = kVec<T>, U = 8;
  constexpr int kColumns = 64 * V;  // of a wave
  __shared__ union {
    struct {
      uint32_t list[kFewTokens], counts[kSortWaves][1 << kFewDigitBits];
    } sort;
    float parts[kSortWaves][kColumns];
    uint32_t has[kZeroRows / 32];
  } lds;
  __shared__ uint32_t sorted[kFewTokens];
  __shared__ uint32_t found[kSortWaves], waves[kSortWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t key[4];
  const uint32_t i0 = wave * kWaveIds + lane * 4;
  load_rows(a.rows, i0, a.tokens, key);

  if (blockIdx.x >= a.buckets) {
    const uint32_t first = (blockIdx.x - a.buckets) * a.zero.rows;
    if (threadIdx.x < kZeroRows / 32) lds.has[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t r = key[e] - first;
      if (key[e] < a.zero.vocab && r < a.zero.rows) atomicOr(&lds.has[r / 32], 1u << (r & 31));
    }
    __syncthreads();
    zero_rows(a.zero, first, lds.has);
    return;
  }

  // the wave's own, in order, to its part of the list
  const uint32_t bucket = blockIdx.x, low = (1u << a.bucket_bits) - 1;
  uint32_t* list = lds.sort.list + wave * kWaveIds;
  uint64_t own[4];
  uint32_t at = 0, mine = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    own[e] = __ballot(key[e] < a.zero.vocab && (key[e] & low) == bucket);
    at += set_before(own[e]);
    mine += (uint32_t)__popcll(own[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (own[e] >> lane & 1) list[at++] = key[e] >> a.bucket_bits << kTokenBits | (i0 + e);
  if (lane == 0) found[wave] = mine;
  __syncthreads();
  uint32_t m = 0;
  for (int w = 0; w < kSortWaves; ++w) m += found[w];
  if (m == 0) return;

  // stable passes by the high bits, from the waves' lists to `sorted`, back to
  // the list as a whole, and so on
  const int passes = max((a.high_bits + kFewDigitBits - 1) / kFewDigitBits, 1);
  const uint32_t each = (m + kSortWaves - 1) / kSortWaves;
  const uint32_t *from = list;
  uint32_t lo = 0, hi = mine, *to = sorted;
  for (int p = 0; p < passes; ++p) {
    const int shift = kTokenBits + p * kFewDigitBits;
    const int bits = min(a.high_bits - p * kFewDigitBits, kFewDigitBits);
    const uint32_t digits = 1u << bits;
    auto& counts = lds.sort.counts;
    for (uint32_t d = lane; d < digits; d += 64) counts[wave][d] = 0;
    for (uint32_t i = lo + lane; i < hi; i += 64)
      atomicAdd(&counts[wave][from[i] >> shift & (digits - 1)], 1u);
    __syncthreads();
    uint32_t all = 0;
    if (threadIdx.x < digits)
      for (int w = 0; w < kSortWaves; ++w) all += counts[w][threadIdx.x];
    uint32_t start = sum_before(all, waves);
    if (threadIdx.x < digits)
      for (int w = 0; w < kSortWaves; ++w) {
        const uint32_t c = counts[w][threadIdx.x];
        counts[w][threadIdx.x] = start;
        start += c;
      }
    __syncthreads();
    for (uint32_t j = lo; j < hi; j += 64) {
      const bool has = j + lane < hi;
      const uint32_t e = has ? from[j + lane] : 0, d = e >> shift & (digits - 1);
      const uint64_t same = same_digit(d, bits, __ballot(has));
      if (has) {
        volatile uint32_t* next = &counts[wave][d];
        const uint32_t first = *next, rank = set_before(same);
        to[first + rank] = e;
        if (rank == 0) *next = first + (uint32_t)__popcll(same);
      }
    }
    __syncthreads();
    from = to;
    to = from == sorted ? lds.sort.list : sorted;
    lo = min((uint32_t)wave * each, m), hi = min(lo + each, m);
  }
  if (from != sorted) {
    for (uint32_t i = threadIdx.x; i < m; i += kSortThreads) sorted[i] = from[i];
    __syncthreads();
  }

  // Sums: waves share the columns, kColumns each, and where there are more
  // waves than that, the sorted tokens.  A run that began in an earlier wave's
  // share is left in LDS for that wave.
  const int blocks = (a.dim + kColumns - 1) / kColumns;
  const int across = min(blocks, kSortWaves), shares = kSortWaves / across;
  const int share = wave / across;
  const uint32_t take = (m + shares - 1) / shares;
  const uint32_t begin = share < shares ? min(share * take, m) : m, end = min(begin + take, m);
  auto row_at = [&](uint32_t i) { return sorted[i] >> kTokenBits; };
  const bool joins = begin > 0 && begin < end && row_at(begin) == row_at(begin - 1);
  const bool goes_on = begin < end && end < m && row_at(end) == row_at(end - 1);
  for (int round = 0; round * across < blocks; ++round) {
    const int block = round * across + wave % across;
    const int e0 = block * kColumns + lane * V;
    const bool active = block < blocks && begin < end;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.0f;
    auto write_row = [&](uint32_t row) {
      auto* out = static_cast<typename W::storage*>(a.zero.dweight) +
                  (int64_t)(row << a.bucket_bits | bucket) * a.dim;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] *= a.scale;
      store_piece<W, V>(out, e0, a.dim, acc);
    };
    bool part = joins;
    uint32_t row = active ? row_at(begin) : 0;
    if (active) {
      for (uint32_t i = begin; i < end; i += U) {
        Chunk<T> raw[U];
        uint32_t entry[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          entry[u] = sorted[min(i + u, end - 1)];
          const S* dy = static_cast<const S*>(a.dy) + (entry[u] & (kFewTokens - 1)) * a.dy_row;
          raw[u] = load_pieces<T>(dy, e0, a.dim);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (i + u >= end) break;
          if (entry[u] >> kTokenBits != row) {
            if (part) {
#pragma unroll
              for (int e = 0; e < V; ++e) lds.parts[wave][lane * V + e] = acc[e];
            } else {
              write_row(row);
            }
            part = false;
            row = entry[u] >> kTokenBits;
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = 0.0f;
          }
          float f[V];
          unpack<T>(raw[u], f);
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += f[e];
        }
      }
      if (part) {
#pragma unroll
        for (int e = 0; e < V; ++e) lds.parts[wave][lane * V + e] = acc[e];
      } else if (!goes_on) {
        write_row(row);
      }
    }
    __syncthreads();
    if (active && goes_on && !part) {
      for (int s = share + 1; s < shares; ++s) {
        if (s * take >= m || row_at(s * take) != row) break;
#pragma unroll
        for (int e = 0; e < V; ++e)
          acc[e] += lds.parts[s * across + wave % across][lane * V + e];
      }
      write_row(row);
    }
    __syncthreads();
  }
}

// ---- backward: the sort of many ------------------------------------------------

// Stable passes by kDigitBits of the row each, from the lowest.  The workgroups
// of a pass each have a run of the entries; embed_count_kernel counts a run's
// digits, embed_place_kernel adds up what the others counted and moves its run.
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSortGroups = 128;  // most workgroups of a pass
static_assert(kSortThreads % kDigits == 0, "threads share the digits' sums evenly");

struct SortArgs {
  const int32_t* rows;  // first pass
  const Entry* in;      // later ones
  Entry* out;
  uint32_t tokens, vocab;
  uint32_t run;  // entries of a workgroup, a multiple of kSortThreads
  int shift, bits;
  uint32_t* counts;  // [workgroups][kDigits]
  uint32_t* total;   // entries in all, which the first pass writes
};

// Calls f(entry, whether there is one) for the entries of a wave's share of the
// run in order, 64 at a time, loads of several ahead.
template <bool FIRST, typename F>
__device__ __forceinline__ void for_share(const SortArgs& a, uint32_t n, F&& f) {
  constexpr int U = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t each = a.run / kSortWaves;
  const uint64_t begin = (uint64_t)blockIdx.x * a.run + wave * each;
  const uint64_t end = min(begin + each, (uint64_t)n);
  for (uint64_t i0 = begin; i0 < end; i0 += 64 * U) {
    Entry e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t i = min(i0 + u * 64 + lane, end - 1);
      if constexpr (FIRST) e[u] = Entry{(uint32_t)a.rows[i], (uint32_t)i};
      else e[u] = a.in[i];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * 64 < end)
        f(e[u], i0 + u * 64 + lane < end && (!FIRST || e[u].row < a.vocab));
  }
}

// The wave's counts of its share's digits, in `counts`.
template <bool FIRST>
__device__ __forceinline__ void count_share(const SortArgs& a, uint32_t n, uint32_t* counts) {
  const uint32_t digits = 1u << a.bits;
  for (uint32_t d = threadIdx.x & 63; d < digits; d += 64) counts[d] = 0;
  for_share<FIRST>(a, n, [&](Entry e, bool has) {
    if (has) atomicAdd(&counts[e.row >> a.shift & (digits - 1)], 1u);
  });
}

template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void embed_count_kernel(SortArgs a) {
  __shared__ uint32_t counts[kSortWaves][kDigits];
  count_share<FIRST>(a, FIRST ? a.tokens : *a.total, counts[threadIdx.x >> 6]);
  __syncthreads();
  if (threadIdx.x >> a.bits) return;
  uint32_t s = 0;
  for (int w = 0; w < kSortWaves; ++w) s += counts[w][threadIdx.x];
  a.counts[(size_t)blockIdx.x * kDigits + threadIdx.x] = s;
}

template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void embed_place_kernel(SortArgs a) {
  __shared__ uint32_t counts[kSortWaves][kDigits];
  __shared__ uint32_t sums[2][kSortThreads], waves[kSortWaves];
  const int wave = threadIdx.x >> 6;
  const uint32_t digits = 1u << a.bits, mask = digits - 1;
  const uint32_t n = FIRST ? a.tokens : *a.total;
  count_share<FIRST>(a, n, counts[wave]);
  // of a digit: all entries, and those of the runs before; several threads each
  {
    const uint32_t d = threadIdx.x & mask, part = threadIdx.x >> a.bits;
    const uint32_t parts = kSortThreads >> a.bits, groups = gridDim.x;
    uint32_t all = 0, before = 0;
    constexpr int U = 8;
    for (uint32_t g0 = part; g0 < groups; g0 += parts * U) {
      uint32_t c[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        c[u] = a.counts[(size_t)min(g0 + u * parts, groups - 1) * kDigits + d];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t g = g0 + u * parts;
        all += g < groups ? c[u] : 0;
        before += g < blockIdx.x ? c[u] : 0;
      }
    }
    sums[0][threadIdx.x] = all, sums[1][threadIdx.x] = before;
    __syncthreads();
    all = before = 0;
    if (threadIdx.x < digits)
      for (uint32_t i = threadIdx.x; i < kSortThreads; i += digits)
        all += sums[0][i], before += sums[1][i];
    uint32_t start = sum_before(all, waves);
    if (FIRST && blockIdx.x == 0 && threadIdx.x == kSortThreads - 1) *a.total = start + all;
    start += before;
    if (threadIdx.x < digits)
      for (int w = 0; w < kSortWaves; ++w) {
        const uint32_t c = counts[w][threadIdx.x];
        counts[w][threadIdx.x] = start;
        start += c;
      }
  }
  __syncthreads();
  for_share<FIRST>(a, n, [&](Entry e, bool has) {
    const uint32_t d = e.row >> a.shift & mask;
    const uint64_t same = same_digit(d, a.bits, __ballot(has));
    if (has) {
      volatile uint32_t* next = &counts[wave][d];
      const uint32_t first = *next, rank = set_before(same);
      a.out[first + rank] = e;
      if (rank == 0) *next = first + (uint32_t)__popcll(same);
    }
  });
}

// ---- backward: the sums of many ------------------------------------------------

constexpr int kHalo = 64;           // entries on either side of a workgroup's that it looks at
constexpr int kWindowEntries = 1024;  // most entries of a workgroup's windows

struct SumArgs {
  const void* dy;
  int64_t dy_row;  // stride in elements
  int dim;
  const Entry* sorted;
  uint32_t tokens;
  const uint32_t* total;
  uint32_t window, short_run, groups;  // groups: workgroups that add up
  float scale;
  float* parts;      // [windows][2][part_dim]: of a run from before, of one that goes on
  int part_dim;
  uint32_t* begins;  // [windows] whether a long run begins here and goes on
  ZeroArgs zero;
};

// The first of the sorted entries whose row is not below `row`, by the 64 lanes
// of a wave.
__device__ __forceinline__ uint32_t first_of(const Entry* sorted, uint32_t total, uint64_t row) {
  uint32_t lo = 0, n = total;  // it is in [lo, lo + n]
  while (n > 0) {
    const uint32_t step = (n + 63) / 64;
    const uint64_t i = (uint64_t)(threadIdx.x & 63) * step;
    const bool below = i < n && sorted[lo + min((uint32_t)i, n - 1)].row < row;
    const uint32_t k = (uint32_t)__popcll(__ballot(below));  // of the lanes' entries
    if (k == 0) break;
    lo += (k - 1) * step + 1;
    n = min(step - 1, n - (k - 1) * step - 1);
  }
  return lo;
}

template <typename T, typename W, int G, int K, int U>
__global__ __launch_bounds__(row_threads(G)) void embed_sum_kernel(SumArgs a) {
  using S = typename T::storage;
  constexpr int V = kVec<T>, THREADS = row_threads(G), GROUPS = THREADS / G;
  constexpr bool SHORT = takes_short(G);
  constexpr int L = G < 64 ? G : 64;  // lanes that look at entries together
  __shared__ union {
    Entry entries[kWindowEntries + 2 * (kHalo + 1)];
    struct { uint32_t bounds[2], has[kZeroRows / 32]; } zero;
  } lds;
  const uint32_t total = *a.total;
  if (blockIdx.x >= a.groups) {
    const uint32_t first = (blockIdx.x - a.groups) * a.zero.rows;
    if (threadIdx.x < kZeroRows / 32) lds.zero.has[threadIdx.x] = 0;
    if (threadIdx.x < 128) {
      const int which = threadIdx.x >> 6;
      const uint32_t i = first_of(a.sorted, total, (uint64_t)first + which * a.zero.rows);
      if ((threadIdx.x & 63) == 0) lds.zero.bounds[which] = i;
    }
    __syncthreads();
    const uint32_t end = lds.zero.bounds[1];
    for (uint32_t i = lds.zero.bounds[0] + threadIdx.x; i < end; i += THREADS) {
      const uint32_t r = a.sorted[i].row - first;
      atomicOr(&lds.zero.has[r / 32], 1u << (r & 31));
    }
    __syncthreads();
    zero_rows(a.zero, first, lds.zero.has);
    return;
  }

  const int j = threadIdx.x % G, group = threadIdx.x / G;
  const int dim = a.dim;
  // the windows' entries and those around them; kNoRow where there are none
  const int64_t base = (int64_t)blockIdx.x * GROUPS * a.window - (kHalo + 1);
  if (base + kHalo + 1 >= total) return;
  const int count_all = GROUPS * (int)a.window + 2 * (kHalo + 1);
  for (int t = threadIdx.x; t < count_all; t += THREADS) {
    const int64_t i = base + t;
    lds.entries[t] = i >= 0 && i < total ? a.sorted[i] : Entry{kNoRow, 0};
  }
  __syncthreads();
  // from here on entries are counted from the workgroup's first, minus the halo
  const Entry* entries = lds.entries;
  const uint32_t window = blockIdx.x * GROUPS + group;
  const int first = kHalo + 1 + group * (int)a.window, last_of_all = (int)min((int64_t)total - base, (int64_t)count_all);
  if (first >= last_of_all) return;
  const int i0 = first, i1 = min(first + (int)a.window, last_of_all);
  const int short_run = (int)a.short_run;

  // Entries of `row` among the short_run from `at` on, or before it.
  auto count = [&](uint32_t row, int at, int step) {
    int n = 0;
    const int shift = (threadIdx.x & 63) / L * L;
    for (int t = 0; t < short_run; t += L) {
      const int k = t + (int)(threadIdx.x % L);
      const bool same = k < short_run && entries[at + step * k].row == row;
      const uint64_t all = __ballot(same) >> shift;
      n += (int)__popcll(L == 64 ? all : all & (((uint64_t)1 << L) - 1));
    }
    return n;
  };
  int at = i0, stop = i1;
  bool joins = false, goes_on = false;  // the first run is a long one's next part; so is the last's
  if (const uint32_t row = entries[i0].row; entries[i0 - 1].row == row) {
    const int back = count(row, i0 - 1, -1);
    if (back == short_run || entries[i0 - back + short_run].row == row) joins = true;
    else at = i0 + count(row, i0, 1);  // whose group has it
  }
  if (const uint32_t row = entries[i1 - 1].row; at < i1 && i1 < last_of_all && entries[i1].row == row) {
    const int back = count(row, i1 - 1, -1);
    if (back == short_run || entries[i1 - back + short_run].row == row) goes_on = true;
    else stop = i1 + count(row, i1, 1);
  }

  float acc[K][V];
  auto clear = [&] {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[k][e] = 0.0f;
  };
  auto write_row = [&](uint32_t row) {
    auto* to = static_cast<typename W::storage*>(a.zero.dweight) + (int64_t)row * dim;
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
  uint32_t row = at < stop ? entries[at].row : 0;
  bool part = joins;
  for (int i = at; i < stop; i += U) {
    Chunk<T> raw[U][K];
    uint32_t rows[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Entry e = entries[min(i + u, stop - 1)];
      rows[u] = e.row;
      const S* from = static_cast<const S*>(a.dy) + (int64_t)e.token * a.dy_row;
#pragma unroll
      for (int k = 0; k < K; ++k) raw[u][k] = load_chunk<T, SHORT>(from, (j + k * G) * V, dim);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= stop) break;
      if (rows[u] != row) {
        if (part) write_part(0);
        else write_row(row);
        part = false;
        row = rows[u];
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

// Adds up the parts of the long runs that begin in a workgroup's share of the
// windows and go on.  Threads share a row's columns, four each, and where
// there are more threads than that, the parts.
constexpr int kJoinThreads = 512, kJoinUnroll = 8, kJoinWindows = 512;
template <typename W>
__global__ __launch_bounds__(kJoinThreads) void embed_join_kernel(SumArgs a, uint32_t share) {
  __shared__ uint32_t list[kJoinWindows], found;
  __shared__ float4 sums[kJoinThreads];
  const uint32_t total = *a.total;
  const uint32_t windows = (uint32_t)(((uint64_t)total + a.window - 1) / a.window);
  const uint64_t first = (uint64_t)blockIdx.x * share;
  if (first >= windows) return;
  // the runs' windows, in whatever order: none has to do with another
  if (threadIdx.x == 0) found = 0;
  __syncthreads();
  const uint64_t w = first + threadIdx.x;
  if (threadIdx.x < share && w < windows && a.begins[w]) list[atomicAdd(&found, 1u)] = (uint32_t)w;
  __syncthreads();
  const int columns = (a.dim + 3) / 4;
  const int across = min(columns, kJoinThreads), shares = kJoinThreads / across;
  const int column = threadIdx.x % across, mine = threadIdx.x / across;
  for (uint32_t r = 0; r < found; ++r) {
    const uint32_t window = list[r];
    const uint64_t begin = (uint64_t)window * a.window;
    const uint32_t row = a.sorted[begin + a.window - 1].row;
    // the windows after it that the run reaches into
    uint32_t more = 0;
    for (;;) {
      const uint64_t i = begin + (uint64_t)(more + 1 + (threadIdx.x & 63)) * a.window;
      const uint64_t same = __ballot(i < total && a.sorted[min(i, (uint64_t)total - 1)].row == row);
      more += (uint32_t)__popcll(same);
      if (~same) break;
    }
    const uint32_t take = (more + shares - 1) / shares;
    const uint32_t lo = min(mine * take, more), hi = mine < shares ? min(lo + take, more) : lo;
    auto* out = static_cast<typename W::storage*>(a.zero.dweight) + (int64_t)row * a.dim;
    for (int c0 = 0; c0 < columns; c0 += across) {
      const int e0 = (c0 + column) * 4;
      const bool has = e0 < a.dim;
      const float* p = a.parts + (int64_t)window * 2 * a.part_dim + e0;
      float4 s = make_float4(0, 0, 0, 0);
      if (has && mine == 0) s = load_any<float4>(p + a.part_dim);
      for (uint32_t k = lo; has && k < hi; k += kJoinUnroll) {
        float4 v[kJoinUnroll];
#pragma unroll
        for (int u = 0; u < kJoinUnroll; ++u)
          v[u] = load_any<float4>(p + (int64_t)min(k + u + 1, hi) * 2 * a.part_dim);
#pragma unroll
        for (int u = 0; u < kJoinUnroll; ++u)
          if (k + u < hi) s.x += v[u].x, s.y += v[u].y, s.z += v[u].z, s.w += v[u].w;
      }
      if (shares > 1) {
        sums[threadIdx.x] = s;
        __syncthreads();
        if (mine == 0)
          for (int i = 1; i < shares; ++i) {
            const float4 v = sums[i * across + column];
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
          }
        __syncthreads();
      }
      if (!has || mine != 0) continue;
      const float f[4] = {s.x * a.scale, s.y * a.scale, s.z * a.scale, s.w * a.scale};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e0 + e < a.dim) out[e0 + e] = from_float<W>(f[e]);
    }
  }
}

// ---- sizes -------------------------------------------------------------------

static int bits_of(uint64_t n) {  // that numbers below n have
  int b = 0;
  while (((uint64_t)1 << b) < n) ++b;
  return b;
}

static bool few_tokens(int64_t tokens, int64_t vocab) {
  return tokens <= kFewTokens && bits_of((uint64_t)vocab) <= kFewVocabBits;
}

// Groups of lanes that hold a row in a workgroup.
static int row_groups(maxsim_dtype dtype, int64_t dim) {
  int groups = 1;
  auto of = [&](auto s) { groups = row_threads(decltype(s)::G) / decltype(s)::G; };
  if (dtype == MAXSIM_FLOAT32) with_shape<kVec<F32>>(dim, of);
  else with_shape<kVec<F16>>(dim, of);
  return groups;
}

struct EmbedLayout {
  int64_t windows;
  uint32_t window;  // tokens of one
  int groups;       // windows of a workgroup
  uint32_t run;     // tokens of a workgroup of the sort
  int part_dim;
  size_t sorted, other, counts, begins, parts, bytes;  // offsets, and all
};
static EmbedLayout embed_layout(maxsim_dtype dtype, int64_t tokens, int64_t vocab, int64_t dim) {
  EmbedLayout l{};
  if (few_tokens(tokens, vocab)) return l;
  l.groups = row_groups(dtype, dim);
  // enough windows to fill the chip, long enough that few runs cross into the next
  const int64_t most = std::min(kWindowEntries / l.groups, 128);
  l.window = (uint32_t)std::min<int64_t>(std::max<int64_t>(tokens / 2048, 8), most);
  l.windows = (tokens + l.window - 1) / l.window;
  l.part_dim = (int)((dim + 7) / 8 * 8);
  const int64_t each = (tokens + kSortGroups - 1) / kSortGroups;
  l.run = (uint32_t)((each + kSortThreads - 1) / kSortThreads * kSortThreads);
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  l.sorted = 256;  // the total first
  l.other = l.sorted + up((size_t)tokens * sizeof(Entry));
  l.counts = l.other + up((size_t)tokens * sizeof(Entry));
  l.begins = l.counts + (size_t)kSortGroups * kDigits * sizeof(uint32_t);
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
  return embed_layout(dtype, tokens, vocab, dim).bytes;
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
  const EmbedLayout l = embed_layout(dtype, tokens, vocab, dim);
  if (l.bytes > 0 && (!workspace || workspace_bytes < l.bytes))
    return fail(MAXSIM_ERR_INVALID, "workspace too small: %zu bytes, %zu needed", workspace_bytes,
                l.bytes);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int element = weight_dtype == MAXSIM_FLOAT32 ? 4 : 2;
  const int bits = bits_of((uint64_t)vocab);
  ZeroArgs zero{dweight, dim * element, (uint32_t)vocab, 0, element};
  zero.rows = (uint32_t)std::min<int64_t>(std::max<int64_t>(kZeroBytes / zero.row_bytes, 1),
                                          kZeroRows);
  const int64_t zero_groups = (vocab + zero.rows - 1) / zero.rows;

  if (few_tokens(tokens, vocab)) {
    FewArgs few{rows, dy, dy_stride, (uint32_t)tokens, (int)dim, std::min(bits, kBucketBits), 0, 0,
                scale, zero};
    few.high_bits = bits - few.bucket_bits;
    few.buckets = tokens > 0 ? 1u << few.bucket_bits : 0;
    const int64_t blocks = few.buckets + zero_groups;
    if (blocks > UINT32_MAX / kSortThreads)
      return fail(MAXSIM_ERR_UNSUPPORTED, "table too large for one launch");
    return with_embed_types(weight_dtype, dtype, [&](auto w, auto t) {
      hipLaunchKernelGGL((embed_few_kernel<decltype(t), decltype(w)>), dim3((unsigned)blocks),
                         dim3(kSortThreads), 0, st, few);
      return check_launch("embed_few_kernel");
    });
  }

  const int64_t sum_groups = (l.windows + l.groups - 1) / l.groups;
  if (sum_groups + zero_groups > UINT32_MAX / 1024)
    return fail(MAXSIM_ERR_UNSUPPORTED, "table or gradient too large for one launch");
  char* ws = static_cast<char*>(workspace);
  uint32_t* total = reinterpret_cast<uint32_t*>(ws);
  Entry* sorted = reinterpret_cast<Entry*>(ws + l.sorted);
  Entry* other = reinterpret_cast<Entry*>(ws + l.other);
  const int passes = std::max((bits + kDigitBits - 1) / kDigitBits, 1);
  SortArgs sort{rows, nullptr, passes & 1 ? sorted : other, (uint32_t)tokens, (uint32_t)vocab, l.run,
                0, (bits + passes - 1) / passes, reinterpret_cast<uint32_t*>(ws + l.counts), total};
  const dim3 runs((unsigned)((tokens + l.run - 1) / l.run));
  for (int p = 0; p < passes; ++p) {
    if (p == 0) {
      hipLaunchKernelGGL(embed_count_kernel<true>, runs, dim3(kSortThreads), 0, st, sort);
      hipLaunchKernelGGL(embed_place_kernel<true>, runs, dim3(kSortThreads), 0, st, sort);
    } else {
      sort.in = sort.out;
      sort.out = sort.out == sorted ? other : sorted;
      sort.shift += sort.bits;
      sort.bits = std::min(sort.bits, bits - sort.shift);
      hipLaunchKernelGGL(embed_count_kernel<false>, runs, dim3(kSortThreads), 0, st, sort);
      hipLaunchKernelGGL(embed_place_kernel<false>, runs, dim3(kSortThreads), 0, st, sort);
    }
    if (int e = check_launch("embed_place_kernel")) return e;
  }
  const SumArgs sum{dy, dy_stride, (int)dim, sorted, (uint32_t)tokens, total, l.window,
                    std::min<uint32_t>(l.window, kHalo), (uint32_t)sum_groups, scale,
                    reinterpret_cast<float*>(ws + l.parts), l.part_dim,
                    reinterpret_cast<uint32_t*>(ws + l.begins), zero};
  return with_embed_types(weight_dtype, dtype, [&](auto w, auto t) {
    using W = decltype(w);
    using T = decltype(t);
    int rc = MAXSIM_OK;
    with_shape<kVec<T>>(dim, [&](auto s) {
      constexpr int G = decltype(s)::G, K = decltype(s)::K;
      constexpr int U = K >= 3 ? 4 : 8;
      hipLaunchKernelGGL((embed_sum_kernel<T, W, G, K, U>),
                         dim3((unsigned)(sum_groups + zero_groups)), dim3(row_threads(G)), 0, st,
                         sum);
      rc = check_launch("embed_sum_kernel");
    });
    if (rc != MAXSIM_OK) return rc;
    const uint32_t share = (uint32_t)std::min<int64_t>((l.windows + 511) / 512, kJoinWindows);
    hipLaunchKernelGGL(embed_join_kernel<W>, dim3((unsigned)((l.windows + share - 1) / share)),
                       dim3(kJoinThreads), 0, st, sum, share);
    return check_launch("embed_join_kernel");
  });
}

}  // extern "C"
