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
// that the ids and the sizes alone decide every order:
//   embed_few_kernel   few tokens: one launch does all of it in LDS;
//   embed_count_kernel, embed_place_kernel   a pass of the sort of many;
//   embed_sum_kernel   groups of lanes add up the tokens of one row each, of
//                      rows with many a part; more write zeros for rows without;
//   embed_join_kernel  adds those parts.
#include <algorithm>

#include "maxsim_host.h"
#include "maxsim_rows.h"
#include "../../include/maxsim_amd_encoder.h"

namespace maxsim {

// ---- forward -----------------------------------------------------------------

// A result of more bytes than this goes past the caches, which then keep the
// table (524288 tokens x 768, fp32 table of 32000 rows, bf16 result, one launch
// after the other: 217 us against 310, or 157 against 284 where 229376 of the
// tokens are padding; with a table that other work has pushed out of the caches
// 289 against 309 and 268 against 276; and 579 against 617 with the layer norm
// that reads the result).  A smaller one is mostly still there for its reader
// (40000 tokens: 18.7 against 20.1 us, but 42.4 against 41.5 with the layer
// norm; 80000, 123 MB: 79 against 90).  Rows that share lines with their neighbours leave pieces of lines behind, which
// costs short ones more than it gives (256000 x 304 bf16: 44 us against 35, x 301
// fp32 99 and 99, x 1038 bf16 137 against 199).
constexpr int64_t kCacheBytes = (int64_t)96 << 20, kCacheRow = 2048;

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

// 16 bytes that the caches need not keep.
template <typename T>
__device__ __forceinline__ void store_past_cache(typename T::storage* p, const Chunk<T>& c) {
  typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
  __builtin_nontemporal_store(Words{c.w[0], c.w[1], c.w[2], c.w[3]}, reinterpret_cast<Words*>(p));
}

// A group of G lanes looks up U tokens, GROUPS apart: their ids (and lengths)
// are asked for together, then their rows.
template <typename W, typename T, int G, int K, int U, bool PAST_CACHE>
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
      const int e0 = (j + k * G) * V;
      if (PAST_CACHE && e0 + V <= dim) store_past_cache(to + e0, pack<T>(f));
      else store_chunk<T>(to, e0, dim, f);
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

// A stretch of the table that a workgroup looks after: rows without a token
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
constexpr int kTokenBits = 11, kFewTokens = 1 << kTokenBits;
constexpr int kBucketBits = 8;   // low bits of a row: a workgroup per CU
constexpr int kFewVocabBits = 32 - kTokenBits + kBucketBits;
constexpr int kFewDigitBits = 8; // high bits that a pass sorts by
constexpr int kFewBlocks = 4;    // of 64 chunks of 16 bytes: a row at most
constexpr int kWaveIds = kFewTokens / kSortWaves;
static_assert(kWaveIds == 64 * 2, "two ids per lane");

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

// Two ids in a row; past the end there is no row.
__device__ __forceinline__ void load_rows(const int32_t* rows, uint32_t i, uint32_t n,
                                          uint32_t (&key)[2]) {
  if (i + 2 <= n) {
    const uint2 q = load_any<uint2>(rows + i);
    key[0] = q.x, key[1] = q.y;
  } else {
    key[0] = i < n ? (uint32_t)rows[i] : kNoRow;
    key[1] = kNoRow;
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
  uint32_t key[2];
  const uint32_t i0 = wave * kWaveIds + lane * 2;
  load_rows(a.rows, i0, a.tokens, key);

  if (blockIdx.x >= a.buckets) {
    const uint32_t first = (blockIdx.x - a.buckets) * a.zero.rows;
    if (threadIdx.x < kZeroRows / 32) lds.has[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
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
  uint64_t own[2];
  uint32_t at = 0, mine = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    own[e] = __ballot(key[e] < a.zero.vocab && (key[e] & low) == bucket);
    at += set_before(own[e]);
    mine += (uint32_t)__popcll(own[e]);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
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

  // Sums: waves share the columns, kColumns each (kFewBlocks of those at most),
  // and the sorted tokens.  A run that began in an earlier wave's share is left
  // in LDS for that wave.
  const int across = (a.dim + kColumns - 1) / kColumns, shares = kSortWaves / across;
  const int share = wave / across;
  const uint32_t take = (m + shares - 1) / shares;
  const uint32_t begin = share < shares ? min(share * take, m) : m, end = min(begin + take, m);
  auto row_at = [&](uint32_t i) { return sorted[i] >> kTokenBits; };
  const bool joins = begin > 0 && begin < end && row_at(begin) == row_at(begin - 1);
  const bool goes_on = begin < end && end < m && row_at(end) == row_at(end - 1);
  const int e0 = wave % across * kColumns + lane * V;
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
  auto leave_part = [&] {
#pragma unroll
    for (int e = 0; e < V; ++e) lds.parts[wave][lane * V + e] = acc[e];
  };
  bool part = joins;
  uint32_t row = begin < end ? row_at(begin) : 0;
  for (uint32_t i = begin; i < end; i += U) {
    Chunk<T> raw[U];
    uint32_t entry[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      entry[u] = sorted[min(i + u, end - 1)];
      const S* dy = static_cast<const S*>(a.dy) + (entry[u] & (kFewTokens - 1)) * a.dy_row;
      raw[u] = load_chunk<T, true>(dy, e0, a.dim);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= end) break;
      if (entry[u] >> kTokenBits != row) {
        if (part) leave_part();
        else write_row(row);
        part = false;
        row = entry[u] >> kTokenBits;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.0f;
      }
      float f[V];
      place_chunk<T, true>(raw[u], e0, a.dim);
      unpack<T>(raw[u], f);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += f[e];
    }
  }
  if (begin < end) {
    if (part) leave_part();
    else if (!goes_on) write_row(row);
  }
  __syncthreads();
  if (goes_on && !part) {
    for (int s = share + 1; s < shares; ++s) {
      if (s * take >= m || row_at(s * take) != row) break;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += lds.parts[s * across + wave % across][lane * V + e];
    }
    write_row(row);
  }
}

// ---- backward: the sort of many ------------------------------------------------

// Stable passes by kDigitBits of the row each, from the lowest.  The workgroups
// of a pass each have a run of the entries; embed_count_kernel counts a run's
// digits, embed_place_kernel adds up what the others counted and moves its run.
// Where the entries are few, each workgroup counts all of them itself, which
// saves the launches (18283 tokens, two passes: the gradient 34.7 us against
// 38.5; 30000: 47.4 against 41.0).
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSortGroups = 128;  // most workgroups of a pass
constexpr int kCountAll = 20480;  // entries that every workgroup counts
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
  uint32_t* begun;   // which it clears, for the sums
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

template <bool FIRST, bool COUNTED>
__global__ __launch_bounds__(kSortThreads) void embed_place_kernel(SortArgs a) {
  __shared__ uint32_t counts[kSortWaves][kDigits];
  __shared__ uint32_t sums[COUNTED ? 2 * kSortThreads : kDigits], waves[kSortWaves];
  const int wave = threadIdx.x >> 6;
  const uint32_t digits = 1u << a.bits, mask = digits - 1;
  const uint32_t n = FIRST ? a.tokens : *a.total;
  count_share<FIRST>(a, n, counts[wave]);
  // of a digit: all entries, and those of the runs before
  uint32_t all = 0, before = 0;
  if constexpr (!COUNTED) {
    // the former in the low half of a word, the latter in the high
    static_assert(kCountAll < 65536, "counts of 16 bits");
    if (threadIdx.x < digits) sums[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t begin = blockIdx.x * a.run;
    constexpr int U = 8;
    for (uint32_t i0 = 0; i0 < n; i0 += kSortThreads * U) {
      uint32_t row[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t i = min(i0 + u * kSortThreads + threadIdx.x, n - 1);
        row[u] = FIRST ? (uint32_t)a.rows[i] : a.in[i].row;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t i = i0 + u * kSortThreads + threadIdx.x;
        if (i < n && row[u] < a.vocab)
          atomicAdd(&sums[row[u] >> a.shift & mask], i < begin ? 0x10001u : 1u);
      }
    }
    __syncthreads();
    if (threadIdx.x < digits)
      all = sums[threadIdx.x] & 0xffff, before = sums[threadIdx.x] >> 16;
  } else {
    // several threads each
    const uint32_t d = threadIdx.x & mask, part = threadIdx.x >> a.bits;
    const uint32_t parts = min((uint32_t)kSortThreads >> a.bits, 16u);
    const uint32_t groups = part < parts ? gridDim.x : 0;
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
    sums[threadIdx.x] = all, sums[kSortThreads + threadIdx.x] = before;
    __syncthreads();
    all = before = 0;
    if (threadIdx.x < digits)
      for (uint32_t i = threadIdx.x; i < digits * parts; i += digits)
        all += sums[i], before += sums[kSortThreads + i];
  }
  uint32_t start = sum_before(all, waves);
  if (FIRST && blockIdx.x == 0 && threadIdx.x == kSortThreads - 1)
    *a.total = start + all, *a.begun = 0;
  start += before;
  if (threadIdx.x < digits)
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = counts[w][threadIdx.x];
      counts[w][threadIdx.x] = start;
      start += c;
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

// A run is a row's sorted tokens.  A workgroup has `span` sorted tokens, whose
// runs its groups of lanes add up one by one, whichever is free the next: a run
// of up to `short_run` tokens where it begins, of a longer one the part in each
// window (spans are whole windows).  Parts of a run that reaches into other
// windows are left in the workspace.  More workgroups write zeros.
constexpr int kMaxShortRun = 64, kMaxSpan = 512;

struct SumArgs {
  const void* dy;
  int64_t dy_row;  // stride in elements
  int dim;
  const Entry* sorted;
  const uint32_t* total;
  uint32_t span, window;  // powers of two
  uint32_t short_run;
  uint32_t spans;         // workgroups that add up
  float scale;
  float* parts;     // [windows][2][part_dim]: of a run from before, of one that begins here
  int part_dim;
  uint2* begins;    // windows where a run begins that goes on, and its row, in any order
  uint32_t* begun;  // their number
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

// The same by one lane, among entries [lo, hi).
__device__ __forceinline__ uint32_t first_among(const Entry* sorted, uint32_t lo, uint32_t hi,
                                                uint64_t row) {
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (sorted[mid].row < row) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// acc = the sum of the rows of dy that token_of(first) to token_of(last - 1)
// name, in that order, U rows in flight.
template <typename T, int G, int K, int U, typename F>
__device__ __forceinline__ void sum_rows(const SumArgs& a, uint32_t first, uint32_t last,
                                         F&& token_of, float (&acc)[K][kVec<T>]) {
  constexpr int V = kVec<T>;
  constexpr bool SHORT = takes_short(G);
  const int j = threadIdx.x % G;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) acc[k][e] = 0.0f;
  for (uint32_t i = first; i < last; i += U) {
    Chunk<T> raw[U][K];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // past the last, the last again: its lines are on their way
      const auto* row = static_cast<const typename T::storage*>(a.dy) +
                        (int64_t)token_of(min(i + u, last - 1)) * a.dy_row;
#pragma unroll
      for (int k = 0; k < K; ++k) raw[u][k] = load_chunk<T, SHORT>(row, (j + k * G) * V, a.dim);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool has = i + u < last;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float f[V];
        place_chunk<T, SHORT>(raw[u][k], (j + k * G) * V, a.dim);
        unpack<T>(raw[u][k], f);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[k][e] += has ? f[e] : 0.0f;
      }
    }
  }
}

template <typename T, typename W, int G, int K, int U>
__global__ __launch_bounds__(row_threads(G)) void embed_sum_kernel(SumArgs a) {
  constexpr int V = kVec<T>, THREADS = row_threads(G);
  __shared__ union {
    struct {
      Entry entries[kMaxSpan + 2 * kMaxShortRun];
      uint32_t list[kMaxSpan], used, next;
    } span;
    struct { uint32_t bounds[2], has[kZeroRows / 32]; } zero;
  } lds;
  const uint32_t total = *a.total;

  if (blockIdx.x >= a.spans) {
    const uint32_t first = (blockIdx.x - a.spans) * a.zero.rows;
    for (int i = threadIdx.x; i < kZeroRows / 32; i += THREADS) lds.zero.has[i] = 0;
    if (threadIdx.x < 128) {
      const int which = threadIdx.x >> 6;
      const uint32_t i = first_of(a.sorted, total, (uint64_t)first + which * a.zero.rows);
      if ((threadIdx.x & 63) == 0) lds.zero.bounds[which] = i;
    }
    __syncthreads();
    // from entries that are few, or by a search for each row: a frequent one's
    // are as many as they like (524288 tokens: the launch 200 us without it)
    const uint32_t lo = lds.zero.bounds[0], hi = lds.zero.bounds[1];
    const uint32_t rows = min(a.zero.rows, a.zero.vocab - first);
    const bool search = hi - lo > 4 * THREADS;
    for (uint32_t t = threadIdx.x; t < (search ? rows : hi - lo); t += THREADS) {
      const uint32_t i = search ? first_among(a.sorted, lo, hi, (uint64_t)first + t) : lo + t;
      const uint32_t r = i < hi ? a.sorted[i].row - first : rows;
      if (r < rows) atomicOr(&lds.zero.has[r / 32], 1u << (r & 31));
    }
    __syncthreads();
    zero_rows(a.zero, first, lds.zero.has);
    return;
  }

  // the span's entries and those around them; kNoRow where there are none
  const int64_t base = (int64_t)blockIdx.x * a.span;
  if (base >= total) return;
  const int span = (int)a.span, short_run = (int)a.short_run;
  for (int t = threadIdx.x; t < span + 2 * short_run; t += THREADS) {
    const int64_t i = base - short_run + t;
    lds.span.entries[t] = i >= 0 && i < total ? a.sorted[i] : Entry{kNoRow, 0};
  }
  if (threadIdx.x == 0) lds.span.used = lds.span.next = 0;
  __syncthreads();
  const Entry* entries = lds.span.entries + short_run;
  // What is to be added up: from entry t on where a run begins with it, or
  // where a window does inside of a long run.  In any order: none has to do
  // with another.
  const int n = (int)min((int64_t)span, (int64_t)total - base), window = (int)a.window;
  for (int t = threadIdx.x; t < n; t += THREADS) {
    const uint32_t row = entries[t].row;
    const bool starts = entries[t - 1].row != row, edge = (t & (window - 1)) == 0;
    if (!starts && !edge) continue;
    int start = t;  // of the run, or short_run before t where it is further
    if (!starts) {
      int lo = t - short_run;
      while (lo < start) {
        const int mid = (lo + start) >> 1;
        if (entries[mid].row == row) start = mid;
        else lo = mid + 1;
      }
    }
    const bool is_long = start == t - short_run || entries[start + short_run].row == row;
    if (!is_long && !starts) continue;
    // its end, or the window's that a long run reaches past
    int lo = t + 1, hi = is_long ? min((t | (window - 1)) + 1, n) : t + short_run;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (entries[mid].row == row) lo = mid + 1;
      else hi = mid;
    }
    lds.span.list[atomicAdd(&lds.span.used, 1u)] = (uint32_t)t | (uint32_t)hi << 16;
  }
  __syncthreads();
  const uint32_t used = lds.span.used;
  const int j = threadIdx.x % G;
  for (;;) {
    uint32_t i = 0;
    if constexpr (G <= 64) {
      if (j == 0) i = atomicAdd(&lds.span.next, 1u);
      i = (uint32_t)__shfl((int)i, (int)(threadIdx.x & 63) / G * G, 64);
    } else {
      i = lds.span.next;
      __syncthreads();
      if (threadIdx.x == 0) lds.span.next = i + 1;
      __syncthreads();
    }
    if (i >= used) break;
    const int lo = lds.span.list[i] & 0xffff, hi = lds.span.list[i] >> 16;
    float acc[K][V];
    sum_rows<T, G, K, U>(a, (uint32_t)lo, (uint32_t)hi,
                         [&](uint32_t i) { return entries[i].token; }, acc);
    const uint32_t row = entries[lo].row;
    const bool from_before = entries[lo - 1].row == row;
    const bool goes_on = entries[hi].row == row;  // only a long one's part ends inside of it
    if (!from_before && !goes_on) {
      auto* to = static_cast<typename W::storage*>(a.zero.dweight) + (int64_t)row * a.dim;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < V; ++e) acc[k][e] *= a.scale;
        store_piece<W, V>(to, (j + k * G) * V, a.dim, acc[k]);
      }
      continue;
    }
    const uint32_t number = (uint32_t)((base + lo) / window);
    float* to = a.parts + ((int64_t)number * 2 + (from_before ? 0 : 1)) * a.part_dim;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int e0 = (j + k * G) * V;
#pragma unroll
      for (int e = 0; e < V; e += 4)
        if (e0 + e < a.part_dim)
          store_any(to + e0 + e, make_float4(acc[k][e], acc[k][e + 1], acc[k][e + 2], acc[k][e + 3]));
    }
    if (!from_before && j == 0) a.begins[atomicAdd(a.begun, 1u)] = make_uint2(number, row);
  }
}

// Adds up the parts of the runs that go on from the window that they begin in,
// a workgroup a run and kJoinColumns of its columns; a thread has four of them,
// and of the parts a share.  Where the runs are few and long, as with a table of
// a few rows, 4 or 16 workgroups divide the columns among them and have as many
// more shares.
constexpr int kJoinThreads = 512, kJoinUnroll = 8, kJoinColumns = 256;
template <typename W>
__global__ __launch_bounds__(kJoinThreads) void embed_join_kernel(SumArgs a) {
  __shared__ float4 sums[kJoinThreads];
  const uint32_t runs = *a.begun, total = *a.total;
  const uint32_t windows = total / a.window;  // of a run: windows / runs on average at most
  const uint32_t split = runs * 16 <= gridDim.x && windows / 64 >= runs  ? 16
                         : runs * 4 <= gridDim.x && windows / 16 >= runs ? 4
                                                                         : 1;
  const int across = kJoinColumns / 4 / split, shares = kJoinThreads / across;
  const int mine = threadIdx.x / across;
  const int e0 = blockIdx.y * kJoinColumns +
                 (blockIdx.x % split * across + threadIdx.x % across) * 4;
  const bool has = e0 < a.dim;
  for (uint32_t r = blockIdx.x / split; r < runs; r += gridDim.x / split) {
    const uint2 run = a.begins[r];
    const uint64_t begin = (uint64_t)run.x * a.window;
    // the windows after it that the run reaches into
    const uint64_t i = begin + (uint64_t)(1 + (threadIdx.x & 63)) * a.window;
    const uint64_t same = __ballot(i < total && a.sorted[min(i, (uint64_t)total - 1)].row == run.y);
    uint32_t more = (uint32_t)__popcll(same);
    if (more == 64) more = (first_of(a.sorted, total, (uint64_t)run.y + 1) - 1) / a.window - run.x;
    const uint32_t take = (more + shares - 1) / shares;
    const uint32_t lo = min(mine * take, more), hi = min(lo + take, more);
    const float* p = a.parts + (int64_t)run.x * 2 * a.part_dim + e0;
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
    sums[threadIdx.x] = s;
    __syncthreads();
    if (mine == 0 && has) {
      static_assert(kJoinThreads / (kJoinColumns / 4) == 8, "shares are a multiple of 8");
      s = make_float4(0, 0, 0, 0);
      for (int i = 0; i < shares; i += 8) {
        float4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = sums[(i + u) * across + threadIdx.x];
#pragma unroll
        for (int u = 0; u < 8; ++u) s.x += v[u].x, s.y += v[u].y, s.z += v[u].z, s.w += v[u].w;
      }
      auto* out = static_cast<typename W::storage*>(a.zero.dweight) + (int64_t)run.y * a.dim;
      const float f[4] = {s.x * a.scale, s.y * a.scale, s.z * a.scale, s.w * a.scale};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e0 + e < a.dim) out[e0 + e] = from_float<W>(f[e]);
    }
    __syncthreads();
  }
}

// ---- sizes -------------------------------------------------------------------

static int bits_of(uint64_t n) {  // that numbers below n have
  int b = 0;
  while (((uint64_t)1 << b) < n) ++b;
  return b;
}

// Whether the one launch is the faster.  A workgroup of it has all tokens of a
// row, so not where rows are few (a table of 6 rows: 496 tokens at most; 3654 of
// 6 rows 41 us against 19, 512 of 16 10 against 17) or so wide that its waves
// share the columns alone (796 x 2560 fp32: 77 against 28; 2048 x 768 bf16 of
// 32000 rows: 14 against 29).  4096 tokens would be 19 against 31, but 153
// against 38 if all are of one row; the limit of 2048 leaves 78 against 31 there.
// No tokens at all are the zeros alone, of rows of any width and number: nothing
// is sorted, and the other path's shares would be empty.
static bool few_tokens(maxsim_dtype dtype, int64_t tokens, int64_t vocab, int64_t dim) {
  if (tokens == 0) return true;
  const int64_t columns = dtype == MAXSIM_FLOAT32 ? 64 * kVec<F32> : 64 * kVec<F16>;
  return tokens <= std::min<int64_t>(256 + 40 * vocab, kFewTokens) && dim <= kFewBlocks * columns &&
         bits_of((uint64_t)vocab) <= kFewVocabBits;
}

// Threads of a workgroup that adds up rows, and the groups of lanes in it that
// hold a row each.
struct RowGroups { int threads, groups; };
static RowGroups row_groups(maxsim_dtype dtype, int64_t dim) {
  RowGroups r{};
  auto of = [&](auto s) {
    constexpr int G = decltype(s)::G;
    r = {row_threads(G), row_threads(G) / G};
  };
  if (dtype == MAXSIM_FLOAT32) with_shape<kVec<F32>>(dim, of);
  else with_shape<kVec<F16>>(dim, of);
  return r;
}

struct EmbedLayout {
  int64_t windows;
  uint32_t window, span, short_run;  // tokens
  uint32_t run;           // tokens of a workgroup of the sort
  int part_dim;
  size_t sorted, other, counts, begins, parts, bytes;  // offsets, and all
};
static EmbedLayout embed_layout(maxsim_dtype dtype, int64_t tokens, int64_t vocab, int64_t dim) {
  EmbedLayout l{};
  if (few_tokens(dtype, tokens, vocab, dim)) return l;
  // a group of lanes has up to 32 tokens, fewer where that leaves CUs idle
  const uint32_t groups = (uint32_t)row_groups(dtype, dim).groups;
  uint32_t share = 32;
  while (share > 2 && tokens / share < 8192) share /= 2;
  l.span = std::min<uint32_t>(std::max<uint32_t>(groups * share, 8), kMaxSpan);
  // what the others have long done when a group ends with it
  l.short_run = std::min<uint32_t>(std::max<uint32_t>(2 * share, 16), kMaxShortRun);
  l.window = std::min(l.span, l.short_run);
  l.windows = (tokens + l.window - 1) / l.window;
  l.part_dim = (int)((dim + 7) / 8 * 8);
  const int64_t each = (tokens + kSortGroups - 1) / kSortGroups;
  l.run = (uint32_t)((each + kSortThreads - 1) / kSortThreads * kSortThreads);
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  l.sorted = 256;  // two numbers first
  l.other = l.sorted + up((size_t)tokens * sizeof(Entry));
  l.counts = l.other + up((size_t)tokens * sizeof(Entry));
  l.begins = l.counts + (size_t)kSortGroups * kDigits * sizeof(uint32_t);
  l.parts = l.begins + up((size_t)l.windows * sizeof(uint2));
  l.bytes = l.parts + (size_t)l.windows * 2 * l.part_dim * sizeof(float);
  return l;
}

static ZeroArgs zero_args(void* dweight, int64_t vocab, int64_t row_bytes, int element) {
  const int64_t rows = std::min<int64_t>(std::max<int64_t>(kZeroBytes / row_bytes, 1), kZeroRows);
  return ZeroArgs{dweight, row_bytes, (uint32_t)vocab, (uint32_t)rows, element};
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
  const int64_t row_bytes = dim * (dtype == MAXSIM_FLOAT32 ? 4 : 2);
  const bool past_cache = all.tokens * row_bytes > kCacheBytes &&
                          (row_bytes % 64 == 0 || row_bytes >= kCacheRow);
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
        if (past_cache)
          hipLaunchKernelGGL((embed_kernel<W, T, G, K, U, true>), dim3((unsigned)blocks),
                             dim3(threads), 0, static_cast<hipStream_t>(stream), a);
        else
          hipLaunchKernelGGL((embed_kernel<W, T, G, K, U, false>), dim3((unsigned)blocks),
                             dim3(threads), 0, static_cast<hipStream_t>(stream), a);
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
  if (few_tokens(dtype, tokens, vocab, dim)) {
    ZeroArgs zero = zero_args(dweight, vocab, dim * element, element);
    // one such workgroup per CU, beside one with a bucket
    zero.rows = std::max(zero.rows, (uint32_t)std::min<int64_t>((vocab + 255) / 256, kZeroRows));
    const int64_t zero_groups = (vocab + zero.rows - 1) / zero.rows;
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

  const ZeroArgs zero = zero_args(dweight, vocab, dim * element, element);
  const int64_t spans = (tokens + l.span - 1) / l.span;
  const int64_t blocks = spans + (vocab + zero.rows - 1) / zero.rows;
  // a launch's threads fit 32 bits, those of 2^31 - 1 tokens of narrow rows too
  if (blocks > UINT32_MAX / row_groups(dtype, dim).threads)
    return fail(MAXSIM_ERR_UNSUPPORTED, "table or gradient too large for one launch");
  char* ws = static_cast<char*>(workspace);
  uint32_t* total = reinterpret_cast<uint32_t*>(ws);
  Entry* sorted = reinterpret_cast<Entry*>(ws + l.sorted);
  Entry* other = reinterpret_cast<Entry*>(ws + l.other);
  const int passes = std::max((bits + kDigitBits - 1) / kDigitBits, 1);
  SortArgs sort{rows, nullptr, passes & 1 ? sorted : other, (uint32_t)tokens, (uint32_t)vocab, l.run,
                0, (bits + passes - 1) / passes, reinterpret_cast<uint32_t*>(ws + l.counts), total, total + 1};
  const dim3 runs((unsigned)((tokens + l.run - 1) / l.run));
  const bool counted = tokens > kCountAll;
  for (int p = 0; p < passes; ++p) {
    if (p > 0) {
      sort.in = sort.out;
      sort.out = sort.out == sorted ? other : sorted;
      sort.shift += sort.bits;
      sort.bits = std::min(sort.bits, bits - sort.shift);
    }
    auto launch = [&](auto first) {
      constexpr bool FIRST = decltype(first)::value;
      const dim3 threads(kSortThreads);
      if (counted) {
        hipLaunchKernelGGL(embed_count_kernel<FIRST>, runs, threads, 0, st, sort);
        hipLaunchKernelGGL((embed_place_kernel<FIRST, true>), runs, threads, 0, st, sort);
      } else {
        hipLaunchKernelGGL((embed_place_kernel<FIRST, false>), runs, threads, 0, st, sort);
      }
    };
    if (p == 0) launch(std::true_type{});
    else launch(std::false_type{});
    if (int e = check_launch("embed_place_kernel")) return e;
  }
  const SumArgs sum{dy, dy_stride, (int)dim, sorted, total, l.span, l.window, l.short_run,
                    (uint32_t)spans, scale,
                    reinterpret_cast<float*>(ws + l.parts), l.part_dim,
                    reinterpret_cast<uint2*>(ws + l.begins), total + 1, zero};
  return with_embed_types(weight_dtype, dtype, [&](auto w, auto t) {
    using W = decltype(w);
    using T = decltype(t);
    int rc = MAXSIM_OK;
    with_shape<kVec<T>>(dim, [&](auto s) {
      constexpr int G = decltype(s)::G, K = decltype(s)::K;
      constexpr int U = 2;
      hipLaunchKernelGGL((embed_sum_kernel<T, W, G, K, U>),
                         dim3((unsigned)blocks), dim3(row_threads(G)), 0, st, sum);
      rc = check_launch("embed_sum_kernel");
    });
    if (rc != MAXSIM_OK) return rc;
    const unsigned blocks = (unsigned)((dim + kJoinColumns - 1) / kJoinColumns);
    hipLaunchKernelGGL(embed_join_kernel<W>,
                       dim3((unsigned)std::min<int64_t>(l.windows, 4096 / blocks), blocks),
                       dim3(kJoinThreads), 0, st, sum);
    return check_launch("embed_join_kernel");
  });
}

}  // extern "C"
