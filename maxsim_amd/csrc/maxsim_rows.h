// Shared device code of the row operators (layer norm, unit rows): a group of
// G lanes holds one row of `dim` elements in registers, K chunks of 16 bytes
// (V elements) per lane, and reduces over the row without leaving the wave
// (G <= 64) or through one LDS word per wave (G = 256, 512, 1024).
//
// Lane j of a group holds chunks j, j + G, ...: consecutive lanes read
// consecutive chunks.  Rows may start at any multiple of the element size;
// the row's last chunk is read and written in pieces where dim is no multiple
// of the chunk.
#pragma once

#include "maxsim_common.h"

namespace maxsim {

template <typename T> constexpr int kVec = 16 / T::bytes;  // elements of a chunk

// gfx950's conversions round to nearest even and keep NaN and infinities.
__device__ __forceinline__ uint32_t bits16(float f, BF16) {
  return __builtin_bit_cast(uint16_t, (__bf16)f);
}
__device__ __forceinline__ uint32_t bits16(float f, F16) {
  return __builtin_bit_cast(uint16_t, (_Float16)f);
}
__device__ __forceinline__ float from16(uint32_t lo16, BF16) {
  return __uint_as_float(lo16 << 16);
}
__device__ __forceinline__ float from16(uint32_t lo16, F16) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)lo16);
}

template <typename T>
__device__ __forceinline__ float to_float(typename T::storage v) {
  if constexpr (T::bytes == 2) return from16(v, T{});
  else return v;
}
template <typename T>
__device__ __forceinline__ typename T::storage from_float(float f) {
  if constexpr (T::bytes == 2) return (uint16_t)bits16(f, T{});
  else return f;
}

// A chunk as it is in memory.
template <typename T> struct Chunk { uint32_t w[4]; };

template <typename T>
__device__ __forceinline__ void unpack(const Chunk<T>& c, float (&f)[kVec<T>]) {
  if constexpr (T::bytes == 2) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = from16(c.w[e] & 0xffffu, T{});
      f[2 * e + 1] = from16(c.w[e] >> 16, T{});
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(c.w[e]);
  }
}

template <typename T>
__device__ __forceinline__ Chunk<T> pack(const float (&f)[kVec<T>]) {
  Chunk<T> c;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (T::bytes == 2)
      c.w[e] = bits16(f[2 * e], T{}) | (bits16(f[2 * e + 1], T{}) << 16);
    else
      c.w[e] = __float_as_uint(f[e]);
  }
  return c;
}

// From and to an address that is only a multiple of the element size (the
// compiler knows what the target's loads and stores need).
template <typename R, typename S>
__device__ __forceinline__ R load_any(const S* p) {
  R v;
  __builtin_memcpy(&v, p, sizeof(v));
  return v;
}
template <typename R, typename S>
__device__ __forceinline__ void store_any(S* p, R v) {
  __builtin_memcpy(p, &v, sizeof(v));
}

// Elements [e0, e0 + V) of a row, those at or past dim as zero: the row's cut
// chunk of n elements comes in at most three pieces, by the bits of n.  For
// rows that are asked for once (unit rows): lanes past the row's end read
// nothing (1000 x 300 x 300 f16: 53 us against 60 with load_chunk).
template <typename T>
__device__ __forceinline__ Chunk<T> load_pieces(const typename T::storage* row, int e0, int dim) {
  if (e0 + kVec<T> <= dim) return load_any<Chunk<T>>(row + e0);
  Chunk<T> r = {};
  if (e0 >= dim) return r;
  const int n = dim - e0;
  const typename T::storage* p = row + e0;
  if constexpr (T::bytes == 4) {
    const uint2 a = n & 2 ? load_any<uint2>(p) : make_uint2(0, 0);
    const uint32_t c = n & 1 ? load_any<uint32_t>(p + (n & 2)) : 0;
    r.w[0] = n & 2 ? a.x : c;
    r.w[1] = a.y;
    r.w[2] = n == 3 ? c : 0;
  } else {
    const uint32_t b = n & 2 ? load_any<uint32_t>(p + (n & 4)) : 0;
    const uint32_t c = n & 1 ? p[n & 6] : 0;
    const uint32_t bc = n & 2 ? b : c, last = n & 2 ? c : 0;
    const uint2 a = n & 4 ? load_any<uint2>(p) : make_uint2(0, 0);
    r.w[0] = n & 4 ? a.x : bc;
    r.w[1] = n & 4 ? a.y : last;
    r.w[2] = n & 4 ? bc : 0;
    r.w[3] = n & 4 ? last : 0;
  }
  return r;
}

// The same in two parts, for rows that are asked for a turn ahead (layer norm):
// the load, whole and without a branch (a chunk that reaches past the row's
// end reads the row's last V elements instead), and, where the data is used,
// the move into place.  Keeping the second away from the loads lets a row's
// loads stay in flight (200000 x 300 bf16, forward and backward: 52 + 78 us
// against 57 + 86 with the branches of load_pieces).  SHORT: the row may be
// shorter than a chunk, and such a one is read by elements.
template <typename T, bool SHORT>
__device__ __forceinline__ Chunk<T> load_chunk(const typename T::storage* row, int e0, int dim) {
  constexpr int V = kVec<T>;
  if (SHORT && dim < V) {
    Chunk<T> r = {};
#pragma unroll
    for (int e = 0; e < V - 1; ++e)
      if (e0 + e < dim) {
        if constexpr (T::bytes == 2) r.w[e / 2] |= (uint32_t)row[e0 + e] << (16 * (e & 1));
        else r.w[e] = __float_as_uint(row[e0 + e]);
      }
    return r;
  }
  return load_any<Chunk<T>>(row + min(e0, dim - V));
}
template <typename T, bool SHORT>
__device__ __forceinline__ void place_chunk(Chunk<T>& c, int e0, int dim) {
  constexpr int V = kVec<T>;
  if (SHORT && dim < V) return;
  const int n = T::bytes * max(e0 - (dim - V), 0);  // bytes that belong before e0
  if (dim % V == 0) {  // all or nothing
#pragma unroll
    for (int i = 0; i < 4; ++i) c.w[i] = n ? 0 : c.w[i];
  } else {
    const uint4 r = drop_bytes(make_uint4(c.w[0], c.w[1], c.w[2], c.w[3]), n);
    c.w[0] = r.x, c.w[1] = r.y, c.w[2] = r.z, c.w[3] = r.w;
  }
}

// The row's cut chunk of n elements goes in at most three pieces, by the bits
// of n.
template <typename T>
__device__ __forceinline__ void store_chunk(typename T::storage* row, int e0, int dim,
                                            const float (&f)[kVec<T>]) {
  const Chunk<T> r = pack<T>(f);
  if (e0 + kVec<T> <= dim) {
    store_any(row + e0, r);
    return;
  }
  if (e0 >= dim) return;
  const int n = dim - e0;
  typename T::storage* p = row + e0;
  if constexpr (T::bytes == 4) {
    if (n & 2) store_any(p, make_uint2(r.w[0], r.w[1]));
    if (n & 1) store_any(p + (n & 2), n & 2 ? r.w[2] : r.w[0]);
  } else {
    if (n & 4) store_any(p, make_uint2(r.w[0], r.w[1]));
    const uint32_t b = n & 4 ? r.w[2] : r.w[0], c = n & 4 ? r.w[3] : r.w[1];
    if (n & 2) store_any(p + (n & 4), b);
    if (n & 1) p[n & 6] = (uint16_t)(n & 2 ? c : b);
  }
}

// N elements of a parameter row of type W in fp32, `fill` where there is no
// parameter and zero past dim.
template <typename W, int N>
__device__ __forceinline__ void load_param(const void* p, int e0, int dim, float fill,
                                           float (&f)[N]) {
  const typename W::storage* w = static_cast<const typename W::storage*>(p);
  constexpr int v = kVec<W>;
  static_assert(N % v == 0, "whole chunks of the parameter's type");
  if (!w) {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = fill;
  } else if (e0 + N <= dim) {
#pragma unroll
    for (int c = 0; c < N / v; ++c) {
      float part[v];
      unpack<W>(load_any<Chunk<W>>(w + e0 + c * v), part);
#pragma unroll
      for (int e = 0; e < v; ++e) f[c * v + e] = part[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = e0 + e < dim ? to_float<W>(w[e0 + e]) : 0.0f;
  }
}

// Whether the shape of G lanes takes rows shorter than a chunk.
constexpr bool takes_short(int G) { return G == 8; }

// Sum over a group of G <= 64 consecutive lanes, in every lane of it, with
// the same bits in each (each step adds the same two values).  All lanes of
// the wave have to be active.
template <int CTRL>
__device__ __forceinline__ uint32_t lane_move(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140, kRotate8 = 0x128;
template <int CTRL>
__device__ __forceinline__ float add_move(float v) {
  return v + __uint_as_float(lane_move<CTRL>(__float_as_uint(v)));
}

template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (G >= 2) v = add_move<kXor1>(v);
  if constexpr (G >= 4) v = add_move<kXor2>(v);
  if constexpr (G >= 8) v = add_move<kHalfMirror>(v);
  if constexpr (G >= 16) v = add_move<kMirror>(v);
  if constexpr (G >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (G >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// Sum over the lanes of the wave that have the same place in their groups of
// G lanes (G = 8 to 64), in every lane.
template <int G>
__device__ __forceinline__ float groups_sum(float v) {
  if constexpr (G <= 8) v = add_move<kRotate8>(v);
  if constexpr (G <= 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (G <= 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// Sums of N values over a group of G lanes.  Groups wider than a wave are
// whole workgroups: the waves' sums meet in `part` (N * G / 64 floats of LDS),
// added in one order by every thread; two `part` used in turn need no second
// barrier, since nobody writes the first again before everybody has passed
// the barrier of the other.
template <int G, int N>
__device__ __forceinline__ void group_sums(float (&v)[N], float* part) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum<(G < 64 ? G : 64)>(v[i]);
  if constexpr (G > 64) {
    constexpr int waves = G / 64;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) part[i * waves + wave] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = part[i * waves];
#pragma unroll
      for (int w = 1; w < waves; ++w) s += part[i * waves + w];
      v[i] = s;
    }
  }
}

// Largest over a group of G lanes, in every lane (wider groups through G / 64
// words of LDS, between barriers of its own).
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v, uint32_t* part) {
#pragma unroll
  for (int off = 1; off < (G < 64 ? G : 64); off <<= 1) v = max(v, __shfl_xor(v, off, 64));
  if constexpr (G > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < G / 64; ++w) v = max(v, part[w]);
    __syncthreads();
  }
  return v;
}

// ---- the shapes (host) -----------------------------------------------------

// Calls f with the group shape for rows of `dim` elements (up to
// MAXSIM_AMD_MAX_DIM) in chunks of V: the one that leaves fewest lanes idle
// among those that hold a row in at most three chunks per lane (four in fp32
// rows past 8192 elements); more lanes than a wave where that is not enough.  (Rows of 768 elements of 16 bits, 96
// chunks of 8: 32 lanes x 3.)  512 threads where they hold a row:
// two such workgroups on a CU work at each other's barriers (layer norm of 8000
// x 12288 bf16 backward 122 us, with 1024 threads 137; 12000 x 8192 forward 72
// against 75).
template <int G_, int K_> struct Shape { static constexpr int G = G_, K = K_; };
template <int V, typename F>
inline void with_shape(int64_t dim, F&& f) {
  const int64_t chunks = (dim + V - 1) / V;
  if (chunks <= 8) f(Shape<8, 1>{});
  else if (chunks <= 16) f(Shape<16, 1>{});
  else if (chunks <= 32) f(Shape<16, 2>{});
  else if (chunks <= 48) f(Shape<16, 3>{});
  else if (chunks <= 64) f(Shape<32, 2>{});
  else if (chunks <= 96) f(Shape<32, 3>{});
  else if (chunks <= 128) f(Shape<64, 2>{});
  else if (chunks <= 192) f(Shape<64, 3>{});
  else if (chunks <= 256) f(Shape<256, 1>{});
  else if (chunks <= 512) f(Shape<256, 2>{});
  else if (chunks <= 768) f(Shape<256, 3>{});
  else if (chunks <= 1024) f(Shape<512, 2>{});
  else if (chunks <= 1536) f(Shape<512, 3>{});
  else if (V == 8 || chunks <= 2048) f(Shape<1024, 2>{});
  else if constexpr (V < 8) f(Shape<1024, 4>{});
}
constexpr int row_threads(int G) { return G > 256 ? G : 256; }

}  // namespace maxsim
