// Shared device code of the row operators (layer norm, unit rows): a group of
// G lanes holds one row of `dim` elements in registers, K chunks of 16 bytes
// per lane, and reduces over the row without leaving the wave (G <= 64) or
// through one LDS word per wave (G = 256, 1024).
//
// Lane j of a group holds chunks j, j + G, ...: consecutive lanes read
// consecutive 16 bytes.  Rows may start at any multiple of the element size
// (load16_any); the row's last chunk is read and written by elements where
// dim is no multiple of the chunk.
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

template <typename T>
__device__ __forceinline__ void unpack16(uint4 v, float (&f)[kVec<T>]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (T::bytes == 2) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = from16(w[e] & 0xffffu, T{});
      f[2 * e + 1] = from16(w[e] >> 16, T{});
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(w[e]);
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&f)[kVec<T>]) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (T::bytes == 2)
      w[e] = bits16(f[2 * e], T{}) | (bits16(f[2 * e + 1], T{}) << 16);
    else
      w[e] = __float_as_uint(f[e]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename S>
__device__ __forceinline__ void store16_any(S* p, uint4 v) {
  __builtin_memcpy(p, &v, sizeof(v));
}

// Elements [e0, e0 + kVec) of a row, those at or past dim as zero.
template <typename T>
__device__ __forceinline__ uint4 load_chunk(const typename T::storage* row, int e0, int dim) {
  if (e0 + kVec<T> <= dim) return load16_any(row + e0);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < kVec<T>; ++e)
    if (e0 + e < dim) {
      if constexpr (T::bytes == 2) w[e / 2] |= (uint32_t)row[e0 + e] << (16 * (e & 1));
      else w[e] = __float_as_uint(row[e0 + e]);
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__device__ __forceinline__ void store_chunk(typename T::storage* row, int e0, int dim,
                                            const float (&f)[kVec<T>]) {
  if (e0 + kVec<T> <= dim) {
    store16_any(row + e0, pack16<T>(f));
    return;
  }
#pragma unroll
  for (int e = 0; e < kVec<T>; ++e)
    if (e0 + e < dim) row[e0 + e] = from_float<T>(f[e]);
}

// N elements of a parameter row of type W in fp32, `fill` where there is no
// parameter and zero past dim.
template <typename W, int N>
__device__ __forceinline__ void load_param(const void* p, int e0, int dim, float fill,
                                           float (&f)[N]) {
  const typename W::storage* w = static_cast<const typename W::storage*>(p);
  constexpr int v = kVec<W>;
  static_assert(N % v == 0 || N < v, "whole chunks of the parameter's type");
  if (!w) {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = fill;
  } else if (N % v == 0 && e0 + N <= dim) {
#pragma unroll
    for (int c = 0; c < N / v; ++c) {
      float part[v];
      unpack16<W>(load16_any(w + e0 + c * v), part);
#pragma unroll
      for (int e = 0; e < v; ++e) f[c * v + e] = part[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = e0 + e < dim ? to_float<W>(w[e0 + e]) : 0.0f;
  }
}

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

// ---- the shapes (host) -----------------------------------------------------

// Calls f with the group shape for rows of `dim` elements (up to
// MAXSIM_AMD_MAX_DIM): the one that leaves fewest lanes idle among those that
// hold a row in at most three chunks per lane; more lanes than a wave where
// that is not enough.  (Rows of 768 elements of 16 bits, 96 chunks: 32 lanes
// x 3.)
template <int G_, int K_> struct Shape { static constexpr int G = G_, K = K_; };
template <typename T, typename F>
inline void with_shape(int64_t dim, F&& f) {
  const int64_t chunks = (dim + kVec<T> - 1) / kVec<T>;
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
  else if (chunks <= 1024) f(Shape<1024, 1>{});
  else if (T::bytes == 2 || chunks <= 2048) f(Shape<1024, 2>{});
  else if constexpr (T::bytes == 4) f(Shape<1024, 4>{});
}
constexpr int row_threads(int G) { return G > 256 ? G : 256; }

}  // namespace maxsim
