// The AdamW step over many tensors at once, with states in 32 or 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps),
//       the two things that leave p added up before the one subtraction
//
// Memory-bound: 28 bytes per element in fp32, 10 in bf16 with 8-bit states.
// A launch takes up to kTensors tensors by their addresses in its arguments
// (nothing is copied to the device or kept there) and cuts each into chunks,
// one per workgroup; a workgroup finds its tensor by one load of the first
// chunks' numbers, a tensor per lane, and a count of those up to its own.
//
// 8-bit states.  A block of 256 elements of a tensor shares, per state, one
// byte: the exponent field E of its largest magnitude.  The code of an element
// is the top of the fp32 pattern of |value| moved down by a power of two that
// puts E at exponent field 14 (m: sign, 4 exponent and 3 mantissa bits) or 30
// (v: 5 and 3 bits, no sign), so that the block's small values reach into
// fp32's subnormal numbers, whose even spacing is the codes' own lowest step.
// The 20 bits below the cut decide the rounding, up or down in proportion, by
// adding 16 random bits in their upper places and half of the last of those (a
// rounding to 2^-16 of a step, without a bias): with b2 = 0.999 a second moment moves by a thousandth
// per step, and nearest rounding to steps of an eighth would never let it
// move.  The random bits are a hash of the element's position, the step and a
// seed: the same call gives the same bits.  A second moment above 0 keeps a
// code above 0, so that no step divides by eps alone.  The step itself uses m
// and v before they are rounded.  E = 255 (a value of the block is not
// finite) reads back as NaN.
#include <cmath>

#include "maxsim_host.h"
#include "maxsim_rows.h"
#include "../../include/maxsim_amd_training.h"

namespace maxsim {

constexpr int kAdamThreads = 256;
constexpr int kLaneElems = 8;  // elements of a lane: 32 lanes are a block
constexpr int kBlock = MAXSIM_AMD_STATE_BLOCK;
static_assert(kBlock == 32 * kLaneElems, "half a wave holds a block");
// One turn per workgroup: with two (and their loads together) the registers
// halve the waves, 384 against 364 us for 66 M fp32 parameters.
constexpr int kChunkElems = kAdamThreads * kLaneElems;
constexpr int64_t kMaxElems = (int64_t)1 << 40;  // of a step: 32-bit block numbers
constexpr int64_t kMaxChunks = UINT32_MAX / kAdamThreads;  // of a launch: threads in 32 bits

// LDS that a workgroup of the 32-bit step asks for and does not use: it keeps a
// CU at two workgroups, 64 KB of loads in flight.  More get into each other's
// way in the memory (66 M fp32 parameters: 346 us with two, 353 with four, 355
// with eight; bf16 273 / 284).  The 8-bit step has half the bytes and more
// arithmetic per element, and needs all eight.
constexpr unsigned kReservedLds = 56 << 10;

// The tensors of a launch, as many as 4 KB of kernel arguments hold (90 in
// the plain 32-bit step, 62 with 8-bit states and masters).
template <int BITS, bool MASTER> struct AdamArgs {
  static constexpr int kTensors =
      (4096 - 128) / (5 * 8 + 4 + (BITS == 8 ? 8 + 4 : 0) + (MASTER ? 8 : 0));
  void* p[kTensors];
  const void* g[kTensors];
  void* m[kTensors];
  void* v[kTensors];
  int64_t n[kTensors];
  uint8_t* scales[BITS == 8 ? kTensors : 1];
  float* master[MASTER ? kTensors : 1];
  uint32_t block[BITS == 8 ? kTensors : 1];  // position of element 0, in blocks
  uint32_t first[kTensors];                  // chunk number of element 0
  int count;
  float lr, decay, b1, r1, b2, r2, eps;  // decay: lr weight_decay; r: 1 - b
  float c1, c2;                          // 1 - b^t
  uint32_t key;
  // read on the device where given: the learning rate, and the step count
  const float* lr_at;
  const int64_t* step_at;
  float weight_decay;
  double beta1, beta2;
  uint64_t seed;
};
static_assert(sizeof(AdamArgs<32, false>) <= 4096 && sizeof(AdamArgs<32, true>) <= 4096 &&
                  sizeof(AdamArgs<8, false>) <= 4096 && sizeof(AdamArgs<8, true>) <= 4096,
              "kernel arguments");

__host__ __device__ inline uint32_t dither_key(uint64_t seed, uint64_t step) {
  return (uint32_t)seed * 0x9e3779b1u + (uint32_t)step * 0x3c6ef373u;
}

constexpr uint32_t kDitherStep = 0x9e3779b1u;
constexpr uint32_t kNan = 0x7fc00000u;

// 32 random bits of one element: multiplications by odd constants (from the
// golden ratio and the roots of 2, 3, 5 and 7) between shifts that bring the
// high bits down.
__device__ __forceinline__ uint32_t dither_bits(uint32_t x) {
  x ^= x >> 16;
  x *= 0x6a09e667u;
  x ^= x >> 15;
  x *= 0xbb67ae85u;
  return x ^ (x >> 16);
}

template <bool SIGNED> struct Code {
  static constexpr int top = SIGNED ? 14 : 30;     // exponent field of the largest
  static constexpr int lowest = SIGNED ? 32 : 48;  // E below this count as it
};

// The exponent that moves codes to values (and, negated, back): E - top.
template <bool SIGNED>
__device__ __forceinline__ int code_shift(int e) {
  return min(max(e, Code<SIGNED>::lowest), 254) - Code<SIGNED>::top;
}

// Byte k of a word of four codes; nan: a NaN's bits where the block stands for
// NaN, else 0.  The low codes are subnormal as fp32 patterns, and exact.
template <bool SIGNED>
__device__ __forceinline__ float decode(uint32_t word, int k, int shift, uint32_t nan) {
  const uint32_t code = word >> (8 * k);
  const float x =
      __builtin_amdgcn_ldexpf(__uint_as_float((code & (SIGNED ? 127u : 255u)) << 20 | nan), shift);
  return SIGNED ? __uint_as_float(__float_as_uint(x) | (code & 128u) << 24) : x;
}
// The code of x in the top byte.
template <bool SIGNED>
__device__ __forceinline__ uint32_t encode(float x, int shift, uint32_t dither20) {
  const float u = __builtin_amdgcn_ldexpf(fabsf(x), -shift);
  const uint32_t q = (__float_as_uint(u) + dither20) << 4;
  if constexpr (SIGNED) return (q & 0x7fffffffu) | (__float_as_uint(x) & 0x80000000u);
  else return max(q, min(__float_as_uint(x), 1u) << 24);
}

// sqrt by the hardware's instruction (1 ulp), whose operand must not be
// subnormal: small ones are moved by an even power of two.
__device__ __forceinline__ float root_of(float v) {
  const bool small = v < 0x1p-96f;
  const float r = __builtin_amdgcn_sqrtf(small ? v * 0x1p64f : v);
  return small ? r * 0x1p-32f : r;
}

// Largest over the 32 lanes of a half wave, in each of them.
template <int CTRL>
__device__ __forceinline__ uint32_t max_move(uint32_t v) {
  return max(v, lane_move<CTRL>(v));
}
__device__ __forceinline__ uint32_t half_max(uint32_t v) {
  v = max_move<kXor1>(v);
  v = max_move<kXor2>(v);
  v = max_move<kHalfMirror>(v);
  v = max_move<kMirror>(v);
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max(r[0], r[1]);
}

// Eight elements at i of n, the ones past the end as zero, and back.
template <typename T, bool FULL>
__device__ __forceinline__ void load8(const void* p, int64_t i, int64_t n, float (&f)[8]) {
  const auto* s = static_cast<const typename T::storage*>(p) + i;
  constexpr int v = kVec<T>;
  if (FULL || i + 8 <= n) {
#pragma unroll
    for (int c = 0; c < 8 / v; ++c) {
      float part[v];
      unpack<T>(load_any<Chunk<T>>(s + c * v), part);
#pragma unroll
      for (int e = 0; e < v; ++e) f[c * v + e] = part[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = i + e < n ? to_float<T>(s[e]) : 0.0f;
  }
}
template <typename T, bool FULL>
__device__ __forceinline__ void store8(void* p, int64_t i, int64_t n, const float (&f)[8]) {
  auto* s = static_cast<typename T::storage*>(p) + i;
  constexpr int v = kVec<T>;
  if (FULL || i + 8 <= n) {
#pragma unroll
    for (int c = 0; c < 8 / v; ++c) {
      float part[v];
#pragma unroll
      for (int e = 0; e < v; ++e) part[e] = f[c * v + e];
      store_any(s + c * v, pack<T>(part));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < n) s[e] = from_float<T>(f[e]);
  }
}
template <bool FULL>
__device__ __forceinline__ uint2 load_codes(const void* p, int64_t i, int64_t n) {
  const uint8_t* s = static_cast<const uint8_t*>(p) + i;
  uint2 c = make_uint2(0, 0);
  if (FULL || i + 8 <= n) {
    __builtin_memcpy(&c, s, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < n) (e < 4 ? c.x : c.y) |= (uint32_t)s[e] << (8 * (e & 3));
  }
  return c;
}
template <bool FULL>
__device__ __forceinline__ void store_codes(void* p, int64_t i, int64_t n, uint2 c) {
  uint8_t* s = static_cast<uint8_t*>(p) + i;
  if (FULL || i + 8 <= n) {
    __builtin_memcpy(s, &c, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < n) s[e] = (uint8_t)((e < 4 ? c.x : c.y) >> (8 * (e & 3)));
  }
}

// The top bytes of eight words, in order.
__device__ __forceinline__ uint2 top_bytes(const uint32_t (&q)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // v_perm_b32 takes bytes 0-3 from its second operand, 4-7 from its first
    const uint32_t lo = __builtin_amdgcn_perm(q[4 * i + 1], q[4 * i], 0x0c0c0703u);
    const uint32_t hi = __builtin_amdgcn_perm(q[4 * i + 3], q[4 * i + 2], 0x07030c0cu);
    w[i] = lo | hi;
  }
  return make_uint2(w[0], w[1]);
}

struct AdamStep {
  float decay, size, root;  // lr weight_decay, lr / c1, 1 / sqrt(c2)
  uint32_t key;
};

// Tensor k's elements from base on.  The quotient is a product with the
// hardware's reciprocal (1 ulp): the update is off by a few 1e-7 of itself,
// and exact roots and quotients made the step bound by arithmetic (bf16 with
// 8-bit states, 66 M parameters: 190 us against 155).
template <typename P, typename Gr, int BITS, bool MASTER, bool FULL>
__device__ __forceinline__ void adam_chunk(const AdamArgs<BITS, MASTER>& a, int k,
                                           const AdamStep& h, int64_t base) {
#pragma clang fp contract(off)
  const int64_t n = a.n[k];
  const int64_t i = base + threadIdx.x * kLaneElems;
  float p[8], g[8], m[8], v[8];
  load8<Gr, FULL>(a.g[k], i, n, g);
  if constexpr (MASTER) load8<F32, FULL>(a.master[k], i, n, p);
  else load8<P, FULL>(a.p[k], i, n, p);
  if constexpr (BITS == 8) {
    const uint2 mc = load_codes<FULL>(a.m[k], i, n), vc = load_codes<FULL>(a.v[k], i, n);
    uint16_t s = 0;
    if (FULL || i < n) __builtin_memcpy(&s, a.scales[k] + 2 * (i / kBlock), 2);
    const int em = s & 255, ev = s >> 8;
    const uint32_t nm = em == 255 ? kNan : 0, nv = ev == 255 ? kNan : 0;
    const int fm = code_shift<true>(em), fv = code_shift<false>(ev);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      m[e] = decode<true>(e < 4 ? mc.x : mc.y, e & 3, fm, nm);
      v[e] = decode<false>(e < 4 ? vc.x : vc.y, e & 3, fv, nv);
    }
  } else {
    load8<F32, FULL>(a.m[k], i, n, m);
    load8<F32, FULL>(a.v[k], i, n, v);
  }
  uint32_t big_m = 0, big_v = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    // unfused, each product rounded: what the 8-bit codes are taken from must
    // not depend on how a compiler contracts
    m[e] = m[e] * a.b1 + g[e] * a.r1;
    v[e] = v[e] * a.b2 + (g[e] * g[e]) * a.r2;
    const float d = __builtin_fmaf(root_of(v[e]), h.root, a.eps);
    // All that leaves p in one number, then one subtraction and its rounding:
    // p (1 - lr decay) first would round twice at p's spacing, and 1 - lr decay
    // itself to steps of 2^-24 (lr decay = 5e-8 decayed 1.6 times as much, 2e-8
    // not at all).  The clamp keeps an infinite p from becoming inf - inf.  The
    // subtraction stays one of its own: fused with a product it is rounded to
    // 16 bits in one step, and a parameter is no longer its master's rounding.
    const float finite = __builtin_amdgcn_fmed3f(p[e], -__FLT_MAX__, __FLT_MAX__);
    p[e] -= __builtin_fmaf(h.decay, finite, h.size * (m[e] * __builtin_amdgcn_rcpf(d)));
    big_m = max(big_m, __float_as_uint(m[e]) & 0x7fffffffu);
    big_v = max(big_v, __float_as_uint(v[e]) & 0x7fffffffu);
  }
  store8<P, FULL>(a.p[k], i, n, p);
  if constexpr (MASTER) store8<F32, FULL>(a.master[k], i, n, p);
  if constexpr (BITS == 8) {
    const int em = max((int)(half_max(big_m) >> 23), Code<true>::lowest);
    const int ev = max((int)(half_max(big_v) >> 23), Code<false>::lowest);
    const int fm = code_shift<true>(em), fv = code_shift<false>(ev);
    const uint64_t at = (uint64_t)a.block[k] * kBlock + (uint64_t)i;
    const uint32_t x0 = (uint32_t)at * kDitherStep + (uint32_t)(at >> 32) * 0xa54ff53bu + h.key;
    uint32_t qm[8], qv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // positions of a lane's eight elements differ in the low word alone
      const uint32_t r = dither_bits(x0 + (uint32_t)e * kDitherStep);
      qm[e] = encode<true>(m[e], fm, (r & 0xffffu) * 16 + 8);
      qv[e] = encode<false>(v[e], fv, (r >> 16) * 16 + 8);
    }
    const uint2 none = make_uint2(0, 0);
    store_codes<FULL>(a.m[k], i, n, em == 255 ? none : top_bytes(qm));
    store_codes<FULL>(a.v[k], i, n, ev == 255 ? none : top_bytes(qv));
    if ((threadIdx.x & 31) == 0 && (FULL || i < n)) {
      const uint16_t s = (uint16_t)(em | ev << 8);
      __builtin_memcpy(a.scales[k] + 2 * (i / kBlock), &s, 2);
    }
  } else {
    store8<F32, FULL>(a.m[k], i, n, m);
    store8<F32, FULL>(a.v[k], i, n, v);
  }
}

template <typename P, typename Gr, int BITS, bool MASTER>
__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(AdamArgs<BITS, MASTER> a) {
  // the last tensor that starts at or before this chunk: one load per wave
  // instead of a chain of them
  const uint32_t chunk = blockIdx.x;
  const int lane = threadIdx.x & 63;
  int k = -1;
#pragma unroll
  for (int i = 0; i < AdamArgs<BITS, MASTER>::kTensors; i += 64)
    k += __popcll(__ballot(i + lane < a.count && a.first[min(i + lane, a.count - 1)] <= chunk));
  float lr = a.lr, decay = a.decay, c1 = a.c1, c2 = a.c2;
  uint32_t key = a.key;
  if (a.lr_at) lr = *a.lr_at, decay = lr * a.weight_decay;
  if (a.step_at) {
    __shared__ float c[2];
    const int64_t step = *a.step_at;
    if (threadIdx.x < 2)
      c[threadIdx.x] = (float)(1.0 - pow(threadIdx.x ? a.beta2 : a.beta1, (double)step));
    __syncthreads();
    c1 = c[0], c2 = c[1];
    key = dither_key(a.seed, (uint64_t)step);
  }
  const AdamStep h{decay, lr / c1, 1.0f / sqrtf(c2), key};
  const int64_t base = (int64_t)(chunk - a.first[k]) * kChunkElems;
  if (base + kChunkElems <= a.n[k]) adam_chunk<P, Gr, BITS, MASTER, true>(a, k, h, base);
  else adam_chunk<P, Gr, BITS, MASTER, false>(a, k, h, base);
}

// The values of 8-bit states in bf16, which holds their 4 significant bits.
__global__ __launch_bounds__(kAdamThreads) void adamw_values_kernel(
    const uint8_t* __restrict__ m, const uint8_t* __restrict__ v,
    const uint8_t* __restrict__ scales, int64_t n, uint16_t* __restrict__ out_m,
    uint16_t* __restrict__ out_v) {
  const int64_t i = ((int64_t)blockIdx.x * kAdamThreads + threadIdx.x) * kLaneElems;
  if (i >= n) return;
  uint16_t s;
  __builtin_memcpy(&s, scales + 2 * (i / kBlock), 2);
  const uint2 mc = load_codes<false>(m, i, n), vc = load_codes<false>(v, i, n);
  const int em = s & 255, ev = s >> 8;
  const uint32_t nm = em == 255 ? kNan : 0, nv = ev == 255 ? kNan : 0;
  const int fm = code_shift<true>(em), fv = code_shift<false>(ev);
  float x[8], y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = decode<true>(e < 4 ? mc.x : mc.y, e & 3, fm, nm);
    y[e] = decode<false>(e < 4 ? vc.x : vc.y, e & 3, fv, nv);
  }
  store8<BF16, false>(out_m, i, n, x);
  store8<BF16, false>(out_v, i, n, y);
}

}  // namespace maxsim

using namespace maxsim;

extern "C" {

int maxsim_amd_adamw_step(maxsim_dtype param_dtype, maxsim_dtype grad_dtype, int state_bits,
                          const maxsim_adamw_tensor* tensors, int64_t count, double lr,
                          const float* lr_on_device, double beta1, double beta2, double eps,
                          double weight_decay, int64_t step, const int64_t* step_on_device,
                          uint64_t seed, void* stream) {
  clear_error();
  if (int e = check_dtype(param_dtype)) return e;
  if (int e = check_dtype(grad_dtype)) return e;
  if (grad_dtype != param_dtype && grad_dtype != MAXSIM_FLOAT32)
    return fail(MAXSIM_ERR_INVALID, "grad_dtype must be param_dtype or float32");
  if (state_bits != 8 && state_bits != 32)
    return fail(MAXSIM_ERR_INVALID, "state_bits must be 8 or 32; got %d", state_bits);
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0))
    return fail(MAXSIM_ERR_INVALID, "betas must be in [0, 1)");
  if (!(eps >= 0.0) || !(weight_decay >= 0.0) || !(lr_on_device || lr >= 0.0))
    return fail(MAXSIM_ERR_INVALID, "lr, eps and weight_decay must be >= 0");
  if (!step_on_device && step < 1) return fail(MAXSIM_ERR_INVALID, "step must be >= 1");
  if (count < 0 || (count > 0 && !tensors)) return fail(MAXSIM_ERR_INVALID, "no tensors");
  const bool master = count > 0 && tensors[0].master;
  for (int64_t i = 0; i < count; ++i) {
    const maxsim_adamw_tensor& t = tensors[i];
    if (t.numel < 0) return fail(MAXSIM_ERR_INVALID, "negative size");
    if (!t.master == master)
      return fail(MAXSIM_ERR_INVALID, "either every tensor has a master or none");
    if (t.numel > 0 &&
        (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (state_bits == 8 && !t.scales)))
      return fail(MAXSIM_ERR_INVALID, "null pointer argument");
    if ((t.numel + kChunkElems - 1) / kChunkElems > kMaxChunks)
      return fail(MAXSIM_ERR_UNSUPPORTED, "tensor too large for one launch");
    if (state_bits == 8 && (t.position % kBlock != 0 || t.position >= (uint64_t)kMaxElems))
      return fail(MAXSIM_ERR_INVALID, "position must be a multiple of 256 below 2^40");
  }
  if (master && param_dtype == MAXSIM_FLOAT32)
    return fail(MAXSIM_ERR_INVALID, "float32 parameters have no master");

  auto run = [&](auto p, auto g, auto bits, auto with_master) -> int {
    constexpr int BITS = decltype(bits)::value;
    constexpr bool MASTER = decltype(with_master)::value;
    using Args = AdamArgs<BITS, MASTER>;
    Args a{};
    a.lr = (float)lr;
    a.decay = (float)(lr * weight_decay);
    a.weight_decay = (float)weight_decay;
    a.b1 = (float)beta1, a.r1 = (float)(1.0 - beta1);
    a.b2 = (float)beta2, a.r2 = (float)(1.0 - beta2);
    a.eps = (float)eps;
    a.c1 = (float)(1.0 - std::pow(beta1, (double)step));
    a.c2 = (float)(1.0 - std::pow(beta2, (double)step));
    a.key = dither_key(seed, (uint64_t)step);
    a.lr_at = lr_on_device, a.step_at = step_on_device;
    a.beta1 = beta1, a.beta2 = beta2, a.seed = seed;
    uint32_t chunks = 0;
    auto launch = [&] {
      hipLaunchKernelGGL((adamw_kernel<decltype(p), decltype(g), BITS, MASTER>), dim3(chunks),
                         dim3(kAdamThreads), BITS == 32 ? kReservedLds : 0,
                         static_cast<hipStream_t>(stream), a);
      a.count = 0, chunks = 0;
      return check_launch("adamw_kernel");
    };
    for (int64_t i = 0; i < count; ++i) {
      const maxsim_adamw_tensor& t = tensors[i];
      if (t.numel == 0) continue;
      const uint32_t more = (uint32_t)((t.numel + kChunkElems - 1) / kChunkElems);
      if (a.count == Args::kTensors || (uint64_t)chunks + more > kMaxChunks)
        if (int e = launch()) return e;
      const int k = a.count++;
      a.p[k] = t.param, a.g[k] = t.grad, a.m[k] = t.exp_avg, a.v[k] = t.exp_avg_sq;
      a.n[k] = t.numel, a.first[k] = chunks;
      if constexpr (BITS == 8) {
        a.scales[k] = t.scales;
        a.block[k] = (uint32_t)(t.position / kBlock);
      }
      if constexpr (MASTER) a.master[k] = t.master;
      chunks += more;
    }
    return a.count > 0 ? launch() : MAXSIM_OK;
  };
  auto with_bits = [&](auto p, auto g, auto with_master) {
    return state_bits == 8 ? run(p, g, std::integral_constant<int, 8>{}, with_master)
                           : run(p, g, std::integral_constant<int, 32>{}, with_master);
  };
  auto with_grad = [&](auto p, auto g) {
    return master ? with_bits(p, g, std::true_type{}) : with_bits(p, g, std::false_type{});
  };
  if (param_dtype == MAXSIM_FLOAT32) return with_bits(F32{}, F32{}, std::false_type{});
  if (param_dtype == MAXSIM_FLOAT16)
    return grad_dtype == MAXSIM_FLOAT32 ? with_grad(F16{}, F32{}) : with_grad(F16{}, F16{});
  return grad_dtype == MAXSIM_FLOAT32 ? with_grad(BF16{}, F32{}) : with_grad(BF16{}, BF16{});
}

int maxsim_amd_adamw_state_values(const uint8_t* exp_avg, const uint8_t* exp_avg_sq,
                                  const uint8_t* scales, int64_t numel, void* values,
                                  void* values_sq, void* stream) {
  clear_error();
  if (numel < 0) return fail(MAXSIM_ERR_INVALID, "negative size");
  if (numel == 0) return MAXSIM_OK;
  if (!exp_avg || !exp_avg_sq || !scales || !values || !values_sq)
    return fail(MAXSIM_ERR_INVALID, "null pointer argument");
  const int64_t blocks = (numel + kAdamThreads * kLaneElems - 1) / (kAdamThreads * kLaneElems);
  if (blocks > kMaxChunks)
    return fail(MAXSIM_ERR_UNSUPPORTED, "tensor too large for one launch");
  hipLaunchKernelGGL(adamw_values_kernel, dim3((unsigned)blocks), dim3(kAdamThreads), 0,
                     static_cast<hipStream_t>(stream), exp_avg, exp_avg_sq, scales, numel,
                     static_cast<uint16_t*>(values), static_cast<uint16_t*>(values_sq));
  return check_launch("adamw_values_kernel");
}

}  // extern "C"
