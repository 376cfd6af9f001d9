// The AdamW step over many tensors at once, with states in 32 or 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Memory-bound: 28 bytes per element in fp32, 10 in bf16 with 8-bit states.
// A launch takes up to kTensors tensors by their addresses in its arguments
// (nothing is copied to the device or kept there) and cuts each into chunks,
// one per workgroup; a workgroup finds its tensor by bisection of the chunk
// counts.
//
// 8-bit states.  A block of 256 elements of a tensor shares, per state, one
// byte: the exponent field E of its largest magnitude.  The code of an element
// is the top of the fp32 pattern of |value| moved down by a power of two that
// puts E at exponent field 14 (m: sign, 4 exponent and 3 mantissa bits) or 30
// (v: 5 and 3 bits, no sign), so that the block's small values reach into
// fp32's subnormal numbers, whose even spacing is the codes' own lowest step.
// The 20 bits below the cut decide the rounding, up or down in proportion, by
// adding 20 random bits: with b2 = 0.999 a second moment moves by a thousandth
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
constexpr int kLaneElems = 8;  // elements of a lane at a time: 32 lanes are a block
constexpr int kBlock = MAXSIM_AMD_STATE_BLOCK;
static_assert(kBlock == 32 * kLaneElems, "half a wave holds a block");
constexpr int kTurns = 2;  // blocks of a lane per workgroup
constexpr int kChunkElems = kAdamThreads * kLaneElems * kTurns;
constexpr int kTensors = 48;  // of one launch: 3.5 KB of its 4 KB of arguments

struct AdamTensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  uint8_t* scales;
  float* master;
  int64_t n;
  uint64_t position;  // of element 0, for the random bits
};

struct AdamArgs {
  AdamTensor t[kTensors];
  uint32_t first[kTensors + 1];  // chunk numbers
  int count;
  float lr, decay, b1, r1, b2, r2, eps;  // r: 1 - b
  float c1, c2;                          // 1 - b^t
  uint32_t key;
  // read on the device where given: the learning rate, and the step count
  const float* lr_at;
  const int64_t* step_at;
  double beta1, beta2;
  uint64_t seed;
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");

__host__ __device__ inline uint32_t dither_key(uint64_t seed, uint64_t step) {
  return (uint32_t)seed * 0x9e3779b1u + (uint32_t)step * 0x3c6ef373u;
}

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

__device__ __forceinline__ float pow2f(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

// Both directions go by two exact factors, of which 2^126 has no place in one
// (E - top spans more than fp32's exponents).
template <bool SIGNED>
__device__ __forceinline__ float decode_factor(int e) {
  return e == 255 ? NAN : pow2f(min(max(e, Code<SIGNED>::lowest), 254) - Code<SIGNED>::top - 126);
}
template <bool SIGNED>
__device__ __forceinline__ float decode(uint32_t code, float factor) {
  const float u = __uint_as_float((SIGNED ? code & 127u : code) << 20);
  const float x = u * 0x1p126f * factor;
  return SIGNED && (code & 128u) ? -x : x;
}
template <bool SIGNED>
__device__ __forceinline__ float encode_factor(int e) {
  return pow2f(Code<SIGNED>::top + 126 - min(max(e, Code<SIGNED>::lowest), 254));
}
template <bool SIGNED>
__device__ __forceinline__ uint32_t encode(float x, float factor, uint32_t dither20) {
  const float u = fabsf(x) * factor * 0x1p-126f;
  uint32_t q = (__float_as_uint(u) + dither20) >> 20;
  if constexpr (SIGNED) q |= (__float_as_uint(x) >> 31) << 7;
  else if (q == 0 && x > 0.0f) q = 1;
  return q;
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
      unpack16<T>(load16_any(s + c * v), part);
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
      store16_any(s + c * v, pack16<T>(part));
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

struct AdamStep {
  float keep, size, root;  // 1 - lr decay, lr / c1, sqrt(c2)
  uint32_t key;
};

// The states of each turn are loaded before any of them is used.
template <typename P, typename Gr, int BITS, bool MASTER, bool FULL>
__device__ __forceinline__ void adam_chunk(const AdamArgs& a, const AdamTensor& t,
                                           const AdamStep& h, int64_t base) {
#pragma clang fp contract(off)
  const int64_t n = t.n;
  float p[kTurns][8], g[kTurns][8], m[kTurns][8], v[kTurns][8];
  uint2 mc[kTurns], vc[kTurns];
  uint16_t sc[kTurns];
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int64_t i = base + (int64_t)(u * kAdamThreads + threadIdx.x) * kLaneElems;
    load8<Gr, FULL>(t.g, i, n, g[u]);
    if constexpr (MASTER) load8<F32, FULL>(t.master, i, n, p[u]);
    else load8<P, FULL>(t.p, i, n, p[u]);
    if constexpr (BITS == 8) {
      mc[u] = load_codes<FULL>(t.m, i, n);
      vc[u] = load_codes<FULL>(t.v, i, n);
      sc[u] = 0;
      if (FULL || i < n) __builtin_memcpy(&sc[u], t.scales + 2 * (i / kBlock), 2);
    } else {
      load8<F32, FULL>(t.m, i, n, m[u]);
      load8<F32, FULL>(t.v, i, n, v[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int64_t i = base + (int64_t)(u * kAdamThreads + threadIdx.x) * kLaneElems;
    if constexpr (BITS == 8) {
      const float fm = decode_factor<true>(sc[u] & 255), fv = decode_factor<false>(sc[u] >> 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m[u][e] = decode<true>((e < 4 ? mc[u].x : mc[u].y) >> (8 * (e & 3)) & 255u, fm);
        v[u][e] = decode<false>((e < 4 ? vc[u].x : vc[u].y) >> (8 * (e & 3)) & 255u, fv);
      }
    }
    uint32_t big_m = 0, big_v = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float ge = g[u][e];
      // unfused, each product rounded: what the 8-bit codes are taken from
      // must not depend on how a compiler contracts
      m[u][e] = m[u][e] * a.b1 + ge * a.r1;
      v[u][e] = v[u][e] * a.b2 + (ge * ge) * a.r2;
      const float d = sqrtf(v[u][e]) / h.root + a.eps;
      p[u][e] = p[u][e] * h.keep - h.size * (m[u][e] / d);
      big_m = max(big_m, __float_as_uint(m[u][e]) & 0x7fffffffu);
      big_v = max(big_v, __float_as_uint(v[u][e]) & 0x7fffffffu);
    }
    store8<P, FULL>(t.p, i, n, p[u]);
    if constexpr (MASTER) store8<F32, FULL>(t.master, i, n, p[u]);
    if constexpr (BITS == 8) {
      const int em = max((int)(half_max(big_m) >> 23), Code<true>::lowest);
      const int ev = max((int)(half_max(big_v) >> 23), Code<false>::lowest);
      const float fm = encode_factor<true>(em), fv = encode_factor<false>(ev);
      const uint64_t at = t.position + (uint64_t)i;
      const uint32_t x0 =
          (uint32_t)at * 0x9e3779b1u + (uint32_t)(at >> 32) * 0xa54ff53bu + h.key;
      uint2 qm = make_uint2(0, 0), qv = make_uint2(0, 0);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // positions of a lane's eight elements differ in the low word alone
        const uint32_t r = dither_bits(x0 + (uint32_t)e * 0x9e3779b1u);
        const uint32_t cm =
            em == 255 ? 0 : encode<true>(m[u][e], fm, (r & 0xffffu) * 16 + 8);
        const uint32_t cv = ev == 255 ? 0 : encode<false>(v[u][e], fv, (r >> 16) * 16 + 8);
        (e < 4 ? qm.x : qm.y) |= cm << (8 * (e & 3));
        (e < 4 ? qv.x : qv.y) |= cv << (8 * (e & 3));
      }
      store_codes<FULL>(t.m, i, n, qm);
      store_codes<FULL>(t.v, i, n, qv);
      if ((threadIdx.x & 31) == 0 && (FULL || i < n)) {
        const uint16_t s = (uint16_t)(em | ev << 8);
        __builtin_memcpy(t.scales + 2 * (i / kBlock), &s, 2);
      }
    } else {
      store8<F32, FULL>(t.m, i, n, m[u]);
      store8<F32, FULL>(t.v, i, n, v[u]);
    }
  }
}

template <typename P, typename Gr, int BITS, bool MASTER>
__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(AdamArgs a) {
  const uint32_t chunk = blockIdx.x;
  int lo = 0, hi = a.count;  // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  const AdamTensor& t = a.t[lo];
  float lr = a.lr, c1 = a.c1, c2 = a.c2;
  uint32_t key = a.key;
  if (a.lr_at) lr = *a.lr_at;
  if (a.step_at) {
    __shared__ float c[2];
    const int64_t step = *a.step_at;
    if (threadIdx.x < 2)
      c[threadIdx.x] = (float)(1.0 - pow(threadIdx.x ? a.beta2 : a.beta1, (double)step));
    __syncthreads();
    c1 = c[0], c2 = c[1];
    key = dither_key(a.seed, (uint64_t)step);
  }
  const AdamStep h{1.0f - lr * a.decay, lr / c1, sqrtf(c2), key};
  const int64_t base = (int64_t)(chunk - a.first[lo]) * kChunkElems;
  if (base + kChunkElems <= t.n) adam_chunk<P, Gr, BITS, MASTER, true>(a, t, h, base);
  else adam_chunk<P, Gr, BITS, MASTER, false>(a, t, h, base);
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
  const float fm = decode_factor<true>(s & 255), fv = decode_factor<false>(s >> 8);
  float x[8], y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = decode<true>((e < 4 ? mc.x : mc.y) >> (8 * (e & 3)) & 255u, fm);
    y[e] = decode<false>((e < 4 ? vc.x : vc.y) >> (8 * (e & 3)) & 255u, fv);
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
    if (t.numel / kChunkElems >= UINT32_MAX / (2 * kAdamThreads))
      return fail(MAXSIM_ERR_UNSUPPORTED, "tensor too large for one launch");
  }
  if (master && param_dtype == MAXSIM_FLOAT32)
    return fail(MAXSIM_ERR_INVALID, "float32 parameters have no master");

  AdamArgs a{};
  a.lr = (float)lr;
  a.decay = (float)weight_decay;
  a.b1 = (float)beta1, a.r1 = (float)(1.0 - beta1);
  a.b2 = (float)beta2, a.r2 = (float)(1.0 - beta2);
  a.eps = (float)eps;
  a.c1 = (float)(1.0 - std::pow(beta1, (double)step));
  a.c2 = (float)(1.0 - std::pow(beta2, (double)step));
  a.key = dither_key(seed, (uint64_t)step);
  a.lr_at = lr_on_device, a.step_at = step_on_device;
  a.beta1 = beta1, a.beta2 = beta2, a.seed = seed;
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto launch = [&] {
    const unsigned blocks = a.first[a.count];
    auto go = [&](auto p, auto g, auto bits, auto mst) {
      hipLaunchKernelGGL(
          (adamw_kernel<decltype(p), decltype(g), decltype(bits)::value, decltype(mst)::value>),
          dim3(blocks), dim3(kAdamThreads), 0, st, a);
    };
    auto bits = [&](auto p, auto g, auto mst) {
      if (state_bits == 8) go(p, g, std::integral_constant<int, 8>{}, mst);
      else go(p, g, std::integral_constant<int, 32>{}, mst);
    };
    auto sixteen = [&](auto p) {
      auto grad = [&](auto g) {
        if (master) bits(p, g, std::true_type{});
        else bits(p, g, std::false_type{});
      };
      if (grad_dtype == MAXSIM_FLOAT32) grad(F32{});
      else grad(p);
    };
    if (param_dtype == MAXSIM_FLOAT32) bits(F32{}, F32{}, std::false_type{});
    else if (param_dtype == MAXSIM_FLOAT16) sixteen(F16{});
    else sixteen(BF16{});
    a.count = 0;
    return check_launch("adamw_kernel");
  };
  for (int64_t i = 0; i < count; ++i) {
    const maxsim_adamw_tensor& t = tensors[i];
    if (t.numel == 0) continue;
    const uint32_t chunks = (uint32_t)((t.numel + kChunkElems - 1) / kChunkElems);
    if (a.count == kTensors ||
        (a.count > 0 && (uint64_t)a.first[a.count] + chunks > UINT32_MAX / kAdamThreads))
      if (int e = launch()) return e;
    a.t[a.count] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.scales, t.master, t.numel,
                    t.position};
    a.first[a.count + 1] = a.first[a.count] + chunks;
    ++a.count;
  }
  return a.count > 0 ? launch() : MAXSIM_OK;
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
  if (blocks > UINT32_MAX / kAdamThreads)
    return fail(MAXSIM_ERR_UNSUPPORTED, "tensor too large for one launch");
  hipLaunchKernelGGL(adamw_values_kernel, dim3((unsigned)blocks), dim3(kAdamThreads), 0,
                     static_cast<hipStream_t>(stream), exp_avg, exp_avg_sq, scales, numel,
                     static_cast<uint16_t*>(values), static_cast<uint16_t*>(values_sq));
  return check_launch("adamw_values_kernel");
}

}  // extern "C"
