// Torch binding of the operators around the scoring kernels (token embeddings,
// layer norm, unit rows, the gradients' norm, AdamW) over the C ABI of
// include/maxsim_amd_training.h and include/maxsim_amd_encoder.h.
//
// The differentiable ones are C++ autograd functions: their backward runs on
// the engine's thread without the interpreter, and both directions go through
// the dispatcher, so that torch.compile records the operators themselves.
// Argument errors are raised here with Python's types (one pass over an
// optimizer's tensors instead of one per check).
#include <ATen/core/CachingHostAllocator.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/library.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <map>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/maxsim_amd_encoder.h"
#include "torch_common.h"

namespace {

using at::Tensor;
using std::optional;
using namespace maxsim_torch;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

maxsim_dtype dtype_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return MAXSIM_FLOAT32;
    case at::kHalf: return MAXSIM_FLOAT16;
    case at::kBFloat16: return MAXSIM_BFLOAT16;
    default: break;
  }
  TORCH_CHECK_TYPE(false, name, " must be float32, float16, or bfloat16; got ", t.scalar_type());
  return MAXSIM_FLOAT32;
}

void check_same_device(const Tensor& t, const char* name, const Tensor& x, const char* first) {
  TORCH_CHECK(t.device() == x.device(), "all tensors must be on the same device; ", first,
              " is on ", x.device(), " but ", name, " is on ", t.device());
}

void check_hip(const Tensor& t, const char* name) {
  TORCH_CHECK(t.device().is_cuda(), name, " must be a HIP (torch 'cuda') tensor");
}

// Memory on t's device, without the dispatcher (0.5 us of a call's 5).
Tensor empty_like_on(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
  return Tensor(at::detail::empty_cuda(sizes, type, t.device(), std::nullopt));
}
Tensor empty_like_on(const Tensor& t, at::IntArrayRef sizes) {
  return empty_like_on(t, sizes, t.scalar_type());
}

// The rows of a tensor [..., dim] as the kernels address them: `outer` groups
// of `inner` rows.  A view where two strides are enough, else a copy.
struct Rows {
  Tensor t;
  int64_t outer = 1, inner = 1, outer_stride = 0, inner_stride = 0;
};

// Whether dims [lo, hi) of t are one dimension with one stride, which is
// then `stride` (0 where there is at most one row).
bool one_stride(const Tensor& t, int64_t lo, int64_t hi, int64_t& rows, int64_t& stride) {
  rows = 1, stride = 0;
  int64_t next = -1;  // what the next outer dimension's stride has to be
  for (int64_t i = hi - 1; i >= lo; --i) {
    if (t.size(i) != 1) {
      if (next < 0) stride = t.stride(i);
      else if (t.stride(i) != next) return false;
      next = t.stride(i) * t.size(i);
    }
    rows *= t.size(i);
  }
  return true;
}

// split: dims before it are `outer`, those from it on (but the last) `inner`.
Rows rows_of(const Tensor& t, int64_t split) {
  Rows r;
  const int64_t last = t.dim() - 1;
  r.t = t;
  const bool in_place =
      (t.size(last) <= 1 || t.stride(last) == 1) &&
      one_stride(t, 0, split, r.outer, r.outer_stride) &&
      one_stride(t, split, last, r.inner, r.inner_stride);
  if (!in_place) {
    r.t = t.contiguous();
    one_stride(r.t, 0, split, r.outer, r.outer_stride);
    one_stride(r.t, split, last, r.inner, r.inner_stride);
  }
  return r;
}

// ---- layer norm --------------------------------------------------------------

struct Norm {
  Rows x;
  Tensor weight, bias;  // undefined: none
  maxsim_dtype dtype, weight_dtype;
  int64_t dim;
};

Tensor norm_param(const optional<Tensor>& p, const char* name, const Tensor& x) {
  if (!p.has_value() || !p->defined()) return Tensor();
  dtype_of(*p, name);
  TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == x.size(-1), name, " must have shape [dim=",
                    x.size(-1), "]; got ", p->sizes());
  TORCH_CHECK_TYPE(p->scalar_type() == x.scalar_type() || p->scalar_type() == at::kFloat, name,
                   " must be float32 or have x's dtype; got ", p->scalar_type());
  check_same_device(*p, name, x, "x");
  return p->contiguous();
}

void check_norm_x(const Tensor& x, double eps) {
  dtype_of(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must have at least 1 dimension");
  TORCH_CHECK_VALUE(x.size(-1) > 0, "dim must be > 0; got ", x.size(-1));
  TORCH_CHECK_VALUE(eps >= 0.0 && eps < 1e30, "eps must be finite and >= 0; got ", eps);
  check_hip(x, "x");
}

Norm prep_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias,
               double eps) {
  check_norm_x(x, eps);
  Norm n;
  n.dtype = dtype_of(x, "x");
  n.weight = norm_param(weight, "weight", x);
  n.bias = norm_param(bias, "bias", x);
  if (n.weight.defined() && n.bias.defined())
    TORCH_CHECK_TYPE(n.weight.scalar_type() == n.bias.scalar_type(),
                     "weight and bias must have the same dtype; got ", n.weight.scalar_type(),
                     " and ", n.bias.scalar_type());
  n.weight_dtype = n.weight.defined() ? dtype_of(n.weight, "weight")
                   : n.bias.defined() ? dtype_of(n.bias, "bias")
                                      : n.dtype;
  n.x = rows_of(x, 0);
  n.dim = x.size(-1);
  return n;
}

const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor run_norm(const Norm& n, double eps, float* mean, float* rstd) {
  Tensor y = empty_like_on(n.x.t, n.x.t.sizes());
  c10::hip::HIPGuardMasqueradingAsCUDA guard(n.x.t.device());
  check_status(maxsim_amd_layer_norm_forward(
      n.dtype, n.weight_dtype, n.x.t.data_ptr(), n.x.inner, n.dim, n.x.inner_stride,
      ptr(n.weight), ptr(n.bias), (float)eps, y.data_ptr(), mean, rstd, current_stream(n.x.t)));
  return y;
}

Tensor maxsim_layer_norm(const Tensor& x, const optional<Tensor>& weight,
                         const optional<Tensor>& bias, double eps) {
  return run_norm(prep_norm(x, weight, bias, eps), eps, nullptr, nullptr);
}

// With what the backward needs: the rows' means, then 1 / sqrt(variance + eps).
std::tuple<Tensor, Tensor> maxsim_layer_norm_forward(const Tensor& x,
                                                     const optional<Tensor>& weight,
                                                     const optional<Tensor>& bias, double eps) {
  const Norm n = prep_norm(x, weight, bias, eps);
  Tensor stats = empty_like_on(x, {2, n.x.inner}, at::kFloat);
  float* s = stats.data_ptr<float>();
  return {run_norm(n, eps, s, s + n.x.inner), stats};
}

// Gradients that are not asked for come back empty.
std::tuple<Tensor, Tensor, Tensor> maxsim_layer_norm_backward(
    const Tensor& dy, const Tensor& x, const Tensor& stats, const optional<Tensor>& weight,
    bool want_dx, bool want_dweight, bool want_dbias, at::ScalarType weight_dtype) {
  check_norm_x(x, 0.0);
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(),
              "dy must have x's shape and dtype");
  check_same_device(dy, "dy", x, "x");
  const Rows xr = rows_of(x, 0), gr = rows_of(dy, 0);
  const int64_t rows = xr.inner, dim = x.size(-1);
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.numel() == 2 * rows &&
                  stats.is_contiguous(),
              "stats must be float32 [2, rows]");
  check_same_device(stats, "stats", x, "x");
  const Tensor w = norm_param(weight, "weight", x);
  const maxsim_dtype dt = dtype_of(x, "x");
  Tensor dx = want_dx ? empty_like_on(x, x.sizes()) : empty_like_on(x, {0});
  Tensor dw = empty_like_on(x, {want_dweight ? dim : 0}, weight_dtype);
  Tensor db = empty_like_on(x, {want_dbias ? dim : 0}, weight_dtype);
  TORCH_CHECK(!w.defined() || w.scalar_type() == weight_dtype, "weight_dtype must be weight's");
  const maxsim_dtype wdt = dtype_of(dw, "weight");
  const bool sums = want_dweight || want_dbias;
  const size_t bytes = sums ? maxsim_amd_layer_norm_backward_workspace_size(dt, rows, dim) : 0;
  Tensor ws;
  if (bytes > 0) ws = empty_like_on(x, {(int64_t)(bytes / sizeof(float))}, at::kFloat);
  const float* s = stats.data_ptr<float>();
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  check_status(maxsim_amd_layer_norm_backward(
      dt, wdt, gr.t.data_ptr(), gr.inner_stride, xr.t.data_ptr(), xr.inner_stride, s, s + rows,
      ptr(w), rows, dim, want_dx ? dx.data_ptr() : nullptr, want_dweight ? dw.data_ptr() : nullptr,
      want_dbias ? db.data_ptr() : nullptr, bytes > 0 ? ws.data_ptr() : nullptr, bytes,
      current_stream(x)));
  return {dx, dw, db};
}

// ---- unit rows ---------------------------------------------------------------

void check_lengths(const Tensor& lengths) {
  TORCH_CHECK_TYPE(lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong,
                   "lengths must be int32 or int64; got ", lengths.scalar_type());
}

void check_unit(const Tensor& x, const optional<Tensor>& lengths, double eps) {
  dtype_of(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && (!lengths.has_value() || x.dim() == 3),
                    lengths.has_value() ? "x must be 3-D [N, L, D] where lengths are given; got "
                                        : "x must have at least 1 dimension; got ",
                    x.sizes());
  TORCH_CHECK_VALUE(x.size(-1) > 0, "dim must be > 0; got ", x.size(-1));
  TORCH_CHECK_VALUE((float)eps >= FLT_MIN && eps < 1e30, "eps must be finite and at least 2^-126, "
                    "the smallest normal float32; got ", eps);
  check_hip(x, "x");
  if (!lengths.has_value()) return;
  check_lengths(*lengths);
  TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == x.size(0),
                    "lengths must have shape [N=", x.size(0), "]; got ", lengths->sizes());
  check_same_device(*lengths, "lengths", x, "x");
}

// Contiguous lengths (or nothing) and how wide they are; the kernels cut them
// to [0, L] themselves.
struct Lengths {
  Tensor t;
  const void* data = nullptr;
  int is64 = 0;
};
Lengths lengths_of(const optional<Tensor>& lengths) {
  Lengths l;
  if (!lengths.has_value()) return l;
  l.t = lengths->contiguous();
  l.is64 = l.t.scalar_type() == at::kLong;
  l.data = l.t.data_ptr();
  return l;
}

const int32_t* i32(const Tensor& t) { return t.defined() ? t.data_ptr<int32_t>() : nullptr; }

// x as sequences x length x dim: with lengths they are given, without them
// rows are told apart by two strides at most.  More rows than a sequence can
// have are as many sequences of one.
Rows unit_rows(const Tensor& x, const Lengths& lengths) {
  Rows r = rows_of(x, x.dim() >= 3 ? x.dim() - 2 : 0);
  if (r.inner > INT32_MAX && !lengths.data) r = rows_of(x, x.dim() - 1);
  return r;
}

Tensor unit_forward(const Tensor& x, const Lengths& lengths, const Tensor& offsets,
                    int64_t packed_rows, double eps) {
  const Rows r = unit_rows(x, lengths);
  Tensor y = offsets.defined() ? empty_like_on(x, {packed_rows, x.size(-1)})
                               : empty_like_on(x, x.sizes());
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  check_status(maxsim_amd_unit_rows_forward(
      dtype_of(x, "x"), r.t.data_ptr(), r.outer, r.inner, x.size(-1), r.outer_stride,
      r.inner_stride, lengths.data, lengths.is64, i32(offsets), packed_rows, (float)eps,
      y.data_ptr(),
      current_stream(x)));
  return y;
}

Tensor unit_backward(const Tensor& dy, const Tensor& x, const Lengths& lengths,
                     const Tensor& offsets, int64_t packed_rows, double eps) {
  TORCH_CHECK(dy.scalar_type() == x.scalar_type(), "dy must have x's dtype");
  check_same_device(dy, "dy", x, "x");
  const Rows r = unit_rows(x, lengths);
  Rows g;
  if (offsets.defined()) {
    g.t = dy.contiguous();
  } else {
    g = unit_rows(dy, lengths);
  }
  Tensor dx = empty_like_on(x, x.sizes());
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  check_status(maxsim_amd_unit_rows_backward(
      dtype_of(x, "x"), g.t.data_ptr(), g.outer_stride, g.inner_stride, r.t.data_ptr(), r.outer,
      r.inner, x.size(-1), r.outer_stride, r.inner_stride, lengths.data, lengths.is64,
      i32(offsets), packed_rows, (float)eps, dx.data_ptr(), current_stream(x)));
  return dx;
}

Tensor maxsim_normalize_embeddings(const Tensor& x, const optional<Tensor>& lengths, double eps) {
  check_unit(x, lengths, eps);
  return unit_forward(x, lengths_of(lengths), Tensor(), 0, eps);
}

Tensor maxsim_normalize_embeddings_backward(const Tensor& dy, const Tensor& x,
                                            const optional<Tensor>& lengths, double eps) {
  check_unit(x, lengths, eps);
  TORCH_CHECK(dy.sizes() == x.sizes(), "dy must have x's shape");
  return unit_backward(dy, x, lengths_of(lengths), Tensor(), 0, eps);
}

// Lengths cut to [0, max_len], the offsets of the packed sequences [N + 1] and
// their rows in all, which the host waits for: in a word of pinned memory that
// the kernel writes, which comes sooner than a copy and a synchronization.
std::tuple<Tensor, Tensor, int64_t> maxsim_length_offsets(const Tensor& lengths,
                                                          int64_t max_len) {
  check_hip(lengths, "lengths");
  check_lengths(lengths);
  TORCH_CHECK_VALUE(lengths.dim() == 1, "lengths must be 1-D; got ", lengths.sizes());
  const Lengths l = lengths_of(lengths);
  const int64_t n = l.t.numel();
  Tensor clamped = empty_like_on(l.t, {n}, at::kInt);
  Tensor offsets = empty_like_on(l.t, {n + 1}, at::kInt);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(l.t.device());
  const auto s = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(l.t.device().index());
  TORCH_CHECK(!capturing(s.stream()),
              "maxsim_amd: packing waits for the lengths and cannot run while the stream is "
              "captured");
  at::DataPtr pinned = at::getHostAllocator(at::kCUDA)->allocate(sizeof(uint64_t));
  uint64_t* word = static_cast<uint64_t*>(pinned.get());
  *word = 0;
  check_status(maxsim_amd_length_offsets(l.data, l.is64, n, max_len, clamped.data_ptr<int32_t>(),
                                         offsets.data_ptr<int32_t>(), word, s.stream()));
  int64_t total = 0;
  try {
    total = wait_for_word(reinterpret_cast<int64_t*>(word), s.stream(), "the offsets") >> 1;
  } catch (...) {
    // the kernel may still write the word
    at::getHostAllocator(at::kCUDA)->record_event(word, pinned.get_context(), s.unwrap());
    throw;
  }
  return {clamped, offsets, total};
}

void check_packed(const Tensor& x, const Tensor& lengths, const Tensor& offsets,
                  int64_t packed_rows, double eps) {
  check_unit(x, lengths, eps);
  TORCH_CHECK(lengths.scalar_type() == at::kInt && offsets.scalar_type() == at::kInt &&
                  lengths.is_contiguous() && offsets.is_contiguous() &&
                  offsets.dim() == 1 && offsets.size(0) == x.size(0) + 1,
              "lengths [N] and offsets [N + 1] must be int32");
  TORCH_CHECK(packed_rows >= 0, "packed_rows must be >= 0");
  check_same_device(offsets, "offsets", x, "x");
}

Tensor maxsim_pack_normalized(const Tensor& x, const Tensor& lengths, const Tensor& offsets,
                              int64_t packed_rows, double eps) {
  check_packed(x, lengths, offsets, packed_rows, eps);
  return unit_forward(x, lengths_of(lengths), offsets, packed_rows, eps);
}

Tensor maxsim_pack_normalized_backward(const Tensor& dy, const Tensor& x, const Tensor& lengths,
                                       const Tensor& offsets, double eps) {
  check_packed(x, lengths, offsets, 0, eps);
  TORCH_CHECK(dy.dim() == 2 && dy.size(1) == x.size(2), "dy must be [rows, dim]");
  return unit_backward(dy, x, lengths_of(lengths), offsets, dy.size(0), eps);
}

// ---- token embeddings ----------------------------------------------------------

struct Embed {
  Tensor weight, ids;
  Lengths lengths;
  int64_t vocab, dim, stride, sequences, length;
  maxsim_dtype weight_dtype, dtype;
  at::ScalarType type;
  std::vector<int64_t> sizes;  // of the result
};

Embed prep_embed(const Tensor& weight, const Tensor& ids, const optional<Tensor>& lengths,
                 double scale, int64_t padding_idx, optional<at::ScalarType> dtype) {
  Embed e;
  e.weight_dtype = dtype_of(weight, "weight");
  TORCH_CHECK_VALUE(weight.dim() == 2, "weight must be 2-D [vocab, dim]; got ", weight.sizes());
  e.vocab = weight.size(0), e.dim = weight.size(1);
  TORCH_CHECK_VALUE(e.dim > 0, "dim must be > 0; got ", e.dim);
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong,
                   "ids must be int32 or int64; got ", ids.scalar_type());
  e.type = dtype.value_or(weight.scalar_type());
  TORCH_CHECK_TYPE(e.type == weight.scalar_type() ||
                       (weight.scalar_type() == at::kFloat &&
                        (e.type == at::kHalf || e.type == at::kBFloat16)),
                   "dtype must be weight's, or float16 or bfloat16 of a float32 weight; got ",
                   e.type, " of ", weight.scalar_type());
  e.dtype = e.type == at::kFloat ? MAXSIM_FLOAT32 : e.type == at::kHalf ? MAXSIM_FLOAT16
                                                                        : MAXSIM_BFLOAT16;
  TORCH_CHECK_VALUE(std::isfinite((float)scale), "scale must be finite; got ", scale);
  TORCH_CHECK_VALUE(padding_idx >= -1 && padding_idx < std::max<int64_t>(e.vocab, 1),
                    "padding_idx must be a row of weight; got ", padding_idx);
  check_hip(weight, "weight");
  check_same_device(ids, "ids", weight, "weight");
  if (lengths.has_value()) {
    TORCH_CHECK_VALUE(ids.dim() == 2, "ids must be 2-D [N, L] where lengths are given; got ",
                      ids.sizes());
    check_lengths(*lengths);
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == ids.size(0),
                      "lengths must have shape [N=", ids.size(0), "]; got ", lengths->sizes());
    check_same_device(*lengths, "lengths", weight, "weight");
    e.sequences = ids.size(0), e.length = ids.size(1);
  } else {
    e.sequences = ids.numel(), e.length = 1;
  }
  // rows may lie anywhere, their elements side by side
  e.weight = e.dim > 1 && weight.stride(1) != 1 ? weight.contiguous() : weight;
  e.stride = e.weight.stride(0);
  e.ids = ids.contiguous();
  e.lengths = lengths_of(lengths);
  e.sizes = ids.sizes().vec();
  e.sizes.push_back(e.dim);
  return e;
}

Tensor run_embed(const Embed& e, double scale, int64_t padding_idx, int32_t* rows) {
  Tensor y = empty_like_on(e.weight, e.sizes, e.type);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(e.weight.device());
  check_status(maxsim_amd_embed_forward(
      e.weight_dtype, e.dtype, e.weight.data_ptr(), e.vocab, e.dim, e.stride, e.ids.data_ptr(),
      e.ids.scalar_type() == at::kLong, e.sequences, e.length, e.lengths.data, e.lengths.is64,
      (float)scale, padding_idx, y.data_ptr(), rows, current_stream(e.weight)));
  return y;
}

// padding_idx: -1 for none.
Tensor maxsim_embed_tokens(const Tensor& weight, const Tensor& ids,
                           const optional<Tensor>& lengths, double scale, int64_t padding_idx,
                           optional<at::ScalarType> dtype) {
  return run_embed(prep_embed(weight, ids, lengths, scale, padding_idx, dtype), scale, padding_idx,
                   nullptr);
}

// With what the backward needs: each token's row of weight, -1 where it has none.
std::tuple<Tensor, Tensor> maxsim_embed_tokens_forward(const Tensor& weight, const Tensor& ids,
                                                       const optional<Tensor>& lengths,
                                                       double scale, int64_t padding_idx,
                                                       optional<at::ScalarType> dtype) {
  const Embed e = prep_embed(weight, ids, lengths, scale, padding_idx, dtype);
  Tensor rows = empty_like_on(weight, {e.ids.numel()}, at::kInt);
  return {run_embed(e, scale, padding_idx, rows.data_ptr<int32_t>()), rows};
}

Tensor maxsim_embed_tokens_backward(const Tensor& dy, const Tensor& rows, int64_t vocab,
                                    double scale, at::ScalarType weight_dtype) {
  const maxsim_dtype dt = dtype_of(dy, "dy");
  check_hip(dy, "dy");
  TORCH_CHECK_VALUE(dy.dim() >= 1 && dy.size(-1) > 0 && vocab >= 0,
                    "dy must be [..., dim] and vocab >= 0; got ", dy.sizes(), " and ", vocab);
  const int64_t dim = dy.size(-1);
  TORCH_CHECK(rows.scalar_type() == at::kInt && rows.is_contiguous() &&
                  rows.numel() * dim == dy.numel(),
              "rows must be contiguous int32, one for each row of dy");
  check_same_device(rows, "rows", dy, "dy");
  TORCH_CHECK_TYPE(weight_dtype == dy.scalar_type() || weight_dtype == at::kFloat,
                   "weight_dtype must be dy's or float32; got ", weight_dtype);
  const int64_t tokens = rows.numel();
  const Rows r = rows_of(dy, 0);
  Tensor dw = empty_like_on(dy, {vocab, dim}, weight_dtype);
  const size_t bytes = maxsim_amd_embed_backward_workspace_size(dt, tokens, vocab, dim);
  Tensor ws = empty_like_on(dy, {(int64_t)bytes}, at::kByte);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dy.device());
  check_status(maxsim_amd_embed_backward(dtype_of(dw, "weight"), dt, r.t.data_ptr(),
                                         r.inner_stride, rows.data_ptr<int32_t>(), tokens, vocab,
                                         dim, (float)scale, dw.data_ptr(), ws.data_ptr(), bytes,
                                         current_stream(dy)));
  return dw;
}

// ---- autograd ----------------------------------------------------------------

// An operator of this library through the dispatcher, looked up once.
#define MAXSIM_CALL(name, ...)                                          \
  ([&] {                                                                \
    static const auto op = c10::Dispatcher::singleton()                 \
                               .findSchemaOrThrow("maxsim_amd::" #name, "") \
                               .typed<decltype(name)>();                \
    return op.call(__VA_ARGS__);                                        \
  }())

bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const optional<Tensor>& t) { return t.has_value() && t->requires_grad(); }

// No function here carries forward-mode tangents, and one that is dropped on
// the way would count as 0.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
// Without a level there are none to look for (an encoder's 197 gradients: 2 us of
// the call's 27).
bool tangents_count() {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
         torch::autograd::ForwardADLevel::try_get_by_idx(0);
}
void refuse_tangents(const char* name, const Tensor& a, const optional<Tensor>& b = std::nullopt,
                     const optional<Tensor>& c = std::nullopt) {
  if (!tangents_count()) return;
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(a) && !(b.has_value() && has_tangent(*b)) &&
                                  !(c.has_value() && has_tangent(*c)),
                              "maxsim_amd: ", name, " has no derivative in forward mode");
}
void refuse_tangents(const char* name, at::TensorList tensors) {
  if (!tangents_count()) return;
  TORCH_CHECK_NOT_IMPLEMENTED(std::none_of(tensors.begin(), tensors.end(), has_tangent),
                              "maxsim_amd: ", name, " has no derivative in forward mode");
}

// A backward's results where its caller records a graph through it
// (create_graph): they hang on what they came from, and a second derivative
// raises instead of counting as 0.
struct OnlyOnce : torch::autograd::Function<OnlyOnce> {
  static variable_list forward(AutogradContext*, const Tensor&, const Tensor&,
                               const optional<Tensor>&, variable_list results) {
    return results;
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "maxsim_amd: the gradient of this function has no derivative of its own");
  }
};

// count: results and the arguments of the forward that have no gradient.
variable_list backward_results(variable_list results, size_t count, const Tensor& dy,
                               const Tensor& x, const optional<Tensor>& weight) {
  if (at::GradMode::is_enabled()) {
    variable_list defined;
    for (const Tensor& t : results)
      if (t.defined()) defined.push_back(t);
    defined = OnlyOnce::apply(dy, x, weight, std::move(defined));
    size_t next = 0;
    for (Tensor& t : results)
      if (t.defined()) t = defined[next++];
  }
  results.resize(count);
  return results;
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& weight,
                        const optional<Tensor>& bias, double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [y, stats] = MAXSIM_CALL(maxsim_layer_norm_forward, x, weight, bias, eps);
    const bool has_w = weight.has_value(), has_b = bias.has_value();
    ctx->save_for_backward({x, has_w ? *weight : Tensor(), stats});
    ctx->saved_data["has_w"] = has_w;
    ctx->saved_data["has_b"] = has_b;
    ctx->saved_data["dtype"] =
        (int64_t)(has_w ? *weight : has_b ? *bias : x).scalar_type();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool has_w = ctx->saved_data["has_w"].toBool(), has_b = ctx->saved_data["has_b"].toBool();
    // edges in the order of the tensors that are there
    const bool want_x = ctx->needs_input_grad(0);
    const bool want_w = has_w && ctx->needs_input_grad(1);
    const bool want_b = has_b && ctx->needs_input_grad(1 + has_w);
    const optional<Tensor> weight = has_w ? optional<Tensor>(saved[1]) : std::nullopt;
    const auto run = [&] {
      at::AutoDispatchBelowADInplaceOrView guard;
      return MAXSIM_CALL(maxsim_layer_norm_backward, grads[0], saved[0], saved[2], weight, want_x,
                         want_w, want_b, (at::ScalarType)ctx->saved_data["dtype"].toInt());
    };
    auto [dx, dw, db] = run();
    return backward_results({want_x ? dx : Tensor(), want_w ? dw : Tensor(), want_b ? db : Tensor()},
                            4, grads[0], saved[0], weight);
  }
};

Tensor layer_norm_autograd(const Tensor& x, const optional<Tensor>& weight,
                           const optional<Tensor>& bias, double eps) {
  refuse_tangents("layer_norm", x, weight, bias);
  if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias)))
    return LayerNormFn::apply(x, weight, bias, eps);
  at::AutoDispatchBelowADInplaceOrView guard;
  return MAXSIM_CALL(maxsim_layer_norm, x, weight, bias, eps);
}

struct NormalizeFn : torch::autograd::Function<NormalizeFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& lengths,
                        double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({x, lengths.has_value() ? *lengths : Tensor()});
    ctx->saved_data["eps"] = eps;
    return MAXSIM_CALL(maxsim_normalize_embeddings, x, lengths, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const optional<Tensor> lengths =
        saved[1].defined() ? optional<Tensor>(saved[1]) : std::nullopt;
    const auto run = [&] {
      at::AutoDispatchBelowADInplaceOrView guard;
      return MAXSIM_CALL(maxsim_normalize_embeddings_backward, grads[0], saved[0], lengths,
                         ctx->saved_data["eps"].toDouble());
    };
    return backward_results({run()}, 3, grads[0], saved[0], std::nullopt);
  }
};

Tensor normalize_autograd(const Tensor& x, const optional<Tensor>& lengths, double eps) {
  refuse_tangents("normalize_embeddings", x);
  if (at::GradMode::is_enabled() && wants(x)) return NormalizeFn::apply(x, lengths, eps);
  at::AutoDispatchBelowADInplaceOrView guard;
  return MAXSIM_CALL(maxsim_normalize_embeddings, x, lengths, eps);
}

struct PackNormalizedFn : torch::autograd::Function<PackNormalizedFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& lengths,
                        const Tensor& offsets, int64_t packed_rows, double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({x, lengths, offsets});
    ctx->saved_data["eps"] = eps;
    return MAXSIM_CALL(maxsim_pack_normalized, x, lengths, offsets, packed_rows, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto run = [&] {
      at::AutoDispatchBelowADInplaceOrView guard;
      return MAXSIM_CALL(maxsim_pack_normalized_backward, grads[0], saved[0], saved[1], saved[2],
                         ctx->saved_data["eps"].toDouble());
    };
    return backward_results({run()}, 5, grads[0], saved[0], std::nullopt);
  }
};

Tensor pack_normalized_autograd(const Tensor& x, const Tensor& lengths, const Tensor& offsets,
                                int64_t packed_rows, double eps) {
  refuse_tangents("pack_normalized_documents", x);
  if (at::GradMode::is_enabled() && wants(x))
    return PackNormalizedFn::apply(x, lengths, offsets, packed_rows, eps);
  at::AutoDispatchBelowADInplaceOrView guard;
  return MAXSIM_CALL(maxsim_pack_normalized, x, lengths, offsets, packed_rows, eps);
}

struct EmbedFn : torch::autograd::Function<EmbedFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids,
                        const optional<Tensor>& lengths, double scale, int64_t padding_idx,
                        optional<at::ScalarType> dtype) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [y, rows] =
        MAXSIM_CALL(maxsim_embed_tokens_forward, weight, ids, lengths, scale, padding_idx, dtype);
    ctx->save_for_backward({rows});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["dtype"] = (int64_t)weight.scalar_type();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto run = [&] {
      at::AutoDispatchBelowADInplaceOrView guard;
      return MAXSIM_CALL(maxsim_embed_tokens_backward, grads[0], saved[0],
                         ctx->saved_data["vocab"].toInt(), ctx->saved_data["scale"].toDouble(),
                         (at::ScalarType)ctx->saved_data["dtype"].toInt());
    };
    return backward_results({run()}, 6, grads[0], saved[0], std::nullopt);
  }
};

Tensor embed_autograd(const Tensor& weight, const Tensor& ids, const optional<Tensor>& lengths,
                      double scale, int64_t padding_idx, optional<at::ScalarType> dtype) {
  refuse_tangents("embed_tokens", weight);
  if (at::GradMode::is_enabled() && wants(weight))
    return EmbedFn::apply(weight, ids, lengths, scale, padding_idx, dtype);
  at::AutoDispatchBelowADInplaceOrView guard;
  return MAXSIM_CALL(maxsim_embed_tokens, weight, ids, lengths, scale, padding_idx, dtype);
}

// ---- AdamW -------------------------------------------------------------------

// The two tensors have their elements in the same order in memory.
bool same_order(const Tensor& a, const Tensor& b) {
  if (a.sizes() != b.sizes()) return false;
  if (a.is_contiguous() && b.is_contiguous()) return true;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}

void check_partner(const Tensor& t, const char* name, const Tensor& p, at::ScalarType type,
                   int64_t i) {
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, "[", i, "] must be ", type, "; got ",
                   t.scalar_type());
  TORCH_CHECK(t.device() == p.device(), "all tensors must be on the same device; params[", i,
              "] is on ", p.device(), " but ", name, "[", i, "] is on ", t.device());
  TORCH_CHECK_VALUE(same_order(t, p), name, "[", i, "] must have the shape and strides of params[",
                    i, "]");
}

// What is written in place: autograd's check of saved tensors goes by this.
void touched(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

const Tensor* device_scalar(const optional<Tensor>& t, const char* name, at::ScalarType type,
                            const Tensor& p) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK_TYPE(t->scalar_type() == type, name, " must be ", type, " as a tensor; got ",
                   t->scalar_type());
  TORCH_CHECK_VALUE(t->numel() == 1, name, " must hold one value; got ", t->sizes());
  TORCH_CHECK(t->device() == p.device(), "all tensors must be on the same device; params[0] is on ",
              p.device(), " but ", name, " is on ", t->device());
  return &*t;
}

// Where a tensor of a step's lists lies; of a gradient, which is only read,
// or of one that is updated.
struct Place {
  uintptr_t begin, end;
  uint32_t list, index;
  bool operator<(const Place& o) const { return begin < o.begin; }
};
constexpr const char* kLists[] = {"params", "grads", "exp_avgs", "exp_avg_sqs", "scales", "masters"};
constexpr uint32_t kGradList = 1;

// Nothing that is updated shares memory with anything else: workgroups of one
// launch would write over each other.  Lists mostly lie in memory as they were
// allocated, one tensor after the other, so that each is merged as it is.
void check_places(std::vector<Place> (&lists)[6]) {
  std::vector<Place> all;
  size_t count = 0;
  for (const std::vector<Place>& list : lists) count += list.size();
  all.reserve(count);
  for (std::vector<Place>& list : lists) {
    if (!std::is_sorted(list.begin(), list.end())) std::sort(list.begin(), list.end());
    const auto before = (ptrdiff_t)all.size();
    all.insert(all.end(), list.begin(), list.end());
    std::inplace_merge(all.begin(), all.begin() + before, all.end());
  }
  const Place none{};
  const Place *written = &none, *read = &none;  // those that reach farthest
  for (const Place& p : all) {
    const bool reads = p.list == kGradList;
    const Place* met = p.begin < written->end          ? written
                       : !reads && p.begin < read->end ? read
                                                       : nullptr;
    TORCH_CHECK_VALUE(!met, kLists[met->list], "[", met->index, "] and ", kLists[p.list], "[",
                      p.index, "] share memory");
    if (!reads) written = &p;
    else if (p.end > read->end) read = &p;
  }
}

void maxsim_adamw_step(at::TensorList params, at::TensorList grads, at::TensorList exp_avgs,
                       at::TensorList exp_avg_sqs, at::TensorList scales, at::TensorList masters,
                       double lr, const optional<Tensor>& lr_tensor, double beta1, double beta2,
                       double eps, double weight_decay, int64_t step,
                       const optional<Tensor>& step_tensor, int64_t seed,
                       const optional<Tensor>& grad_scale) {
  const size_t n = params.size();
  TORCH_CHECK_VALUE(grads.size() == n && exp_avgs.size() == n && exp_avg_sqs.size() == n &&
                        (scales.empty() || scales.size() == n) &&
                        (masters.empty() || masters.size() == n),
                    "adamw_step needs lists of one length; got ", n, " params, ", grads.size(),
                    " grads, ", exp_avgs.size(), " exp_avgs, ", exp_avg_sqs.size(),
                    " exp_avg_sqs, ", scales.size(), " scales, ", masters.size(), " masters");
  TORCH_CHECK_VALUE(lr_tensor.has_value() || (lr >= 0.0 && lr < 1e30),
                    "lr must be finite and >= 0; got ", lr);
  TORCH_CHECK_VALUE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0,
                    "betas must be in [0, 1); got ", beta1, " and ", beta2);
  TORCH_CHECK_VALUE(eps >= 0.0 && eps < 1e30, "eps must be finite and >= 0; got ", eps);
  TORCH_CHECK_VALUE(weight_decay >= 0.0 && weight_decay < 1e30,
                    "weight_decay must be finite and >= 0; got ", weight_decay);
  TORCH_CHECK_VALUE(step_tensor.has_value() || step >= 1, "step must be >= 1; got ", step);
  if (n == 0) return;
  const Tensor* lr_at = device_scalar(lr_tensor, "lr", at::kFloat, params[0]);
  const Tensor* step_at = device_scalar(step_tensor, "step", at::kLong, params[0]);
  const Tensor* scale_at = device_scalar(grad_scale, "grad_scale", at::kFloat, params[0]);
  const bool eight = !scales.empty();
  const at::ScalarType state = eight ? at::kByte : at::kFloat;

  at::AutoDispatchBelowADInplaceOrView below;  // a gradient's copy records nothing
  // tensors of one (parameter, gradient) type go together
  using Types = std::pair<maxsim_dtype, maxsim_dtype>;
  std::map<Types, std::vector<maxsim_adamw_tensor>> groups;
  Types of{};  // of the tensor before, whose group is `group`
  std::vector<maxsim_adamw_tensor>* group = nullptr;
  std::vector<Tensor> copies;  // gradients in their parameters' order
  std::vector<Place> places[6];
  for (auto& list : places) list.reserve(n);
  const auto place = [&](uint32_t list, const void* at, int64_t bytes, size_t i) {
    const auto begin = reinterpret_cast<uintptr_t>(at);
    places[list].push_back({begin, begin + (uintptr_t)bytes, list, (uint32_t)i});
  };
  uint64_t position = 0;
  for (size_t i = 0; i < n; ++i) {
    const Tensor& p = params[i];
    const maxsim_dtype dt = dtype_of(p, "params");
    TORCH_CHECK(p.device() == params[0].device(),
                "all tensors must be on the same device; params[0] is on ", params[0].device(),
                " but params[", i, "] is on ", p.device());
    check_hip(p, "params");
    TORCH_CHECK_VALUE(p.is_non_overlapping_and_dense(), "params[", i,
                      "] must cover its memory without gaps or overlaps");
    Tensor g = grads[i];
    TORCH_CHECK_TYPE(g.layout() == at::kStrided, "grads[", i, "] must be dense");
    TORCH_CHECK_TYPE(g.scalar_type() == p.scalar_type() || g.scalar_type() == at::kFloat, "grads[",
                     i, "] must be float32 or have its parameter's dtype; got ", g.scalar_type());
    TORCH_CHECK(g.device() == p.device(), "all tensors must be on the same device; params[", i,
                "] is on ", p.device(), " but grads[", i, "] is on ", g.device());
    TORCH_CHECK_VALUE(g.sizes() == p.sizes(), "grads[", i, "] must have shape ", p.sizes(),
                      "; got ", g.sizes());
    if (!same_order(g, p)) {
      copies.push_back(at::empty_strided(p.sizes(), p.strides(), g.options()));
      copies.back().copy_(g);
      g = copies.back();
    }
    check_partner(exp_avgs[i], "exp_avgs", p, state, (int64_t)i);
    check_partner(exp_avg_sqs[i], "exp_avg_sqs", p, state, (int64_t)i);
    const int64_t numel = p.numel();
    const int64_t blocks = (numel + MAXSIM_AMD_STATE_BLOCK - 1) / MAXSIM_AMD_STATE_BLOCK;
    if (eight) {
      const Tensor& s = scales[i];
      TORCH_CHECK_TYPE(s.scalar_type() == at::kByte, "scales[", i, "] must be uint8; got ",
                       s.scalar_type());
      TORCH_CHECK(s.device() == p.device(), "all tensors must be on the same device; params[", i,
                  "] is on ", p.device(), " but scales[", i, "] is on ", s.device());
      TORCH_CHECK_VALUE(s.dim() == 2 && s.size(0) == blocks && s.size(1) == 2 && s.is_contiguous(),
                        "scales[", i, "] must be contiguous [", blocks, ", 2]; got ", s.sizes());
    }
    if (!masters.empty()) {
      TORCH_CHECK_TYPE(dt != MAXSIM_FLOAT32, "params[", i, "] is float32 and takes no master");
      check_partner(masters[i], "masters", p, at::kFloat, (int64_t)i);
    }
    const maxsim_adamw_tensor t{p.data_ptr(), g.data_ptr(), exp_avgs[i].data_ptr(),
                                exp_avg_sqs[i].data_ptr(),
                                eight ? scales[i].data_ptr<uint8_t>() : nullptr,
                                masters.empty() ? nullptr : masters[i].data_ptr<float>(), numel,
                                position};
    const Types types{dt, dtype_of(g, "grads")};
    if (!group || types != of) {
      of = types;
      group = &groups[types];
      group->reserve(n);
    }
    group->push_back(t);
    position += (uint64_t)blocks * MAXSIM_AMD_STATE_BLOCK;
    if (numel == 0) continue;
    const int64_t held = numel * (int64_t)p.element_size(), f32 = 4 * numel;
    place(0, t.param, held, i);
    place(2, t.exp_avg, eight ? numel : f32, i);
    place(3, t.exp_avg_sq, eight ? numel : f32, i);
    if (eight) place(4, t.scales, 2 * blocks, i);
    if (t.master) place(5, t.master, f32, i);
    // a thread has read its elements before it writes them: a gradient may be
    // a tensor of its own type that its parameter's step updates
    const bool wide = g.scalar_type() == at::kFloat, alike = g.scalar_type() == p.scalar_type();
    const bool own = (alike && t.grad == t.param) ||
                     (wide && t.grad == t.master) ||
                     (wide && !eight && (t.grad == t.exp_avg || t.grad == t.exp_avg_sq));
    if (!own) place(kGradList, t.grad, alike ? held : f32, i);
  }
  check_places(places);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(params[0].device());
  for (const auto& [types, tensors] : groups)
    check_status(maxsim_amd_adamw_step_scaled(
        types.first, types.second, eight ? 8 : 32, tensors.data(), (int64_t)tensors.size(),
        scale_at ? scale_at->data_ptr<float>() : nullptr, lr,
        lr_at ? lr_at->data_ptr<float>() : nullptr, beta1, beta2, eps, weight_decay, step,
        step_at ? step_at->data_ptr<int64_t>() : nullptr, (uint64_t)seed,
        current_stream(params[0])));
  for (const at::TensorList& l : {params, exp_avgs, exp_avg_sqs, scales, masters})
    for (const Tensor& t : l) touched(t);
}

// ---- the gradients' norm -------------------------------------------------------

struct Grads {
  std::vector<maxsim_grad_tensor> list;
  std::vector<Tensor> copies;
};

// in_place: the tensors themselves are written, so that each covers its memory
// and shares it with no other.
Grads prep_grads(at::TensorList grads, bool in_place) {
  Grads g;
  g.list.reserve(grads.size());
  std::vector<Place> places;
  if (in_place) places.reserve(grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor& t = grads[i];
    TORCH_CHECK_TYPE(t.layout() == at::kStrided, "grads[", i, "] must be dense");
    const maxsim_dtype dt = dtype_of(t, "grads");
    TORCH_CHECK(t.device() == grads[0].device(),
                "all tensors must be on the same device; grads[0] is on ", grads[0].device(),
                " but grads[", i, "] is on ", t.device());
    check_hip(t, "grads");
    const bool dense = t.is_non_overlapping_and_dense();
    TORCH_CHECK_VALUE(dense || !in_place, "grads[", i,
                      "] must cover its memory without gaps or overlaps");
    if (!dense) g.copies.push_back(t.contiguous());
    const Tensor& from = dense ? t : g.copies.back();
    const int64_t numel = from.numel();
    g.list.push_back({from.data_ptr(), numel, dt});
    if (in_place && numel > 0) {
      const auto begin = reinterpret_cast<uintptr_t>(from.data_ptr());
      places.push_back({begin, begin + (uintptr_t)numel * from.element_size(), 0, (uint32_t)i});
    }
  }
  if (!std::is_sorted(places.begin(), places.end())) std::sort(places.begin(), places.end());
  for (size_t i = 1; i < places.size(); ++i)
    TORCH_CHECK_VALUE(places[i - 1].end <= places[i].begin, "grads[", places[i - 1].index,
                      "] and grads[", places[i].index, "] share memory");
  return g;
}

void check_clip(double max_norm, double eps) {
  TORCH_CHECK_VALUE(max_norm >= 0.0, "max_norm must be >= 0; got ", max_norm);
  TORCH_CHECK_VALUE(eps >= 0.0 && eps < 1e30, "eps must be finite and >= 0; got ", eps);
}

// Norm and factor of what prep_grads gave; clip: which is then clipped.
std::tuple<Tensor, Tensor> run_grad_norm(const Grads& g, const Tensor& like, double max_norm,
                                         double eps, bool clip) {
  Tensor norm = empty_like_on(like, {}, at::kFloat), factor = empty_like_on(like, {}, at::kFloat);
  const int64_t count = (int64_t)g.list.size();
  const size_t bytes = maxsim_amd_grad_norm_workspace_size(g.list.data(), count);
  Tensor ws = empty_like_on(like, {(int64_t)bytes}, at::kByte);
  check_status((clip ? maxsim_amd_clip_grads : maxsim_amd_grad_norm)(
      g.list.data(), count, max_norm, eps, norm.data_ptr<float>(), factor.data_ptr<float>(),
      ws.data_ptr(), bytes, current_stream(like)));
  return {norm, factor};
}

std::tuple<Tensor, Tensor> maxsim_clip_factor(at::TensorList grads, double max_norm, double eps) {
  check_clip(max_norm, eps);
  TORCH_CHECK_VALUE(!grads.empty(), "needs at least one gradient");
  at::AutoDispatchBelowADInplaceOrView below;  // a gradient's copy records nothing
  const Grads g = prep_grads(grads, false);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(grads[0].device());
  return run_grad_norm(g, grads[0], max_norm, eps, false);
}

Tensor maxsim_clip_grad_norm(at::TensorList grads, double max_norm, double eps) {
  check_clip(max_norm, eps);
  TORCH_CHECK_VALUE(!grads.empty(), "needs at least one gradient");
  at::AutoDispatchBelowADInplaceOrView below;
  const Grads g = prep_grads(grads, true);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(grads[0].device());
  const Tensor norm = std::get<0>(run_grad_norm(g, grads[0], max_norm, eps, true));
  for (const Tensor& t : grads) touched(t);
  return norm;
}

// The norm, the factor and clipping record nothing in reverse mode: they are
// for gradients, which seldom have any of their own.
std::tuple<Tensor, Tensor> clip_factor_autograd(at::TensorList grads, double max_norm, double eps) {
  refuse_tangents("clip_factor", grads);
  at::AutoDispatchBelowADInplaceOrView guard;
  return MAXSIM_CALL(maxsim_clip_factor, grads, max_norm, eps);
}

Tensor clip_grad_norm_autograd(at::TensorList grads, double max_norm, double eps) {
  refuse_tangents("clip_grad_norm", grads);
  // as torch's operators in place: what stands there is a parameter, where
  // torch.nn.utils' function would have taken one for its gradient
  if (at::GradMode::is_enabled())
    for (size_t i = 0; i < grads.size(); ++i)
      TORCH_CHECK(!grads[i].requires_grad() || !grads[i].is_leaf(), "grads[", i,
                  "] is a leaf that requires grad: clip_grad_norm takes the gradients, not the "
                  "parameters (under torch.no_grad() any tensor)");
  at::AutoDispatchBelowADInplaceOrView guard;
  return MAXSIM_CALL(maxsim_clip_grad_norm, grads, max_norm, eps);
}

// The values of 8-bit states, in bf16 (which holds them exactly).
std::tuple<Tensor, Tensor> maxsim_adamw_state_values(const Tensor& exp_avg,
                                                     const Tensor& exp_avg_sq,
                                                     const Tensor& scales) {
  check_hip(exp_avg, "exp_avg");
  for (const Tensor* t : {&exp_avg, &exp_avg_sq, &scales}) {
    TORCH_CHECK_TYPE(t->scalar_type() == at::kByte, "8-bit states must be uint8; got ",
                     t->scalar_type());
    check_same_device(*t, "a state", exp_avg, "exp_avg");
  }
  TORCH_CHECK_VALUE(exp_avg.is_non_overlapping_and_dense() && same_order(exp_avg_sq, exp_avg),
                    "exp_avg and exp_avg_sq must have the same shape and strides");
  const int64_t n = exp_avg.numel();
  const int64_t blocks = (n + MAXSIM_AMD_STATE_BLOCK - 1) / MAXSIM_AMD_STATE_BLOCK;
  TORCH_CHECK_VALUE(scales.dim() == 2 && scales.size(0) == blocks && scales.size(1) == 2 &&
                        scales.is_contiguous(),
                    "scales must be contiguous [", blocks, ", 2]; got ", scales.sizes());
  const auto opts = exp_avg.options().dtype(at::kBFloat16);
  Tensor m = at::empty_strided(exp_avg.sizes(), exp_avg.strides(), opts);
  Tensor v = at::empty_strided(exp_avg.sizes(), exp_avg.strides(), opts);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(exp_avg.device());
  check_status(maxsim_amd_adamw_state_values(
      exp_avg.data_ptr<uint8_t>(), exp_avg_sq.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), n,
      m.data_ptr(), v.data_ptr(), current_stream(exp_avg)));
  return {m, v};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(maxsim_amd, m) {
  // none of these is the reference's, whose training example leaves them to torch
  m.def("maxsim_layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("maxsim_layer_norm_forward(Tensor x, Tensor? weight, Tensor? bias, float eps) "
        "-> (Tensor, Tensor)");
  m.def("maxsim_layer_norm_backward(Tensor dy, Tensor x, Tensor stats, Tensor? weight, "
        "bool want_dx, bool want_dweight, bool want_dbias, ScalarType weight_dtype) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("maxsim_normalize_embeddings(Tensor x, Tensor? lengths, float eps) -> Tensor");
  m.def("maxsim_normalize_embeddings_backward(Tensor dy, Tensor x, Tensor? lengths, float eps) "
        "-> Tensor");
  m.def("maxsim_length_offsets(Tensor lengths, int max_len) -> (Tensor, Tensor, int)");
  m.def("maxsim_pack_normalized(Tensor x, Tensor lengths, Tensor offsets, int packed_rows, "
        "float eps) -> Tensor");
  m.def("maxsim_pack_normalized_backward(Tensor dy, Tensor x, Tensor lengths, Tensor offsets, "
        "float eps) -> Tensor");
  m.def("maxsim_adamw_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, "
        "Tensor(c!)[] exp_avg_sqs, Tensor(d!)[] scales, Tensor(e!)[] masters, float lr, "
        "Tensor? lr_tensor, float beta1, float beta2, float eps, float weight_decay, int step, "
        "Tensor? step_tensor, int seed, Tensor? grad_scale=None) -> ()");
  m.def("maxsim_embed_tokens(Tensor weight, Tensor ids, Tensor? lengths, float scale, "
        "int padding_idx, ScalarType? dtype) -> Tensor");
  m.def("maxsim_embed_tokens_forward(Tensor weight, Tensor ids, Tensor? lengths, float scale, "
        "int padding_idx, ScalarType? dtype) -> (Tensor, Tensor)");
  m.def("maxsim_embed_tokens_backward(Tensor dy, Tensor rows, int vocab, float scale, "
        "ScalarType weight_dtype) -> Tensor");
  m.def("maxsim_clip_factor(Tensor[] grads, float max_norm, float eps) -> (Tensor, Tensor)");
  m.def("maxsim_clip_grad_norm(Tensor(a!)[] grads, float max_norm, float eps) -> Tensor");
  m.def("maxsim_adamw_state_values(Tensor exp_avg, Tensor exp_avg_sq, Tensor scales) "
        "-> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(maxsim_amd, CUDA, m) {
  m.impl("maxsim_layer_norm", &maxsim_layer_norm);
  m.impl("maxsim_layer_norm_forward", &maxsim_layer_norm_forward);
  m.impl("maxsim_layer_norm_backward", &maxsim_layer_norm_backward);
  m.impl("maxsim_normalize_embeddings", &maxsim_normalize_embeddings);
  m.impl("maxsim_normalize_embeddings_backward", &maxsim_normalize_embeddings_backward);
  m.impl("maxsim_length_offsets", &maxsim_length_offsets);
  m.impl("maxsim_pack_normalized", &maxsim_pack_normalized);
  m.impl("maxsim_pack_normalized_backward", &maxsim_pack_normalized_backward);
  m.impl("maxsim_adamw_step", &maxsim_adamw_step);
  m.impl("maxsim_adamw_state_values", &maxsim_adamw_state_values);
  m.impl("maxsim_embed_tokens", &maxsim_embed_tokens);
  m.impl("maxsim_embed_tokens_forward", &maxsim_embed_tokens_forward);
  m.impl("maxsim_embed_tokens_backward", &maxsim_embed_tokens_backward);
  m.impl("maxsim_clip_factor", &maxsim_clip_factor);
  m.impl("maxsim_clip_grad_norm", &maxsim_clip_grad_norm);
}

// a sparse gradient comes here to be refused by name
TORCH_LIBRARY_IMPL(maxsim_amd, SparseCUDA, m) {
  m.impl("maxsim_adamw_step", &maxsim_adamw_step);
  m.impl("maxsim_clip_factor", &maxsim_clip_factor);
  m.impl("maxsim_clip_grad_norm", &maxsim_clip_grad_norm);
}

TORCH_LIBRARY_IMPL(maxsim_amd, AutogradCUDA, m) {
  m.impl("maxsim_layer_norm", &layer_norm_autograd);
  m.impl("maxsim_normalize_embeddings", &normalize_autograd);
  m.impl("maxsim_pack_normalized", &pack_normalized_autograd);
  m.impl("maxsim_embed_tokens", &embed_autograd);
  m.impl("maxsim_clip_factor", &clip_factor_autograd);
  m.impl("maxsim_clip_grad_norm", &clip_grad_norm_autograd);
  // nothing to record, and its hundreds of tensors need not be looked at for it
  m.impl("maxsim_adamw_step", torch::CppFunction::makeFallthrough());
}
