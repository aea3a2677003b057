// The row operators (layer norm, activations, token log probabilities) for
// Python: argument checks, memory, launches and autograd nodes over the C ABI of
// include/pratchya_fp8.h, in one call from functional.py.
//
// Why not ctypes and torch.autograd.Function as for the quantized arrays: these
// operators' kernels take 3 to 80 us where a Python forward and backward took 110
// us, 60 of them the interpreter's work on the engine's thread.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <mutex>
#include <numeric>
#include <optional>

#include "pratchya_fp8.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

// A status other than PRATCHYA_OK; PRATCHYA_EINVAL becomes a ValueError instead.
struct LibraryError : std::runtime_error {
  int rc;
  LibraryError(int rc, const std::string& what) : std::runtime_error(what), rc(rc) {}
};

void check(int rc, const char* what) {
  if (rc == PRATCHYA_OK) return;
  const std::string msg = std::string(what) + ": " + pratchya_last_error();
  TORCH_CHECK_VALUE(rc != PRATCHYA_EINVAL, msg);
  throw LibraryError(rc, msg + " (status " + std::to_string(rc) + ")");
}

void require_gpu(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "pratchya_amd runs on the GPU only; got a tensor on ", t.device(),
              " (there is no CPU fallback)");
}

int float_code(const Tensor& t, const char* what) {
  if (t.scalar_type() == at::kBFloat16) return PRATCHYA_DT_BF16;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, what, ": unsupported dtype torch.",
                   t.scalar_type() == at::kHalf ? "float16" : t.scalar_type() == at::kDouble ? "float64"
                                                                                             : toString(t.scalar_type()),
                   "; expected float32 or bfloat16");
  return PRATCHYA_DT_F32;
}

hipStream_t stream_of(const Tensor& t) {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// Straight from the device's allocator: at::empty's dispatch costs as much again.
Tensor new_empty(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}

void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// An array read as rows of its last axis: itself where its rows are one stride
// apart (slices of a wider array, broadcast rows), else a contiguous copy.
struct RowArray {
  Tensor t;
  int64_t rows, width, ld;
};
RowArray as_rows(const Tensor& x, const char* what) {
  TORCH_CHECK_VALUE(x.dim() > 0, what, " needs an array of rows");
  const int64_t width = x.size(-1), rows = width ? x.numel() / width : 0;
  if (x.is_contiguous()) return {x, rows, width, width};
  if (x.stride(-1) == 1) {
    int64_t step = -1, span = 0;
    bool even = true;
    for (int64_t d = x.dim() - 2; d >= 0 && even; --d) {
      if (x.size(d) == 1) continue;
      if (step < 0) step = x.stride(d);
      else even = x.stride(d) == span;
      span = x.stride(d) * x.size(d);
    }
    if (even) return {x, rows, width, step < 0 ? width : step};
  }
  return {x.contiguous(), rows, width, width};
}

// A [width] vector of parameters.
struct Param {
  void* p = nullptr;
  int code = PRATCHYA_DT_F32;
};
Param param(const MaybeTensor& v, int64_t width, const Tensor& x, const char* what) {
  if (!v) return {};
  TORCH_CHECK_VALUE(v->dim() == 1 && v->size(0) == width && v->device() == x.device(), what, " of shape ", v->sizes(),
                    " on ", v->device(), " for rows of ", width, " on ", x.device());
  TORCH_CHECK_VALUE(v->is_contiguous(), what, " must be contiguous");
  return {v->data_ptr(), float_code(*v, what)};
}

// An input as the backward pass reads it: the array, or its quantized form.
struct Kept {
  Tensor x, sc8, sc32;
  int64_t blk = 0;
};

Kept stored_buffers(int64_t rows, int64_t width, int64_t blk, const Tensor& like) {
  const int64_t n = rows * (width / blk), K = std::gcd(std::max<int64_t>(1, blk / 16), n), M = n / K;
  return {new_empty({rows, width}, at::kFloat8_e4m3fn, like), new_empty({M, K}, at::kFloat8_e8m0fnu, like),
          new_empty({M, 1, 1}, at::kFloat, like), blk};
}

void check_block(int64_t a, int64_t blk, int64_t width, const char* what) {
  TORCH_CHECK_VALUE(a == 1 && (blk == 16 || blk == 32 || blk == 64 || blk == 128) && width % blk == 0, what,
                    ": block grid (", a, ", ", blk, ") for rows of ", width,
                    "; expected (1, b) with b of (16, 32, 64, 128) dividing them");
}

struct Grid {
  int64_t a = 1, b = 0;      // b = 0: not stored
};

// The source arguments of a backward entry point, checked against its cotangent.
struct Source {
  RowArray x;
  int code;
};
Source source(const Kept& k, const RowArray& dy, const char* what) {
  if (!k.blk) {
    TORCH_CHECK_VALUE(k.x.numel() == dy.rows * dy.width && k.x.scalar_type() == dy.t.scalar_type() &&
                          k.x.device() == dy.t.device(),
                      what, ": an input of ", k.x.sizes(), " ", k.x.scalar_type(), " for a cotangent of [", dy.rows, ", ",
                      dy.width, "] ", dy.t.scalar_type());
    const RowArray x = as_rows(k.x, what);
    TORCH_CHECK_VALUE(x.width == dy.width, what, ": an input of ", k.x.sizes(), " for a cotangent of [", dy.rows, ", ",
                      dy.width, "]");
    return {x, float_code(x.t, what)};
  }
  const int64_t n = dy.rows * (dy.width / k.blk);
  TORCH_CHECK_VALUE(k.x.dim() == 2 && k.x.size(0) == dy.rows && k.x.size(1) == dy.width && k.x.is_contiguous() &&
                        k.sc8.is_contiguous() && k.sc32.is_contiguous() && k.sc8.numel() == n &&
                        k.sc32.numel() * std::gcd(std::max<int64_t>(1, k.blk / 16), n) == n &&
                        k.x.element_size() == 1 && k.sc8.element_size() == 1 && k.sc32.scalar_type() == at::kFloat &&
                        k.x.device() == dy.t.device(),
                    what, ": a stored input of ", k.x.sizes(), " for a cotangent of [", dy.rows, ", ", dy.width, "]");
  return {{k.x, dy.rows, dy.width, dy.width}, PRATCHYA_DT_E4M3};
}

// --------------------------------------------------------------------------
// layer norm
// --------------------------------------------------------------------------
struct Normed {
  Tensor y, stats;
  Kept kept;
};

Normed layer_norm_fwd(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps, int64_t groups,
                      bool want_stats, const Grid& grid) {
  const char* what = "layer_norm";
  require_gpu(x);
  const int code = float_code(x, what);
  const RowArray r = as_rows(x, what);
  TORCH_CHECK_VALUE(groups >= 1 && r.width % groups == 0, what, ": ", groups, " groups do not divide rows of ", r.width);
  const Param w = param(weight, r.width, x, "layer_norm: weight"), b = param(bias, r.width, x, "layer_norm: bias");
  if (grid.b) {
    check_block(grid.a, grid.b, r.width, what);
    TORCH_CHECK_VALUE(r.width / groups % 8 == 0, what, ": block grid for ", groups, " groups of ", r.width / groups,
                      " elements; an 8-bit input needs groups of a multiple of 8");
  }
  const c10::DeviceGuard guard(x.device());
  const hipStream_t stream = stream_of(x);
  Normed out;
  out.y = new_empty(x.sizes(), x.scalar_type(), x);
  if (want_stats) out.stats = new_empty({r.rows * groups, 2}, at::kFloat, x);
  uint8_t *x8 = nullptr, *sc8 = nullptr;
  float* sc32 = nullptr;
  if (grid.b) {
    out.kept = stored_buffers(r.rows, r.width, grid.b, x);
    uint8_t* p8 = static_cast<uint8_t*>(out.kept.x.data_ptr());
    uint8_t* ps8 = static_cast<uint8_t*>(out.kept.sc8.data_ptr());
    float* ps32 = static_cast<float*>(out.kept.sc32.data_ptr());
    if (pratchya_layer_norm_stores(r.width, groups, grid.b)) {
      x8 = p8;
      sc8 = ps8;
      sc32 = ps32;
    } else if (x.numel()) {      // scale groups run over the rows' ends: the quantizer's own pass
      Tensor q = r.t.contiguous();
      if (reinterpret_cast<uintptr_t>(q.data_ptr()) % 16) q = q.clone();
      const int64_t bytes = (int64_t)pratchya_quantize_workspace_bytes(code, 1, r.rows, r.width, 1, grid.b);
      const Tensor ws = bytes ? new_empty({bytes}, at::kByte, x) : Tensor();
      check(pratchya_quantize(q.data_ptr(), code, 1, r.rows, r.width, 1, grid.b, p8, ps8, ps32, address(ws),
                              (size_t)bytes, stream),
            "quantize");
    }
  }
  check(pratchya_layer_norm(r.t.data_ptr(), r.ld, code, w.p, w.code, b.p, b.code, r.rows, r.width, groups, (float)eps,
                            out.y.data_ptr(), static_cast<float*>(address(out.stats)), x8, sc8, sc32, grid.b, stream),
        what);
  return out;
}

// dx, dw and db, undefined where not needed.
std::array<Tensor, 3> layer_norm_bwd(const Kept& kept, const Tensor& cotangent, const MaybeTensor& weight,
                                     const Tensor& stats, int64_t groups, std::array<bool, 3> need,
                                     at::ScalarType bias_type) {
  const char* what = "layer_norm_bwd";
  require_gpu(cotangent);
  const int code = float_code(cotangent, what);
  const RowArray dy = as_rows(cotangent, what);
  TORCH_CHECK_VALUE(groups >= 1 && dy.width % groups == 0, what, ": ", groups, " groups do not divide rows of ",
                    dy.width);
  TORCH_CHECK_VALUE(stats.numel() == 2 * dy.rows * groups && stats.is_contiguous() &&
                        stats.scalar_type() == at::kFloat && stats.device() == cotangent.device(),
                    what, ": statistics of ", stats.sizes(), " for ", dy.rows, " rows of ", groups, " segments");
  const Source src = source(kept, dy, what);
  const Param w = param(weight, dy.width, cotangent, "layer_norm_bwd: weight");
  const c10::DeviceGuard guard(cotangent.device());
  std::array<Tensor, 3> out;
  const at::ScalarType w_type = weight ? weight->scalar_type() : at::kFloat;
  const bool some = dy.rows && dy.width;
  if (need[0]) out[0] = new_empty(cotangent.sizes(), cotangent.scalar_type(), cotangent);
  if (need[1]) out[1] = new_empty({dy.width}, w_type, cotangent);
  if (need[2]) out[2] = new_empty({dy.width}, bias_type, cotangent);
  Tensor ws;
  int64_t bytes = 0;
  if (some && (need[1] || need[2])) {
    bytes = pratchya_layer_norm_bwd_workspace_bytes(dy.rows, dy.width, groups);
    ws = new_empty({bytes}, at::kByte, cotangent);
  } else if (!some) {
    for (int i = 1; i < 3; ++i)
      if (out[i].defined()) out[i].zero_();
  }
  check(pratchya_layer_norm_bwd(
            src.x.t.data_ptr(), src.x.ld, src.code, static_cast<const uint8_t*>(address(kept.sc8)),
            static_cast<const float*>(address(kept.sc32)), kept.blk, dy.t.data_ptr(), dy.ld, code, w.p, w.code,
            static_cast<const float*>(stats.data_ptr()), dy.rows, dy.width, groups, address(out[0]), address(out[1]),
            w_type == at::kBFloat16 ? PRATCHYA_DT_BF16 : PRATCHYA_DT_F32, address(out[2]),
            bias_type == at::kBFloat16 ? PRATCHYA_DT_BF16 : PRATCHYA_DT_F32, address(ws), bytes, stream_of(cotangent)),
        what);
  return out;
}

// --------------------------------------------------------------------------
// activations
// --------------------------------------------------------------------------
struct Activated {
  Tensor y;
  Kept kept;
};

Activated activation_fwd(const Tensor& x, int kind, const Grid& grid) {
  const char* what = "activation";
  require_gpu(x);
  const int code = float_code(x, what);
  const RowArray r = as_rows(x, what);
  if (grid.b) check_block(grid.a, grid.b, r.width, what);
  const c10::DeviceGuard guard(x.device());
  Activated out;
  out.y = new_empty(x.sizes(), x.scalar_type(), x);
  if (grid.b) out.kept = stored_buffers(r.rows, r.width, grid.b, x);
  check(pratchya_activation(r.t.data_ptr(), r.ld, code, kind, r.rows, r.width, out.y.data_ptr(),
                            static_cast<uint8_t*>(address(out.kept.x)), static_cast<uint8_t*>(address(out.kept.sc8)),
                            static_cast<float*>(address(out.kept.sc32)), grid.b, stream_of(x)),
        what);
  return out;
}

Tensor activation_bwd(const Kept& kept, const Tensor& cotangent, int kind) {
  const char* what = "activation_bwd";
  require_gpu(cotangent);
  const int code = float_code(cotangent, what);
  const RowArray dy = as_rows(cotangent, what);
  const Source src = source(kept, dy, what);
  const c10::DeviceGuard guard(cotangent.device());
  const Tensor dx = new_empty(cotangent.sizes(), cotangent.scalar_type(), cotangent);
  check(pratchya_activation_bwd(src.x.t.data_ptr(), src.x.ld, src.code,
                                static_cast<const uint8_t*>(address(kept.sc8)),
                                static_cast<const float*>(address(kept.sc32)), kept.blk, dy.t.data_ptr(), dy.ld, code,
                                kind, dy.rows, dy.width, dx.data_ptr(), stream_of(cotangent)),
        what);
  return dx;
}

// --------------------------------------------------------------------------
// token log probabilities
// --------------------------------------------------------------------------
constexpr int64_t kMaxTop = 64;

struct Scored {
  Tensor logprobs, entropy, top_logprobs, top_tokens, stats, tokens;
};

Scored token_logprobs_fwd(const Tensor& logits, const Tensor& tokens, bool entropy, int64_t top, bool want_stats) {
  const char* what = "token_logprobs";
  require_gpu(logits);
  require_gpu(tokens);
  const int code = float_code(logits, what);
  TORCH_CHECK_VALUE(logits.dim() > 0 && tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1) &&
                        tokens.device() == logits.device(),
                    what, ": tokens of ", tokens.sizes(), " on ", tokens.device(), " for logits of ", logits.sizes(),
                    " on ", logits.device());
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt, what, ": tokens of ",
                   tokens.scalar_type(), "; expected int64 or int32");
  const int64_t vocab = logits.size(-1);
  TORCH_CHECK_VALUE(vocab >= 1 && top >= 0 && top <= vocab && top <= kMaxTop, what, ": ", top, " alternatives of ",
                    vocab, " (0 to ", kMaxTop, ", at most the vocabulary)");
  const c10::DeviceGuard guard(logits.device());
  const RowArray r = as_rows(logits, what);
  Scored out;
  out.tokens = tokens.scalar_type() == at::kLong && tokens.is_contiguous() ? tokens : tokens.to(at::kLong).contiguous();
  out.logprobs = new_empty(tokens.sizes(), at::kFloat, logits);
  if (entropy) out.entropy = new_empty(tokens.sizes(), at::kFloat, logits);
  if (want_stats) out.stats = new_empty({r.rows, 3}, at::kFloat, logits);
  Tensor ws;
  int64_t bytes = 0;
  if (top) {
    c10::DimVector shape(tokens.sizes());
    shape.push_back(top);
    out.top_logprobs = new_empty(shape, at::kFloat, logits);
    out.top_tokens = new_empty(shape, at::kLong, logits);
    bytes = pratchya_token_logprobs_workspace_bytes(r.rows, vocab, (int)top);
    if (bytes) ws = new_empty({bytes}, at::kByte, logits);
  }
  check(pratchya_token_logprobs(r.t.data_ptr(), r.ld, code, static_cast<const int64_t*>(out.tokens.data_ptr()), r.rows,
                                vocab, (int)top, static_cast<float*>(out.logprobs.data_ptr()),
                                static_cast<float*>(address(out.entropy)), static_cast<float*>(address(out.stats)),
                                static_cast<float*>(address(out.top_logprobs)),
                                static_cast<int64_t*>(address(out.top_tokens)), address(ws), bytes, stream_of(logits)),
        what);
  return out;
}

Tensor token_logprobs_bwd(const Tensor& logits, const Tensor& tokens, const Tensor& stats, Tensor g, Tensor gh) {
  const char* what = "token_logprobs_bwd";
  require_gpu(logits);
  const int code = float_code(logits, what);
  const c10::DeviceGuard guard(logits.device());
  const RowArray r = as_rows(logits, what);
  TORCH_CHECK_VALUE(tokens.numel() == r.rows && tokens.device() == logits.device() && stats.dim() == 2 &&
                        stats.size(0) == r.rows && stats.size(1) == 3 && stats.is_contiguous() &&
                        stats.scalar_type() == at::kFloat && stats.device() == logits.device(),
                    what, ": statistics of ", stats.sizes(), " and ", tokens.numel(), " tokens for logits of ",
                    logits.sizes());
  for (Tensor* t : {&g, &gh}) {
    if (!t->defined()) continue;
    TORCH_CHECK_VALUE(t->numel() == r.rows && t->scalar_type() == at::kFloat && t->device() == logits.device(), what,
                      ": a cotangent of ", t->sizes(), " ", t->scalar_type(), " for ", r.rows, " rows");
    *t = t->contiguous();
  }
  const Tensor tok = tokens.to(at::kLong).contiguous();
  const Tensor dx = new_empty(logits.sizes(), logits.scalar_type(), logits);
  check(pratchya_token_logprobs_bwd(r.t.data_ptr(), r.ld, code, static_cast<const int64_t*>(tok.data_ptr()),
                                    static_cast<const float*>(stats.data_ptr()), static_cast<const float*>(address(g)),
                                    static_cast<const float*>(address(gh)), r.rows, r.width, dx.data_ptr(),
                                    stream_of(logits)),
        what);
  return dx;
}

// --------------------------------------------------------------------------
// embedding
// --------------------------------------------------------------------------
// Tokens as the kernels read them: int64, contiguous.
Tensor token_array(const Tensor& tokens, const Tensor& like, const char* what) {
  TORCH_CHECK_VALUE(tokens.device() == like.device(), what, ": tokens on ", tokens.device(), " for an array on ",
                    like.device());
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt, what, ": tokens of ",
                   tokens.scalar_type(), "; expected int64 or int32");
  return tokens.scalar_type() == at::kLong && tokens.is_contiguous() ? tokens : tokens.to(at::kLong).contiguous();
}

struct Embedded {
  Tensor y, tokens;
};

Embedded embedding_fwd(const Tensor& table, const Tensor& tokens, double scale) {
  const char* what = "embedding";
  require_gpu(table);
  require_gpu(tokens);
  const int code = float_code(table, what);
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) >= 1, what, ": a table of ", table.sizes(),
                    "; expected [vocabulary, width]");
  const c10::DeviceGuard guard(table.device());
  Embedded out;
  out.tokens = token_array(tokens, table, what);
  const RowArray r = as_rows(table, what);
  c10::DimVector shape(tokens.sizes());
  shape.push_back(table.size(1));
  out.y = new_empty(shape, table.scalar_type(), table);
  check(pratchya_embedding(r.t.data_ptr(), r.ld, code, static_cast<const int64_t*>(out.tokens.data_ptr()),
                           tokens.numel(), table.size(0), table.size(1), (float)scale, out.y.data_ptr(),
                           stream_of(table)),
        what);
  return out;
}

Tensor embedding_bwd(const Tensor& cotangent, const Tensor& tokens, int64_t vocab, double scale) {
  const char* what = "embedding_bwd";
  require_gpu(cotangent);
  const int code = float_code(cotangent, what);
  const c10::DeviceGuard guard(cotangent.device());
  const int64_t width = cotangent.size(-1), n = tokens.numel();
  const RowArray dy = as_rows(cotangent, what);
  const Tensor dtable = new_empty({vocab, width}, cotangent.scalar_type(), cotangent);
  const int64_t bytes = pratchya_embedding_bwd_workspace_bytes(n, vocab, width);
  const Tensor ws = new_empty({bytes}, at::kByte, cotangent);
  check(pratchya_embedding_bwd(dy.t.data_ptr(), dy.ld, code, static_cast<const int64_t*>(tokens.data_ptr()), n, vocab,
                               width, (float)scale, dtable.data_ptr(), ws.data_ptr(), bytes, stream_of(cotangent)),
        what);
  return dtable;
}

// --------------------------------------------------------------------------
// cross entropy of an output head
// --------------------------------------------------------------------------
// A weight [C, V] as the library reads it: its rows, or those of the table [V, C]
// whose transposed view it is.
struct HeadWeight {
  Tensor t;
  int64_t ld;
  bool rows;
};
HeadWeight head_weight(const Tensor& w) {
  if (w.stride(1) == 1 || w.size(1) == 1) {
    if (w.stride(1) == 1 && (w.size(0) == 1 || w.stride(0) >= w.size(1)))
      return {w, w.size(0) == 1 ? w.size(1) : w.stride(0), false};
  }
  if (w.stride(0) == 1 && (w.size(1) == 1 || w.stride(1) >= w.size(0)))
    return {w, w.size(1) == 1 ? w.size(0) : w.stride(1), true};
  return {w.contiguous(), w.size(1), false};
}

struct HeadLoss {
  Tensor loss, stats, targets;
};

HeadLoss head_loss_fwd(const Tensor& x, const Tensor& weight, const Tensor& targets, double smoothing, bool want_stats) {
  const char* what = "linear_cross_entropy";
  require_gpu(x);
  require_gpu(weight);
  require_gpu(targets);
  const int code = float_code(x, what);
  TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type(), what, ": a weight of ", weight.scalar_type(), " for x of ",
                   x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() > 0 && weight.dim() == 2 && weight.size(0) == x.size(-1) && weight.size(0) >= 1 &&
                        weight.size(1) >= 1 && weight.device() == x.device(),
                    what, ": a weight of ", weight.sizes(), " on ", weight.device(), " for x of ", x.sizes(), " on ",
                    x.device());
  TORCH_CHECK_VALUE(targets.sizes() == x.sizes().slice(0, x.dim() - 1), what, ": targets of ", targets.sizes(),
                    " for x of ", x.sizes());
  TORCH_CHECK_VALUE(smoothing >= 0.0 && smoothing <= 1.0, what, ": label smoothing of ", smoothing, "; expected 0 to 1");
  const c10::DeviceGuard guard(x.device());
  HeadLoss out;
  out.targets = token_array(targets, x, what);
  const RowArray r = as_rows(x, what);
  const HeadWeight w = head_weight(weight);
  out.loss = new_empty(targets.sizes(), at::kFloat, x);
  if (want_stats) out.stats = new_empty({r.rows, 2}, at::kFloat, x);
  const int64_t bytes = pratchya_linear_cross_entropy_workspace_bytes(
      r.t.data_ptr(), r.ld, w.t.data_ptr(), w.ld, code, w.rows, r.rows, r.width, weight.size(1), 0, 0);
  const Tensor ws = bytes ? new_empty({bytes}, at::kByte, x) : Tensor();
  check(pratchya_linear_cross_entropy(r.t.data_ptr(), r.ld, w.t.data_ptr(), w.ld, code, w.rows,
                                      static_cast<const int64_t*>(out.targets.data_ptr()), r.rows, r.width,
                                      weight.size(1), (float)smoothing, static_cast<float*>(out.loss.data_ptr()),
                                      static_cast<float*>(address(out.stats)), address(ws), bytes, stream_of(x)),
        what);
  return out;
}

// dx and dw, undefined where not needed; dw has the weight's layout.
std::array<Tensor, 2> head_loss_bwd(const Tensor& x, const Tensor& weight, const Tensor& targets, const Tensor& stats,
                                    Tensor g, double smoothing, std::array<bool, 2> need) {
  const char* what = "linear_cross_entropy_bwd";
  const int code = float_code(x, what);
  const c10::DeviceGuard guard(x.device());
  const RowArray r = as_rows(x, what);
  const HeadWeight w = head_weight(weight);
  const int64_t vocab = weight.size(1);
  TORCH_CHECK_VALUE(g.numel() == r.rows && g.scalar_type() == at::kFloat && g.device() == x.device(), what,
                    ": a cotangent of ", g.sizes(), " ", g.scalar_type(), " for ", r.rows, " rows");
  g = g.contiguous();
  std::array<Tensor, 2> out;
  if (need[0]) out[0] = new_empty(x.sizes(), x.scalar_type(), x);
  Tensor dw;
  if (need[1]) dw = w.rows ? new_empty({vocab, r.width}, x.scalar_type(), x) : new_empty({r.width, vocab}, x.scalar_type(), x);
  const int64_t bytes = pratchya_linear_cross_entropy_workspace_bytes(
      r.t.data_ptr(), r.ld, w.t.data_ptr(), w.ld, code, w.rows, r.rows, r.width, vocab, need[0], need[1]);
  const Tensor ws = bytes ? new_empty({bytes}, at::kByte, x) : Tensor();
  check(pratchya_linear_cross_entropy_bwd(r.t.data_ptr(), r.ld, w.t.data_ptr(), w.ld, code, w.rows,
                                          static_cast<const int64_t*>(targets.data_ptr()),
                                          static_cast<const float*>(stats.data_ptr()),
                                          static_cast<const float*>(g.data_ptr()), r.rows, r.width, vocab,
                                          (float)smoothing, address(out[0]), address(dw), address(ws), bytes,
                                          stream_of(x)),
        what);
  if (need[1]) out[1] = w.rows ? dw.t() : dw;
  return out;
}

// --------------------------------------------------------------------------
// linear attention
// --------------------------------------------------------------------------
// Arguments of the kernels from arrays [B, T, H, D] (or [B, H, D], one token).
struct Mix {
  Tensor q, k, v, decay, lengths, state;
  int code = 0, g_code = 0;
  int64_t B = 0, T = 0, H = 0, dk = 0, dv = 0;
  std::array<int64_t, 15> strides{};

  const int64_t* length_ptr() const { return static_cast<const int64_t*>(address(lengths)); }
  const float* state_ptr() const { return static_cast<const float*>(address(state)); }
};

// Itself where its last axis is contiguous, else a contiguous copy.
Tensor last_contiguous(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

Mix mix_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const MaybeTensor& state,
             const MaybeTensor& lengths, bool one, const char* what) {
  for (const Tensor* t : {&q, &k, &v, &decay}) require_gpu(*t);
  Mix m;
  m.code = float_code(q, what);
  m.g_code = float_code(decay, what);
  const int64_t axes = one ? 3 : 4;
  TORCH_CHECK_VALUE(q.dim() == axes && k.sizes() == q.sizes() && v.dim() == axes &&
                        v.sizes().slice(0, axes - 1) == q.sizes().slice(0, axes - 1) &&
                        decay.sizes() == q.sizes().slice(0, axes - 1),
                    what, ": q of ", q.sizes(), ", k of ", k.sizes(), ", v of ", v.sizes(), ", log_decay of ",
                    decay.sizes(), "; expected [batch", one ? "" : ", length", ", heads, width], decays without a width");
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), what, ": q, k and v of ",
                   q.scalar_type(), ", ", k.scalar_type(), " and ", v.scalar_type());
  TORCH_CHECK_VALUE(k.device() == q.device() && v.device() == q.device() && decay.device() == q.device(), what,
                    ": arrays on different devices");
  m.B = q.size(0);
  m.T = one ? 1 : q.size(1);
  m.H = q.size(axes - 2);
  m.dk = q.size(-1);
  m.dv = v.size(-1);
  TORCH_CHECK_VALUE(m.H >= 1 && m.dk >= 1 && m.dv >= 1, what, ": q of ", q.sizes(), " and v of ", v.sizes());
  m.q = last_contiguous(q);
  m.k = last_contiguous(k);
  m.v = last_contiguous(v);
  m.decay = decay;
  int i = 0;
  for (const Tensor* t : {&m.q, &m.k, &m.v, &m.decay})
    for (int64_t d = 0; d < axes - 1; ++d) m.strides[i++] = t->stride(d);
  if (state) {
    TORCH_CHECK_VALUE(state->dim() == 4 && state->size(0) == m.B && state->size(1) == m.H && state->size(2) == m.dk &&
                          state->size(3) == m.dv && state->device() == q.device(),
                      what, ": a state of ", state->sizes(), " on ", state->device(), "; expected [", m.B, ", ", m.H, ", ",
                      m.dk, ", ", m.dv, "] on ", q.device());
    TORCH_CHECK_TYPE(state->scalar_type() == at::kFloat, what, ": a state of ", state->scalar_type(),
                     "; expected float32");
    m.state = one ? *state : state->contiguous();
  }
  if (lengths) {
    require_gpu(*lengths);
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == m.B && lengths->device() == q.device(), what,
                      ": lengths of ", lengths->sizes(), " on ", lengths->device(), " for ", m.B, " sequences");
    TORCH_CHECK_TYPE(lengths->scalar_type() == at::kLong || lengths->scalar_type() == at::kInt, what, ": lengths of ",
                     lengths->scalar_type(), "; expected int64 or int32");
    m.lengths = lengths->to(at::kLong).contiguous();
  }
  return m;
}

struct Mixed {
  Tensor out, state, starts;
};

Mixed linear_attention_fwd(const Mix& m, double scale, bool train) {
  Mixed r;
  r.out = new_empty({m.B, m.T, m.H, m.dv}, m.q.scalar_type(), m.q);
  r.state = new_empty({m.B, m.H, m.dk, m.dv}, at::kFloat, m.q);
  // what a backward pass reads, and what this call alone does
  const int64_t floats = pratchya_linear_attention_starts_floats(m.B, m.T, m.H, m.dk, m.dv, m.code, train),
                kept = pratchya_linear_attention_states_floats(m.B, m.T, m.H, m.dk, m.dv, m.code, train);
  Tensor parts;
  if (floats) {
    r.starts = new_empty({kept}, at::kFloat, m.q);
    parts = new_empty({floats - kept}, at::kFloat, m.q);
  }
  check(pratchya_linear_attention_parts(
            m.q.data_ptr(), m.k.data_ptr(), m.v.data_ptr(), m.code, m.decay.data_ptr(), m.g_code, m.strides.data(),
            m.length_ptr(), m.state_ptr(), m.B, m.T, m.H, m.dk, m.dv, (float)scale, train, r.out.data_ptr(),
            static_cast<float*>(r.state.data_ptr()), static_cast<float*>(address(r.starts)),
            static_cast<float*>(address(parts)), stream_of(m.q)),
        "linear_attention");
  return r;
}

// dq, dk, dv, the decays' and the state's gradient, the last two undefined where not needed.
std::array<Tensor, 5> linear_attention_bwd(Mix m, const Tensor& starts, const Tensor& state_out, const Tensor& dout,
                                           const Tensor& dstate_out, double scale, bool want_decay, bool want_state) {
  const char* what = "linear_attention_bwd";
  // a cotangent of one output only: the other one's is 0
  Tensor d = dout.defined() ? dout : at::zeros({}, m.q.options()).expand({m.B, m.T, m.H, m.dv});
  TORCH_CHECK_VALUE(d.dim() == 4 && d.size(0) == m.B && d.size(1) == m.T && d.size(2) == m.H && d.size(3) == m.dv &&
                        d.scalar_type() == m.q.scalar_type() && d.device() == m.q.device(),
                    what, ": a cotangent of ", d.sizes(), " ", d.scalar_type());
  d = last_contiguous(d);
  for (int i = 0; i < 3; ++i) m.strides[12 + i] = d.stride(i);
  const Tensor ds = dstate_out.defined() ? dstate_out.to(at::kFloat).contiguous() : Tensor();
  std::array<Tensor, 5> out;
  out[0] = new_empty({m.B, m.T, m.H, m.dk}, m.q.scalar_type(), m.q);
  out[1] = new_empty({m.B, m.T, m.H, m.dk}, m.q.scalar_type(), m.q);
  out[2] = new_empty({m.B, m.T, m.H, m.dv}, m.q.scalar_type(), m.q);
  if (want_decay) out[3] = new_empty({m.B, m.T, m.H}, m.decay.scalar_type(), m.q);
  if (want_state) out[4] = new_empty({m.B, m.H, m.dk, m.dv}, at::kFloat, m.q);
  const int64_t bytes = pratchya_linear_attention_bwd_workspace_bytes(m.B, m.T, m.H, m.dk, m.dv, m.code);
  const Tensor ws = bytes ? new_empty({bytes}, at::kByte, m.q) : Tensor();
  check(pratchya_linear_attention_bwd(
            m.q.data_ptr(), m.k.data_ptr(), m.v.data_ptr(), m.code, m.decay.data_ptr(), m.g_code, m.strides.data(),
            m.length_ptr(), m.state_ptr(), static_cast<const float*>(address(state_out)),
            static_cast<const float*>(address(starts)), d.data_ptr(), static_cast<const float*>(address(ds)), m.B, m.T,
            m.H, m.dk, m.dv, (float)scale, out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), address(out[3]),
            static_cast<float*>(address(out[4])), address(ws), bytes, stream_of(m.q)),
        what);
  return out;
}

// --------------------------------------------------------------------------
// autograd nodes
// --------------------------------------------------------------------------
// Gradients of gradients are not computed: with create_graph the results are
// differentiable into an error, as torch's once_differentiable has it (they count as
// differentiable, since the error's node is attached to those only).
variable_list once(variable_list&& grads, const char* what) {
  if (!at::GradMode::is_enabled()) return std::move(grads);
  for (Tensor& g : grads)
    if (g.defined()) g.set_requires_grad(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + ": its gradient cannot be differentiated again", (int)grads.size());
  return (*error)(std::move(grads));
}

// A node's saved arrays are read and given up under its mutex: backward passes of
// several threads may share a graph, and run without the interpreter's lock.
struct KeptNode : torch::autograd::Node {
  SavedVariable x_, sc8_, sc32_;
  int64_t blk_ = 0;
  void keep(const Tensor& x, const Kept& k) {
    blk_ = k.blk;
    x_ = SavedVariable(k.blk ? k.x : x, false);
    if (blk_) {
      sc8_ = SavedVariable(k.sc8, false);
      sc32_ = SavedVariable(k.sc32, false);
    }
  }
  Kept kept() const {
    Kept k;
    k.blk = blk_;
    k.x = x_.unpack();
    if (blk_) {
      k.sc8 = sc8_.unpack();
      k.sc32 = sc32_.unpack();
    }
    return k;
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    release();
  }

 protected:
  virtual void release() {
    x_.reset_data();
    sc8_.reset_data();
    sc32_.reset_data();
  }
};

struct PratchyaLayerNormBackward : KeptNode {
  SavedVariable weight_, stats_;
  bool has_weight_ = false;
  int64_t groups_ = 1;
  at::ScalarType bias_type_ = at::kFloat;
  variable_list apply(variable_list&& grads) override {
    variable_list out(3);
    if (!grads[0].defined()) return out;
    Kept x;
    MaybeTensor weight;
    Tensor stats;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      x = kept();
      if (has_weight_) weight = weight_.unpack();
      stats = stats_.unpack();
    }
    auto got = layer_norm_bwd(x, grads[0], weight, stats, groups_,
                              {task_should_compute_output(0), task_should_compute_output(1),
                               task_should_compute_output(2)},
                              bias_type_);
    for (int i = 0; i < 3; ++i) out[i] = std::move(got[i]);
    return once(std::move(out), "layer_norm");
  }

 protected:
  void release() override {
    KeptNode::release();
    weight_.reset_data();
    stats_.reset_data();
  }
};

struct PratchyaActivationBackward : KeptNode {
  int kind_ = 0;
  variable_list apply(variable_list&& grads) override {
    variable_list out(1);
    if (!grads[0].defined()) return out;
    Kept x;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      x = kept();
    }
    out[0] = activation_bwd(x, grads[0], kind_);
    return once(std::move(out), "activation");
  }
};

struct PratchyaTokenLogprobsBackward : torch::autograd::Node {
  SavedVariable logits_, tokens_, stats_;
  variable_list apply(variable_list&& grads) override {
    variable_list out(1);
    const Tensor g = grads[0], gh = grads.size() > 1 ? grads[1] : Tensor();
    if (!g.defined() && !gh.defined()) return out;
    Tensor logits, tokens, stats;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      logits = logits_.unpack();
      tokens = tokens_.unpack();
      stats = stats_.unpack();
    }
    out[0] = token_logprobs_bwd(logits, tokens, stats, g, gh);
    return once(std::move(out), "token_logprobs");
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    logits_.reset_data();
    tokens_.reset_data();
    stats_.reset_data();
  }
};

struct PratchyaEmbeddingBackward : torch::autograd::Node {
  SavedVariable tokens_;
  int64_t vocab_ = 0;
  double scale_ = 1.0;
  variable_list apply(variable_list&& grads) override {
    variable_list out(1);
    if (!grads[0].defined()) return out;
    Tensor tokens;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      tokens = tokens_.unpack();
    }
    out[0] = embedding_bwd(grads[0], tokens, vocab_, scale_);
    return once(std::move(out), "embedding");
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    tokens_.reset_data();
  }
};

struct PratchyaLinearCrossEntropyBackward : torch::autograd::Node {
  SavedVariable x_, weight_, targets_, stats_;
  double smoothing_ = 0.0;
  variable_list apply(variable_list&& grads) override {
    variable_list out(2);
    if (!grads[0].defined()) return out;
    Tensor x, weight, targets, stats;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      x = x_.unpack();
      weight = weight_.unpack();
      targets = targets_.unpack();
      stats = stats_.unpack();
    }
    auto got = [&] {
      at::NoGradGuard no;
      return head_loss_bwd(x, weight, targets, stats, grads[0], smoothing_,
                           {task_should_compute_output(0), task_should_compute_output(1)});
    }();
    for (int i = 0; i < 2; ++i) out[i] = std::move(got[i]);
    return once(std::move(out), "linear_cross_entropy");
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    x_.reset_data();
    weight_.reset_data();
    targets_.reset_data();
    stats_.reset_data();
  }
};

struct PratchyaLinearAttentionBackward : torch::autograd::Node {
  SavedVariable q_, k_, v_, decay_, state_, lengths_, starts_, state_out_;
  bool has_state_ = false, has_lengths_ = false;
  double scale_ = 1.0;
  variable_list apply(variable_list&& grads) override {
    variable_list out(5);
    const Tensor dout = grads[0], dstate = grads.size() > 1 ? grads[1] : Tensor();
    if (!dout.defined() && !dstate.defined()) return out;
    Tensor q, k, v, decay, starts, state_out;
    MaybeTensor state, lengths;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      q = q_.unpack();
      k = k_.unpack();
      v = v_.unpack();
      decay = decay_.unpack();
      if (has_state_) state = state_.unpack();
      if (has_lengths_) lengths = lengths_.unpack();
      starts = starts_.unpack();
      // read where it meets a cotangent of its own
      if (dstate.defined()) state_out = state_out_.unpack(shared_from_this());
    }
    auto got = [&] {
      at::NoGradGuard no;
      const c10::DeviceGuard guard(q.device());
      const Mix m = mix_args(q, k, v, decay, state, lengths, false, "linear_attention_bwd");
      return linear_attention_bwd(m, starts, state_out, dout, dstate, scale_, task_should_compute_output(3),
                                  has_state_ && task_should_compute_output(4));
    }();
    for (int i = 0; i < 5; ++i)
      if (task_should_compute_output(i)) out[i] = std::move(got[i]);
    return once(std::move(out), "linear_attention");
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&q_, &k_, &v_, &decay_, &state_, &lengths_, &starts_, &state_out_}) s->reset_data();
  }
};

bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const MaybeTensor& t) { return t && t->requires_grad(); }
Tensor or_none(const MaybeTensor& t) { return t ? *t : Tensor(); }

// The nodes hold reverse-mode gradients only.  An input with a forward-mode tangent
// would give an output without one, whose derivative counts as 0.
void refuse_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), what, ": no forward-mode derivative; the input has a tangent");
}
void refuse_tangent(const MaybeTensor& t, const char* what) {
  if (t) refuse_tangent(*t, what);
}

template <typename N>
std::shared_ptr<N> new_node() {
  return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps, int64_t groups,
                  Grid grid) {
  refuse_tangent(x, "layer_norm");
  refuse_tangent(weight, "layer_norm: weight");
  refuse_tangent(bias, "layer_norm: bias");
  const bool grad = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias));
  if (!grad) return layer_norm_fwd(x, weight, bias, eps, groups, false, {}).y;
  Normed r;
  {
    at::NoGradGuard no;
    if (!wants_grad(x) && !wants_grad(weight)) grid = {};      // only db: x is not read
    r = layer_norm_fwd(x, weight, bias, eps, groups, true, grid);
  }
  auto node = new_node<PratchyaLayerNormBackward>();
  node->set_next_edges(torch::autograd::collect_next_edges(x, or_none(weight), or_none(bias)));
  node->keep(x, r.kept);
  node->stats_ = SavedVariable(r.stats, false);
  node->has_weight_ = weight.has_value();
  if (weight) node->weight_ = SavedVariable(*weight, false);
  node->groups_ = groups;
  if (bias) node->bias_type_ = bias->scalar_type();
  torch::autograd::set_history(r.y, node);
  return r.y;
}

Tensor activation(const Tensor& x, int kind, const Grid& grid) {
  refuse_tangent(x, "activation");
  if (!(at::GradMode::is_enabled() && wants_grad(x))) return activation_fwd(x, kind, {}).y;
  Activated r;
  {
    at::NoGradGuard no;
    r = activation_fwd(x, kind, grid);
  }
  auto node = new_node<PratchyaActivationBackward>();
  node->set_next_edges(torch::autograd::collect_next_edges(x));
  node->keep(x, r.kept);
  node->kind_ = kind;
  torch::autograd::set_history(r.y, node);
  return r.y;
}

Scored token_logprobs(const Tensor& logits, const Tensor& tokens, bool entropy, int64_t top) {
  refuse_tangent(logits, "token_logprobs");
  const bool grad = at::GradMode::is_enabled() && wants_grad(logits);
  Scored r;
  {
    at::NoGradGuard no;
    r = token_logprobs_fwd(logits, tokens, entropy, top, grad);
  }
  if (!grad) return r;
  auto node = new_node<PratchyaTokenLogprobsBackward>();
  node->set_next_edges(torch::autograd::collect_next_edges(logits));
  node->logits_ = SavedVariable(logits, false);
  node->tokens_ = SavedVariable(r.tokens, false);
  node->stats_ = SavedVariable(r.stats, false);
  torch::autograd::set_history(r.logprobs, node);
  if (entropy) torch::autograd::set_history(r.entropy, node);
  return r;
}

Tensor embedding(const Tensor& table, const Tensor& tokens, double scale) {
  refuse_tangent(table, "embedding");
  const bool grad = at::GradMode::is_enabled() && wants_grad(table);
  Embedded r;
  {
    at::NoGradGuard no;
    r = embedding_fwd(table, tokens, scale);
  }
  if (!grad) return r.y;
  auto node = new_node<PratchyaEmbeddingBackward>();
  node->set_next_edges(torch::autograd::collect_next_edges(table));
  node->tokens_ = SavedVariable(r.tokens, false);
  node->vocab_ = table.size(0);
  node->scale_ = scale;
  torch::autograd::set_history(r.y, node);
  return r.y;
}

Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const Tensor& targets, double smoothing) {
  refuse_tangent(x, "linear_cross_entropy");
  refuse_tangent(weight, "linear_cross_entropy: weight");
  const bool grad = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight));
  HeadLoss r;
  {
    at::NoGradGuard no;
    r = head_loss_fwd(x, weight, targets, smoothing, grad);
  }
  if (!grad) return r.loss;
  auto node = new_node<PratchyaLinearCrossEntropyBackward>();
  node->set_next_edges(torch::autograd::collect_next_edges(x, weight));
  node->x_ = SavedVariable(x, false);
  node->weight_ = SavedVariable(weight, false);
  node->targets_ = SavedVariable(r.targets, false);
  node->stats_ = SavedVariable(r.stats, false);
  node->smoothing_ = smoothing;
  torch::autograd::set_history(r.loss, node);
  return r.loss;
}

Mixed linear_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const MaybeTensor& state,
                       const MaybeTensor& lengths, double scale) {
  const char* what = "linear_attention";
  for (const Tensor* t : {&q, &k, &v, &decay}) refuse_tangent(*t, what);
  refuse_tangent(state, what);
  const bool grad = at::GradMode::is_enabled() &&
                    (wants_grad(q) || wants_grad(k) || wants_grad(v) || wants_grad(decay) || wants_grad(state));
  Mixed r;
  Tensor lens;
  {
    at::NoGradGuard no;
    const c10::DeviceGuard guard(q.device());
    const Mix m = mix_args(q, k, v, decay, state, lengths, false, what);
    lens = m.lengths;
    r = linear_attention_fwd(m, scale, grad);
  }
  if (!grad) return r;
  auto node = new_node<PratchyaLinearAttentionBackward>();
  node->set_next_edges(torch::autograd::collect_next_edges(q, k, v, decay, or_none(state)));
  node->q_ = SavedVariable(q, false);
  node->k_ = SavedVariable(k, false);
  node->v_ = SavedVariable(v, false);
  node->decay_ = SavedVariable(decay, false);
  node->has_state_ = state.has_value();
  if (state) node->state_ = SavedVariable(*state, false);
  node->has_lengths_ = lengths.has_value();
  if (lengths) node->lengths_ = SavedVariable(lens, false);
  node->starts_ = SavedVariable(r.starts, false);
  node->scale_ = scale;
  torch::autograd::set_history(r.out, node);
  torch::autograd::set_history(r.state, node);
  node->state_out_ = SavedVariable(r.state, true);
  return r;
}

Tensor linear_attention_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const Tensor& state,
                             double scale) {
  const char* what = "linear_attention_step";
  for (const Tensor* t : {&q, &k, &v, &decay, &state}) {
    refuse_tangent(*t, what);
    TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && t->requires_grad()), what,
                      ": no gradient (the state is updated in place); linear_attention has one");
  }
  require_gpu(state);
  const c10::DeviceGuard guard(q.device());
  const Mix m = mix_args(q, k, v, decay, state, std::nullopt, true, what);
  TORCH_CHECK_VALUE(m.state.is_contiguous() && reinterpret_cast<uintptr_t>(m.state.data_ptr()) % 16 == 0, what,
                    ": the state must be contiguous and 16-byte aligned");
  const Tensor out = new_empty({m.B, m.H, m.dv}, q.scalar_type(), q);
  check(pratchya_linear_attention_step(m.q.data_ptr(), m.k.data_ptr(), m.v.data_ptr(), m.code, m.decay.data_ptr(),
                                       m.g_code, m.strides.data(), static_cast<float*>(m.state.data_ptr()), m.B, m.H,
                                       m.dk, m.dv, (float)scale, out.data_ptr(), stream_of(q)),
        what);
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return out;
}

// --------------------------------------------------------------------------
// Python
// --------------------------------------------------------------------------
const Tensor& tensor_arg(PyObject* o, const char* what) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, ": expected a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
MaybeTensor maybe_arg(PyObject* o, const char* what) {
  if (o == Py_None) return std::nullopt;
  return tensor_arg(o, what);
}
int64_t int_arg(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
double float_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
bool bool_arg(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
Grid grid_arg(PyObject* o) {
  if (o == Py_None) return {};
  THPObjectPtr pair(PySequence_Fast(o, "a block grid is a pair (a, b)"));
  if (!pair) throw python_error();
  TORCH_CHECK_VALUE(PySequence_Fast_GET_SIZE(pair.get()) == 2, "a block grid is a pair (a, b)");
  Grid g = {int_arg(PySequence_Fast_GET_ITEM(pair.get(), 0)), int_arg(PySequence_Fast_GET_ITEM(pair.get(), 1))};
  TORCH_CHECK_VALUE(g.b > 0, "block grid (", g.a, ", ", g.b, ") for rows");
  return g;
}
Kept kept_arg(PyObject* o, const Grid& grid, const char* what) {
  if (!grid.b) return {tensor_arg(o, what), Tensor(), Tensor(), 0};
  THPObjectPtr parts(PySequence_Fast(o, "a stored input is (payload, e8m0 scales, group maxima)"));
  if (!parts) throw python_error();
  TORCH_CHECK_VALUE(PySequence_Fast_GET_SIZE(parts.get()) == 3,
                    "a stored input is (payload, e8m0 scales, group maxima)");
  auto at_ = [&](int i) { return tensor_arg(PySequence_Fast_GET_ITEM(parts.get(), i), what); };
  return {at_(0), at_(1), at_(2), grid.b};
}

PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
PyObject* wrap_all(std::initializer_list<PyObject*> items) {
  PyObject* tuple = PyTuple_New((Py_ssize_t)items.size());
  Py_ssize_t i = 0;
  for (PyObject* o : items) {
    if (tuple) PyTuple_SET_ITEM(tuple, i++, o);
    else Py_XDECREF(o);
  }
  return tuple;
}
PyObject* wrap(const Kept& k) {
  if (!k.blk) Py_RETURN_NONE;
  return wrap_all({wrap(k.x), wrap(k.sc8), wrap(k.sc32)});
}

PyObject* raise_library_error(const LibraryError& e) {
  THPObjectPtr lib(PyImport_ImportModule("pratchya_amd._lib"));
  if (!lib) return nullptr;
  THPObjectPtr type(
      PyObject_GetAttrString(lib, e.rc == PRATCHYA_EUNSUPPORTED ? "PratchyaUnsupported" : "PratchyaError"));
  if (type) PyErr_SetString(type, e.what());
  return nullptr;
}

// A method of `N` positional arguments around `body`, which has no GIL inside `unlocked`.
template <Py_ssize_t N, typename F>
PyObject* method(const char* name, Py_ssize_t n, F body) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == N, name, " takes ", N, " arguments, got ", n);
  try {
    return body();
  } catch (const LibraryError& e) {
    return raise_library_error(e);
  }
  END_HANDLE_TH_ERRORS
}
template <typename F>
auto unlocked(F f) {
  pybind11::gil_scoped_release release;
  return f();
}

PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<6>("layer_norm", n, [&] {
    const Tensor& x = tensor_arg(a[0], "layer_norm");
    const MaybeTensor w = maybe_arg(a[1], "layer_norm: weight"), b = maybe_arg(a[2], "layer_norm: bias");
    const double eps = float_arg(a[3]);
    const int64_t groups = int_arg(a[4]);
    const Grid grid = grid_arg(a[5]);
    return wrap(unlocked([&] { return layer_norm(x, w, b, eps, groups, grid); }));
  });
}
PyObject* py_layer_norm_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<7>("layer_norm_fwd", n, [&] {
    const Tensor& x = tensor_arg(a[0], "layer_norm");
    const MaybeTensor w = maybe_arg(a[1], "layer_norm: weight"), b = maybe_arg(a[2], "layer_norm: bias");
    at::NoGradGuard no;
    const Normed r = layer_norm_fwd(x, w, b, float_arg(a[3]), int_arg(a[4]), bool_arg(a[5]), grid_arg(a[6]));
    return wrap_all({wrap(r.y), wrap(r.stats), wrap(r.kept)});
  });
}
PyObject* py_layer_norm_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<10>("layer_norm_bwd", n, [&] {
    const Grid grid = grid_arg(a[5]);
    const Kept kept = kept_arg(a[0], grid, "layer_norm_bwd");
    TORCH_CHECK_TYPE(THPDtype_Check(a[9]), "layer_norm_bwd: the bias's dtype is a torch.dtype");
    const at::ScalarType bias = reinterpret_cast<THPDtype*>(a[9])->scalar_type;
    TORCH_CHECK_TYPE(bias == at::kFloat || bias == at::kBFloat16, "layer_norm_bwd: unsupported bias dtype ", bias);
    at::NoGradGuard no;
    const auto r = layer_norm_bwd(kept, tensor_arg(a[1], "layer_norm_bwd"), maybe_arg(a[2], "layer_norm_bwd: weight"),
                                  tensor_arg(a[3], "layer_norm_bwd"), int_arg(a[4]),
                                  {bool_arg(a[6]), bool_arg(a[7]), bool_arg(a[8])}, bias);
    return wrap_all({wrap(r[0]), wrap(r[1]), wrap(r[2])});
  });
}
PyObject* py_activation(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<3>("activation", n, [&] {
    const Tensor& x = tensor_arg(a[0], "activation");
    const int kind = (int)int_arg(a[1]);
    const Grid grid = grid_arg(a[2]);
    return wrap(unlocked([&] { return activation(x, kind, grid); }));
  });
}
PyObject* py_activation_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<3>("activation_fwd", n, [&] {
    at::NoGradGuard no;
    const Activated r = activation_fwd(tensor_arg(a[0], "activation"), (int)int_arg(a[1]), grid_arg(a[2]));
    return wrap_all({wrap(r.y), wrap(r.kept)});
  });
}
PyObject* py_activation_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<4>("activation_bwd", n, [&] {
    at::NoGradGuard no;
    return wrap(activation_bwd(kept_arg(a[0], grid_arg(a[3]), "activation_bwd"), tensor_arg(a[1], "activation_bwd"),
                               (int)int_arg(a[2])));
  });
}
PyObject* py_token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<4>("token_logprobs", n, [&] {
    const Tensor &x = tensor_arg(a[0], "token_logprobs"), &tokens = tensor_arg(a[1], "token_logprobs");
    const bool entropy = bool_arg(a[2]);
    const int64_t top = int_arg(a[3]);
    const Scored r = unlocked([&] { return token_logprobs(x, tokens, entropy, top); });
    return wrap_all({wrap(r.logprobs), wrap(r.entropy), wrap(r.top_logprobs), wrap(r.top_tokens)});
  });
}
PyObject* py_token_logprobs_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<5>("token_logprobs_fwd", n, [&] {
    at::NoGradGuard no;
    const Scored r = token_logprobs_fwd(tensor_arg(a[0], "token_logprobs"), tensor_arg(a[1], "token_logprobs"),
                                        bool_arg(a[2]), int_arg(a[3]), bool_arg(a[4]));
    return wrap_all({wrap(r.logprobs), wrap(r.entropy), wrap(r.top_logprobs), wrap(r.top_tokens), wrap(r.stats)});
  });
}
PyObject* py_token_logprobs_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<5>("token_logprobs_bwd", n, [&] {
    const char* what = "token_logprobs_bwd";
    at::NoGradGuard no;
    return wrap(token_logprobs_bwd(tensor_arg(a[0], what), tensor_arg(a[1], what), tensor_arg(a[2], what),
                                   or_none(maybe_arg(a[3], what)), or_none(maybe_arg(a[4], what))));
  });
}

PyObject* py_embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<3>("embedding", n, [&] {
    const Tensor &table = tensor_arg(a[0], "embedding"), &tokens = tensor_arg(a[1], "embedding");
    const double scale = float_arg(a[2]);
    return wrap(unlocked([&] { return embedding(table, tokens, scale); }));
  });
}

PyObject* py_linear_cross_entropy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<4>("linear_cross_entropy", n, [&] {
    const char* what = "linear_cross_entropy";
    const Tensor &x = tensor_arg(a[0], what), &w = tensor_arg(a[1], what), &targets = tensor_arg(a[2], what);
    const double smoothing = float_arg(a[3]);
    return wrap(unlocked([&] { return linear_cross_entropy(x, w, targets, smoothing); }));
  });
}

PyObject* py_linear_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<7>("linear_attention", n, [&] {
    const char* what = "linear_attention";
    const Tensor &q = tensor_arg(a[0], what), &k = tensor_arg(a[1], what), &v = tensor_arg(a[2], what),
                 &decay = tensor_arg(a[3], what);
    const MaybeTensor state = maybe_arg(a[4], what), lengths = maybe_arg(a[5], what);
    const double scale = float_arg(a[6]);
    const Mixed r = unlocked([&] { return linear_attention(q, k, v, decay, state, lengths, scale); });
    return wrap_all({wrap(r.out), wrap(r.state)});
  });
}
PyObject* py_linear_attention_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return method<6>("linear_attention_step", n, [&] {
    const char* what = "linear_attention_step";
    const Tensor &q = tensor_arg(a[0], what), &k = tensor_arg(a[1], what), &v = tensor_arg(a[2], what),
                 &decay = tensor_arg(a[3], what), &state = tensor_arg(a[4], what);
    const double scale = float_arg(a[5]);
    return wrap(unlocked([&] { return linear_attention_step(q, k, v, decay, state, scale); }));
  });
}

#define PRATCHYA_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {PRATCHYA_METHOD(layer_norm),         PRATCHYA_METHOD(layer_norm_fwd),
                         PRATCHYA_METHOD(layer_norm_bwd),     PRATCHYA_METHOD(activation),
                         PRATCHYA_METHOD(activation_fwd),     PRATCHYA_METHOD(activation_bwd),
                         PRATCHYA_METHOD(token_logprobs),     PRATCHYA_METHOD(token_logprobs_fwd),
                         PRATCHYA_METHOD(token_logprobs_bwd), PRATCHYA_METHOD(embedding),
                         PRATCHYA_METHOD(linear_cross_entropy), PRATCHYA_METHOD(linear_attention),
                         PRATCHYA_METHOD(linear_attention_step),
                         {nullptr, nullptr, 0, nullptr}};
#undef PRATCHYA_METHOD

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_row_ops", "Row operators over libpratchya_fp8.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__row_ops(void) { return PyModule_Create(&module); }
