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
// autograd nodes
// --------------------------------------------------------------------------
// Gradients of gradients are not computed: with create_graph the results are
// differentiable into an error, as torch's once_differentiable has it.
variable_list once(variable_list&& grads, const char* what) {
  if (!at::GradMode::is_enabled()) return std::move(grads);
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

#define PRATCHYA_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {PRATCHYA_METHOD(layer_norm),         PRATCHYA_METHOD(layer_norm_fwd),
                         PRATCHYA_METHOD(layer_norm_bwd),     PRATCHYA_METHOD(activation),
                         PRATCHYA_METHOD(activation_fwd),     PRATCHYA_METHOD(activation_bwd),
                         PRATCHYA_METHOD(token_logprobs),     PRATCHYA_METHOD(token_logprobs_fwd),
                         PRATCHYA_METHOD(token_logprobs_bwd), {nullptr, nullptr, 0, nullptr}};
#undef PRATCHYA_METHOD

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_row_ops", "Row operators over libpratchya_fp8.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__row_ops(void) { return PyModule_Create(&module); }
