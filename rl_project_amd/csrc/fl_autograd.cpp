// score_tokens, layer_norm, lm_head_logprobs, qk_norm_rope and the calls on a paged
// cache as a torch extension over the C ABI (include/fl_sampler.h): the launches with their allocations, and the
// autograd nodes.  The kernels are the library's; what is here would cost more
// than the small calls' kernels in Python.  (Host time of layer_norm 255x1025,
// forward and gradients: 110 us with a Python node, which waits for the
// interpreter on the engine's own thread, 73 us so; score_tokens 1x50257 with 5
// alternatives: 20 us over ctypes, 11.6 us so.)
//
// The Python callers of score_tokens, layer_norm and lm_head_logprobs have checked
// every argument; those of the others pass theirs on, and they are checked here (in
// Python the checks of a decode step's calls take longer than its kernels).  The
// entry points come from the library that Python loaded (bind).
#include <torch/extension.h>

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <ATen/ExpandUtils.h>
#include <ATen/MemoryOverlap.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <cmath>
#include <optional>
#include <sstream>
#include <string>
#include <vector>

#include "../../include/fl_sampler.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Entry {
  decltype(&fl_last_error) last_error = nullptr;
  decltype(&fl_score_tokens) score = nullptr;
  decltype(&fl_score_workspace_bytes) score_ws = nullptr;
  decltype(&fl_score_tokens_grad) score_grad = nullptr;
  decltype(&fl_layer_norm) norm = nullptr;
  decltype(&fl_layer_norm_grad) norm_grad = nullptr;
  decltype(&fl_layer_norm_grad_workspace_bytes) norm_ws = nullptr;
  decltype(&fl_head_logprobs) head = nullptr;
  decltype(&fl_head_workspace_bytes) head_ws = nullptr;
  decltype(&fl_head_logprobs_grad) head_grad = nullptr;
  decltype(&fl_head_grad_workspace_bytes) head_grad_ws = nullptr;
  decltype(&fl_qk_norm_rope) rope = nullptr;
  decltype(&fl_qk_norm_rope_grad) rope_grad = nullptr;
  decltype(&fl_qk_norm_rope_grad_workspace_bytes) rope_grad_ws = nullptr;
  decltype(&fl_cache_write) cache_write = nullptr;
  decltype(&fl_cache_read) cache_read = nullptr;
  decltype(&fl_paged_attention) attn = nullptr;
  decltype(&fl_paged_attention_workspace_bytes) attn_ws = nullptr;
} L;

void bind(const std::vector<uintptr_t>& p) {
  TORCH_CHECK(p.size() == 18, "fl_autograd: 18 entry points expected");
  auto at = [&](size_t i, auto& f) { f = reinterpret_cast<std::decay_t<decltype(f)>>(p[i]); };
  at(0, L.last_error), at(1, L.score), at(2, L.score_ws), at(3, L.score_grad), at(4, L.norm), at(5, L.norm_grad),
      at(6, L.norm_ws), at(7, L.head), at(8, L.head_ws), at(9, L.head_grad), at(10, L.head_grad_ws),
      at(11, L.rope), at(12, L.rope_grad), at(13, L.rope_grad_ws), at(14, L.cache_write), at(15, L.cache_read), at(16, L.attn),
      at(17, L.attn_ws);
}

void check(int rc, const char* what) {
  if (rc == FL_OK) return;
  const std::string msg = std::string(what) + " failed (" + std::to_string(rc) + "): " + L.last_error();
  if (rc == FL_EINVAL) C10_THROW_ERROR(ValueError, msg);
  if (rc == FL_ENOTSUP) C10_THROW_ERROR(NotImplementedError, msg);
  C10_THROW_ERROR(Error, msg);
}

int dtype_of(at::ScalarType t) {
  return t == at::kFloat ? FL_DTYPE_F32 : t == at::kBFloat16 ? FL_DTYPE_BF16 : FL_DTYPE_F16;
}

// [rows, n] with contiguous rows (a copy where they are not)
Tensor rows_of(const Tensor& x) {
  if (x.dim() == 2 && x.is_contiguous()) return x;
  Tensor r = x.reshape({-1, x.size(-1)});
  if ((r.size(1) > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < r.size(1))) r = r.contiguous();
  return r;
}
// The head's: rows that 16-byte loads can take, and an offset of their stride
Tensor hidden_rows(const Tensor& x) {
  Tensor h = x.reshape({-1, x.size(-1)});
  if (h.stride(1) != 1 || (h.size(0) > 1 && (h.stride(0) < h.size(1) || h.stride(0) % 8 != 0 || h.stride(0) > (1 << 21))))
    h = h.contiguous();
  if (reinterpret_cast<uintptr_t>(h.data_ptr()) % 16 != 0) h = h.clone(at::MemoryFormat::Contiguous);
  return h;
}
int64_t row_stride(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

template <class T = void>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor bytes(size_t n, const Tensor& like) {
  return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}

// Results of a backward pass that has none of its own: one that is asked to
// record its graph returns results that raise when differentiated.
variable_list once(variable_list out) {
  if (!at::GradMode::is_enabled()) return out;
  for (Tensor& t : out)   // (results of leaves that need no gradient would get no node)
    if (t.defined()) t.requires_grad_(true);
  auto e = std::make_shared<torch::autograd::DelayedError>(
      "this call is differentiable once: its gradients have no gradients", static_cast<int>(out.size()));
  return (*e)(std::move(out));
}

// A backward pass under stream capture is refused, as the forward calls refuse to
// record their graph there: the engine synchronises with the streams that the
// leaves' other graphs ran on.
void refuse_capture(const char* functional) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
    C10_THROW_ERROR(Error, std::string("backward under stream capture: call ") + functional);
}

// No call has a forward-mode derivative: an input with a tangent is refused, not
// taken without it.
bool dual(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool dual(const OptTensor& t) { return t && dual(*t); }
template <class... T>
void refuse_tangents(const char* what, const T&... t) {
  if ((dual(t) || ...) && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    C10_THROW_ERROR(NotImplementedError, std::string(what) + " has no forward-mode derivative");
}
void refuse_tangents(const char* what, const variable_list& v) {
  for (const Tensor& t : v) refuse_tangents(what, t);
}

Tensor upstream(const Tensor& g) { return g.defined() ? g.contiguous() : g; }

// ---------------------------------------------------------------- layer norm
// y, and the statistics [2, rows] (mean, rstd) if asked for
std::pair<Tensor, Tensor> norm_forward(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, bool keep) {
  const Tensor x2 = rows_of(x);
  const Tensor w = weight ? weight->contiguous() : Tensor(), b = bias ? bias->contiguous() : Tensor();
  const Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  const Tensor stats = keep ? floats({2, x2.size(0)}, x) : Tensor();
  fl_norm_args a = {};
  a.struct_size = sizeof(a);
  a.dtype = dtype_of(x.scalar_type());
  a.wdtype = w.defined() ? dtype_of(w.scalar_type()) : b.defined() ? dtype_of(b.scalar_type()) : a.dtype;
  a.eps = static_cast<float>(eps);
  a.x = x2.data_ptr();
  a.rows = x2.size(0), a.dim = x2.size(1), a.ld = row_stride(x2);
  a.weight = ptr(w), a.bias = ptr(b);
  a.out = y.data_ptr(), a.out_ld = a.dim;
  if (keep) a.out_mean = ptr<float>(stats), a.out_rstd = a.out_mean + a.rows;
  const c10::DeviceGuard guard(x.device());
  check(L.norm(&a, stream_of(x)), "fl_layer_norm");
  return {y, stats};
}

// dx, dweight, dbias, each undefined where not asked for (bias_type: none)
variable_list norm_backward(const Tensor& grad, const Tensor& x, const Tensor& weight, const Tensor& stats, bool need_x,
                            bool need_w, std::optional<at::ScalarType> wtype, std::optional<at::ScalarType> bias_type) {
  const Tensor x2 = rows_of(x), g2 = rows_of(grad), w = weight.defined() ? weight.contiguous() : Tensor();
  const int64_t D = x2.size(1);
  variable_list out(3);
  if (need_x) out[0] = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  if (need_w) out[1] = at::empty({D}, w.options());
  if (bias_type) out[2] = at::empty({D}, x.options().dtype(*bias_type));
  fl_norm_grad_args a = {};
  a.struct_size = sizeof(a);
  a.dtype = dtype_of(x.scalar_type());
  a.wdtype = wtype ? dtype_of(*wtype) : a.dtype;
  a.x = x2.data_ptr();
  a.rows = x2.size(0), a.dim = D, a.ld = row_stride(x2);
  a.weight = ptr(w);
  a.grad = g2.data_ptr(), a.grad_ld = row_stride(g2);
  a.mean = ptr<float>(stats), a.rstd = a.mean + a.rows;
  a.out_dx = ptr(out[0]), a.out_ld = D;
  a.out_dweight = ptr(out[1]), a.out_dbias = ptr(out[2]);
  if (a.out_dx == nullptr && a.out_dweight == nullptr && a.out_dbias == nullptr) return out;
  Tensor ws;
  if (a.out_dweight != nullptr || a.out_dbias != nullptr) {
    size_t n = 0;
    check(L.norm_ws(a.rows, D, a.dtype, &n), "fl_layer_norm_grad_workspace_bytes");
    ws = bytes(n, x);
    a.workspace = ws.data_ptr(), a.workspace_bytes = static_cast<int64_t>(n);
  }
  const c10::DeviceGuard guard(x.device());
  check(L.norm_grad(&a, stream_of(x)), "fl_layer_norm_grad");
  return out;
}

std::optional<at::ScalarType> type_of(const OptTensor& t) {
  return t ? std::optional<at::ScalarType>(t->scalar_type()) : std::nullopt;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    auto [y, stats] = norm_forward(x, weight, bias, eps, true);
    ctx->save_for_backward({x, weight ? *weight : Tensor()});
    ctx->saved_data["stats"] = stats;   // (this node's own: no caller sees or changes it)
    ctx->saved_data["bias"] = bias ? static_cast<int64_t>(bias->scalar_type()) : int64_t{-1};
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_capture("layer_norm_backward");
    refuse_tangents("layer_norm_backward", grads);
    const auto saved = ctx->get_saved_variables();
    const int64_t b = ctx->saved_data["bias"].toInt();
    const auto btype = b >= 0 ? std::optional<at::ScalarType>(static_cast<at::ScalarType>(b)) : std::nullopt;
    const bool has_w = saved[1].defined();
    variable_list out;
    {
      const at::NoGradGuard no_grad;
      // (the edges are those of the tensors given: without a weight the bias is the second)
      const bool need_b = btype && ctx->needs_input_grad(has_w ? 2 : 1);
      out = norm_backward(grads[0], saved[0], saved[1], ctx->saved_data["stats"].toTensor(), ctx->needs_input_grad(0),
                          has_w && ctx->needs_input_grad(1), has_w ? std::optional(saved[1].scalar_type()) : btype,
                          need_b ? btype : std::nullopt);
    }
    out.emplace_back();   // (eps)
    return once(std::move(out));
  }
};

// ---------------------------------------------------------------- scores
// logprob, entropy, lse, rank, top ids, top logprobs, saved: undefined where not
// asked for
variable_list score_forward(const Tensor& logits, const OptTensor& tokens, int64_t top_k, bool entropy, bool lse, bool rank,
                            int64_t ignore_index, bool save) {
  const Tensor x = rows_of(logits);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const auto opt = logits.options();
  variable_list out(7);
  if (tokens) out[0] = floats(lead, x);
  if (entropy) out[1] = floats(lead, x);
  if (lse) out[2] = floats(lead, x);
  if (rank) out[3] = at::empty(lead, opt.dtype(at::kInt));
  if (top_k > 0) {
    std::vector<int64_t> top(lead.begin(), lead.end());
    top.push_back(top_k);
    out[4] = at::empty(top, opt.dtype(at::kLong));
    out[5] = floats(top, x);
  }
  if (save) out[6] = floats({x.size(0), 4}, x);
  fl_score_args a = {};
  a.struct_size = sizeof(a);
  a.dtype = dtype_of(x.scalar_type());
  a.logits = x.data_ptr();
  a.rows = x.size(0), a.vocab = x.size(1), a.ld = row_stride(x);
  a.tokens = tokens ? ptr<int64_t>(*tokens) : nullptr;
  a.ignore_index = ignore_index, a.top_k = top_k;
  a.out_logprob = ptr<float>(out[0]), a.out_entropy = ptr<float>(out[1]), a.out_lse = ptr<float>(out[2]);
  a.out_rank = ptr<int32_t>(out[3]), a.out_top_ids = ptr<int64_t>(out[4]), a.out_top_logprobs = ptr<float>(out[5]);
  a.out_saved = ptr<float>(out[6]);
  size_t n = 0;
  check(L.score_ws(a.rows, a.vocab, top_k, &n), "fl_score_workspace_bytes");
  Tensor ws;
  if (n > 0) {
    ws = bytes(n, x);
    a.workspace = ws.data_ptr(), a.workspace_bytes = static_cast<int64_t>(n);
  }
  const c10::DeviceGuard guard(x.device());
  check(L.score(&a, stream_of(x)), "fl_score_tokens");
  return out;
}

Tensor score_backward(const Tensor& logits, const Tensor& tokens, const Tensor& saved, const Tensor& ga, const Tensor& gb,
                      const Tensor& gc, int64_t ignore_index) {
  const Tensor x = rows_of(logits);
  const Tensor out = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
  fl_score_grad_args a = {};
  a.struct_size = sizeof(a);
  a.dtype = dtype_of(x.scalar_type());
  a.logits = x.data_ptr();
  a.rows = x.size(0), a.vocab = x.size(1), a.ld = row_stride(x);
  a.tokens = ptr<int64_t>(tokens);
  a.ignore_index = ignore_index;
  a.saved = ptr<float>(saved);
  a.grad_logprob = ptr<float>(ga), a.grad_entropy = ptr<float>(gb), a.grad_lse = ptr<float>(gc);
  a.out_grad = out.data_ptr(), a.out_ld = a.vocab;
  const c10::DeviceGuard guard(x.device());
  check(L.score_grad(&a, stream_of(x)), "fl_score_tokens_grad");
  return out;
}

// What a node of up to three differentiable results keeps beside its tensors
void keep(AutogradContext* ctx, const Tensor& saved, bool lp, bool ent, bool lse, int64_t ignore_index) {
  ctx->set_materialize_grads(false);
  ctx->saved_data["saved"] = saved;   // (this node's own: no caller sees or changes it)
  ctx->saved_data["has"] = (lp ? 1 : 0) | (ent ? 2 : 0) | (lse ? 4 : 0);
  ctx->saved_data["ignore"] = ignore_index;
}
// The upstream gradients of logprob, entropy, lse; false if there is none
bool upstreams(AutogradContext* ctx, const variable_list& grads, Tensor (&g)[3]) {
  const int64_t has = ctx->saved_data["has"].toInt();
  bool any = false;
  for (size_t i = 0, k = 0; i < 3; ++i)
    if (has & (1 << i)) {
      g[i] = upstream(grads[k++]);
      any = any || g[i].defined();
    }
  return any;
}

// Results: those asked for, in the order logprob, entropy, lse, rank, top ids,
// top logprobs.
struct Score : torch::autograd::Function<Score> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& tokens, int64_t top_k, bool entropy,
                               bool lse, bool rank, int64_t ignore_index) {
    const variable_list r = score_forward(logits, tokens, top_k, entropy, lse, rank, ignore_index, true);
    ctx->save_for_backward({logits, tokens ? *tokens : Tensor()});
    keep(ctx, r[6], tokens.has_value(), entropy, lse, ignore_index);
    variable_list out, plain;
    for (size_t i = 0; i < 6; ++i)
      if (r[i].defined()) {
        out.push_back(r[i]);
        if (i >= 3) plain.push_back(r[i]);
      }
    ctx->mark_non_differentiable(plain);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_capture("score_tokens_backward");
    refuse_tangents("score_tokens_backward", grads);
    const auto kept = ctx->get_saved_variables();
    Tensor g[3];
    variable_list out(7);
    if (!upstreams(ctx, grads, g)) return out;
    {
      const at::NoGradGuard no_grad;
      out[0] = score_backward(kept[0], kept[1], ctx->saved_data["saved"].toTensor(), g[0], g[1], g[2],
                              ctx->saved_data["ignore"].toInt());
    }
    return once(std::move(out));
  }
};

// The gradient of a statistic that another kernel computed: value (float32, the
// logits' leading dimensions) is passed on, bit for bit, as the tokens'
// log-probability or, without tokens, as the entropy.  The backward pass takes
// the softmax's statistics by itself (one more read of the logits).
struct Stat : torch::autograd::Function<Stat> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& value, const OptTensor& tokens,
                        int64_t ignore_index) {
    ctx->save_for_backward({logits, tokens ? *tokens : Tensor()});
    ctx->saved_data["ignore"] = ignore_index;
    if (!tokens) ctx->saved_data["entropy"] = value.clone();   // (the result may be changed)
    return value.detach();
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_capture("score_tokens_backward");
    refuse_tangents("score_tokens_backward", grads);
    const auto kept = ctx->get_saved_variables();
    const Tensor &x = kept[0], &tokens = kept[1], none;
    const int64_t ignore = ctx->saved_data["ignore"].toInt();
    const bool lp = tokens.defined();
    variable_list out(4);
    {
      const at::NoGradGuard no_grad;
      const Tensor g = upstream(grads[0]), saved = score_forward(x, std::nullopt, 0, !lp, false, false, ignore, true)[6];
      // (the value's own entropy: NaN, and so the gradient, where a logit is -inf)
      if (!lp) saved.select(1, 2).copy_(ctx->saved_data["entropy"].toTensor().reshape({-1}));
      out[0] = score_backward(x, tokens, saved, lp ? g : none, lp ? none : g, none, ignore);
    }
    return once(std::move(out));
  }
};

// ---------------------------------------------------------------- head
// logprob, entropy, lse, saved: undefined where not asked for
variable_list head_forward(const Tensor& hidden, const Tensor& weight, const OptTensor& tokens, bool entropy, bool lse,
                           int64_t ignore_index, bool save) {
  const Tensor h = hidden_rows(hidden);
  const auto lead = hidden.sizes().slice(0, hidden.dim() - 1);
  variable_list out(4);
  if (tokens) out[0] = floats(lead, h);
  if (entropy) out[1] = floats(lead, h);
  if (lse) out[2] = floats(lead, h);
  if (save) out[3] = floats({h.size(0), 4}, h);
  fl_head_args a = {};
  a.struct_size = sizeof(a);
  a.dtype = FL_DTYPE_BF16;
  a.hidden = h.data_ptr(), a.weight = weight.data_ptr();
  a.rows = h.size(0), a.dim = h.size(1), a.vocab = weight.size(0), a.ld_hidden = row_stride(h);
  a.tokens = tokens ? ptr<int64_t>(*tokens) : nullptr;
  a.ignore_index = ignore_index;
  a.out_logprob = ptr<float>(out[0]), a.out_entropy = ptr<float>(out[1]), a.out_lse = ptr<float>(out[2]);
  a.out_saved = ptr<float>(out[3]);
  size_t n = 0;
  check(L.head_ws(a.rows, a.vocab, &n), "fl_head_workspace_bytes");
  const Tensor ws = bytes(n, h);
  a.workspace = ws.data_ptr(), a.workspace_bytes = static_cast<int64_t>(n);
  const c10::DeviceGuard guard(h.device());
  check(L.head(&a, stream_of(h)), "fl_head_logprobs");
  return out;
}

// dhidden, dweight: undefined where not asked for
variable_list head_backward(const Tensor& hidden, const Tensor& weight, const Tensor& tokens, const Tensor& saved, const Tensor& ga,
                            const Tensor& gb, const Tensor& gc, int64_t ignore_index, bool need_h, bool need_w) {
  const Tensor h = hidden_rows(hidden);
  variable_list out(2);
  if (need_h) out[0] = at::empty(hidden.sizes(), hidden.options().memory_format(at::MemoryFormat::Contiguous));
  if (need_w)   // (no rows: no sums)
    out[1] = h.size(0) == 0 ? at::zeros(weight.sizes(), weight.options()) : at::empty(weight.sizes(), weight.options());
  if (!need_h && !need_w) return out;
  fl_head_grad_args a = {};
  a.struct_size = sizeof(a);
  a.dtype = FL_DTYPE_BF16;
  a.hidden = h.data_ptr(), a.weight = weight.data_ptr();
  a.rows = h.size(0), a.dim = h.size(1), a.vocab = weight.size(0), a.ld_hidden = row_stride(h);
  a.tokens = ptr<int64_t>(tokens);
  a.ignore_index = ignore_index;
  a.saved = ptr<float>(saved);
  a.grad_logprob = ptr<float>(ga), a.grad_entropy = ptr<float>(gb), a.grad_lse = ptr<float>(gc);
  a.out_dhidden = ptr(out[0]), a.out_dweight = ptr(out[1]);
  size_t n = 0;
  check(L.head_grad_ws(a.rows, a.dim, a.vocab, need_h ? 1 : 0, &n), "fl_head_grad_workspace_bytes");
  const Tensor ws = bytes(n, h);
  a.workspace = ws.data_ptr(), a.workspace_bytes = static_cast<int64_t>(n);
  const c10::DeviceGuard guard(h.device());
  check(L.head_grad(&a, stream_of(h)), "fl_head_logprobs_grad");
  return out;
}

// Results: those asked for, in the order logprob, entropy, lse.
struct Head : torch::autograd::Function<Head> {
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const OptTensor& tokens,
                               bool entropy, bool lse, int64_t ignore_index) {
    const variable_list r = head_forward(hidden, weight, tokens, entropy, lse, ignore_index, true);
    ctx->save_for_backward({hidden, weight, tokens ? *tokens : Tensor()});
    keep(ctx, r[3], tokens.has_value(), entropy, lse, ignore_index);
    variable_list out;
    for (size_t i = 0; i < 3; ++i)
      if (r[i].defined()) out.push_back(r[i]);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_capture("lm_head_logprobs_backward");
    refuse_tangents("lm_head_logprobs_backward", grads);
    const auto kept = ctx->get_saved_variables();
    Tensor g[3];
    if (!upstreams(ctx, grads, g)) return variable_list(6);
    variable_list out;
    {
      const at::NoGradGuard no_grad;
      out = head_backward(kept[0], kept[1], kept[2], ctx->saved_data["saved"].toTensor(), g[0], g[1], g[2],
                          ctx->saved_data["ignore"].toInt(), ctx->needs_input_grad(0), ctx->needs_input_grad(1));
    }
    out.resize(6);
    return once(std::move(out));
  }
};

// ---------------------------------------------------------------- checks
template <class... T>
std::string text(const T&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  return s.str();
}
#define VALUE_CHECK(cond, ...) \
  if (!(cond)) C10_THROW_ERROR(ValueError, text(__VA_ARGS__))
#define SUPPORT_CHECK(cond, ...) \
  if (!(cond)) C10_THROW_ERROR(NotImplementedError, text(__VA_ARGS__))

bool is_row_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
bool same_lead(const Tensor& a, const Tensor& b, int64_t n) { return a.sizes().slice(0, n) == b.sizes().slice(0, n); }
bool graded(const Tensor& t) { return t.requires_grad(); }
bool graded(const OptTensor& t) { return t && t->requires_grad(); }

// What qk_norm_rope and its backward take; returns positions and inv_freq as the
// kernels read them.
std::pair<Tensor, Tensor> check_rope(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& inv_freq,
                                     const OptTensor& qw, const OptTensor& kw, bool norm) {
  for (const Tensor* t : {&q, &k}) {
    const char* name = t == &q ? "q" : "k";
    VALUE_CHECK(t->is_cuda(), name, " must be on a ROCm device (no CPU fallback)");
    SUPPORT_CHECK(is_row_type(t->scalar_type()), name, " dtype ", t->scalar_type(), " is not supported (float32, bfloat16, float16)");
  }
  VALUE_CHECK(q.dim() >= 3 && k.dim() == q.dim() && same_lead(q, k, q.dim() - 2) && q.size(-1) == k.size(-1),
              "q [..., heads, dim] and k [..., kv_heads, dim] do not match: ", q.sizes(), ", ", k.sizes());
  VALUE_CHECK(k.scalar_type() == q.scalar_type() && k.device() == q.device(), "q and k must share a dtype and a device");
  const int64_t D = q.size(-1);
  VALUE_CHECK(D >= 2 && D % 2 == 0, "the head dimension must be even and at least 2, not ", D);
  VALUE_CHECK(q.size(-2) >= 1 && k.size(-2) >= 1, "q and k need at least one head");
  VALUE_CHECK((positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong) && positions.device() == q.device(),
              "positions must be int32 or int64 on ", q.device());
  VALUE_CHECK(inv_freq.dim() == 1 && inv_freq.device() == q.device() &&
                  (inv_freq.scalar_type() == at::kDouble || inv_freq.scalar_type() == at::kFloat) && 2 * inv_freq.size(0) <= D,
              "inv_freq must be float64 or float32, of at most ", D / 2, " values, on ", q.device());
  VALUE_CHECK(norm || (!qw && !kw), "weights belong to the norm: give eps");
  for (const OptTensor* w : {&qw, &kw}) {
    if (!*w) continue;
    const char* name = w == &qw ? "q_weight" : "k_weight";
    VALUE_CHECK((*w)->dim() == 1 && (*w)->size(0) == D && (*w)->device() == q.device(), name, " must be [", D, "] on ", q.device());
    SUPPORT_CHECK((*w)->scalar_type() == q.scalar_type() || (*w)->scalar_type() == at::kFloat, name, " dtype ", (*w)->scalar_type(),
                  " is neither q's nor float32");
  }
  SUPPORT_CHECK(!qw || !kw || qw->scalar_type() == kw->scalar_type(), "q_weight and k_weight must share a dtype");
  const auto lead = q.sizes().slice(0, q.dim() - 2);
  Tensor p = positions;
  if (p.sizes() != lead) {
    VALUE_CHECK(at::is_expandable_to(p.sizes(), lead), "positions ", p.sizes(), " do not expand to ", lead);
    p = p.expand(lead);
  }
  const at::NoGradGuard no_grad;
  return {p.contiguous(), inv_freq.to(at::kDouble).contiguous()};
}

void check_grad_of(const OptTensor& g, const Tensor& x, const char* name) {
  VALUE_CHECK(!g || (g->sizes() == x.sizes() && g->scalar_type() == x.scalar_type() && g->device() == x.device()), name,
              " must match its input in shape, dtype and device");
}

void check_cache(const Tensor& k, const Tensor& v, const OptTensor& ks, const OptTensor& vs) {
  VALUE_CHECK(k.is_cuda(), "the cache must be on a ROCm device (no CPU fallback)");
  VALUE_CHECK(k.dim() == 4 && v.dim() == 4 && v.size(0) == k.size(0) && v.size(1) == k.size(1) && v.size(2) == k.size(3) &&
                  v.size(3) == k.size(2),
              "k [pages, heads, page_size, dim] and v [pages, heads, dim, page_size] do not match: ", k.sizes(), ", ", v.sizes());
  const auto t = k.scalar_type();
  SUPPORT_CHECK(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat8_e4m3fn, "cache dtype ", t,
                " is not supported (bfloat16, float16, float8_e4m3fn)");
  VALUE_CHECK(v.scalar_type() == t && v.device() == k.device() && k.is_contiguous() && v.is_contiguous(),
              "k and v must share a dtype and a device and be contiguous");
  const int64_t S = k.size(2), D = k.size(3);
  VALUE_CHECK(S == 16 || S == 32 || S == 64 || S == 128, "page_size ", S, " is none of 16, 32, 64, 128");
  VALUE_CHECK(k.size(0) >= 1 && k.size(1) >= 1 && D >= 8 && D % 8 == 0 && D <= FL_CACHE_MAX_DIM, k.size(0), " pages, ", k.size(1),
              " heads, dim ", D, ": at least one of each, dim a multiple of 8 up to ", FL_CACHE_MAX_DIM);
  for (const OptTensor* s : {&ks, &vs}) {
    if (t != at::kFloat8_e4m3fn) {
      VALUE_CHECK(!*s, "scales belong to a float8_e4m3fn cache");
      continue;
    }
    VALUE_CHECK(*s && (*s)->scalar_type() == at::kByte && (*s)->sizes() == k.sizes().slice(0, 3) && (*s)->device() == k.device() &&
                    (*s)->is_contiguous(),
                "a float8_e4m3fn cache needs k_scale and v_scale: contiguous uint8 ", k.sizes().slice(0, 3));
  }
}

void check_tokens(const Tensor& ck, const Tensor& table, const Tensor& lengths, const OptTensor& starts, int64_t rows) {
  VALUE_CHECK(table.dim() == 2 && table.scalar_type() == at::kInt && table.device() == ck.device() &&
                  (table.size(1) <= 1 || table.stride(1) == 1),
              "table must be int32 [B, width] on ", ck.device(), ", its rows contiguous");
  const int64_t B = table.size(0);
  VALUE_CHECK(lengths.dim() == 1 && lengths.size(0) == B && lengths.scalar_type() == at::kInt && lengths.device() == ck.device() &&
                  lengths.is_contiguous(),
              "lengths must be contiguous int32 [", B, "] on ", ck.device());
  if (!starts) {
    VALUE_CHECK(rows == 0 || (B > 0 && rows % B == 0), rows, " tokens are not as many for each of ", B, " sequences: give starts");
  } else
    VALUE_CHECK(starts->dim() == 1 && starts->size(0) == B + 1 && starts->scalar_type() == at::kInt && starts->device() == ck.device() &&
                    starts->is_contiguous(),
                "starts must be contiguous int32 [", B + 1, "] on ", ck.device());
}

int64_t lead_rows(const Tensor& x) {
  int64_t n = 1;
  for (int64_t i = 0; i + 2 < x.dim(); ++i) n *= x.size(i);
  return n;
}

void no_gradient(const char* what, bool any) {
  if (any && at::GradMode::is_enabled())
    C10_THROW_ERROR(Error, std::string(what) + " records no gradient: call it under torch.no_grad(), or detach what requires one");
}

// A tensor that a call writes through its pointer: what autograd saved of it is out of date.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(const OptTensor& t) {
  if (t) written(*t);
}

// ---------------------------------------------------------------- norms and rotation
// [tokens, heads, dim] whose last dimension is contiguous (a copy where it is not,
// or where the leading dimensions do not fold)
Tensor heads_of(const Tensor& x) {
  Tensor r = x.dim() == 3 ? x : x.reshape({-1, x.size(-2), x.size(-1)});
  bool fine = r.size(2) <= 1 || r.stride(2) == 1;
  for (int i = 0; i < 2; ++i) fine = fine && (r.size(i) <= 1 || r.stride(i) >= 0);
  return fine ? r : r.contiguous();
}

struct RopeSettings {
  double eps, gain;
  bool norm, interleaved;
};

// The arguments that both passes share; q2, k2: [tokens, heads, dim], or undefined
// for a side that has no part in the call.
fl_rope_args rope_args(const Tensor& q2, const Tensor& k2, const Tensor& qw, const Tensor& kw, const Tensor& positions,
                       const Tensor& inv_freq, const RopeSettings& s) {
  const Tensor& any = q2.defined() ? q2 : k2;
  fl_rope_args a = {};
  a.struct_size = sizeof(a);
  a.dtype = dtype_of(any.scalar_type());
  a.wdtype = qw.defined() ? dtype_of(qw.scalar_type()) : kw.defined() ? dtype_of(kw.scalar_type()) : a.dtype;
  a.flags = (s.interleaved ? FL_ROPE_INTERLEAVED : 0) | (positions.scalar_type() == at::kInt ? FL_ROPE_POSITIONS32 : 0);
  a.tokens = any.size(0), a.dim = any.size(2), a.rotated = 2 * inv_freq.size(0);
  if (q2.defined()) a.q = q2.data_ptr(), a.heads = q2.size(1), a.q_ld = q2.stride(0), a.q_hs = q2.stride(1);
  if (k2.defined()) a.k = k2.data_ptr(), a.kv_heads = k2.size(1), a.k_ld = k2.stride(0), a.k_hs = k2.stride(1);
  a.positions = positions.data_ptr();
  a.inv_freq = ptr<double>(inv_freq);
  a.q_weight = ptr(qw), a.k_weight = ptr(kw);
  a.eps = static_cast<float>(s.eps), a.gain = static_cast<float>(s.gain), a.norm = s.norm ? 1 : 0;
  return a;
}

variable_list rope_forward(const Tensor& q, const Tensor& k, const OptTensor& qw, const OptTensor& kw, const Tensor& positions,
                           const Tensor& inv_freq, const RopeSettings& s) {
  const Tensor q2 = heads_of(q), k2 = heads_of(k), w1 = qw ? qw->contiguous() : Tensor(), w2 = kw ? kw->contiguous() : Tensor();
  variable_list out{at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous)),
                    at::empty(k.sizes(), k.options().memory_format(at::MemoryFormat::Contiguous))};
  fl_rope_args a = rope_args(q2, k2, w1, w2, positions, inv_freq, s);
  a.out_q = out[0].data_ptr(), a.out_k = out[1].data_ptr();
  const c10::DeviceGuard guard(q.device());
  check(L.rope(&a, stream_of(q)), "fl_qk_norm_rope");
  return out;
}

// dq, dk, dwq, dwk: undefined where not asked for, and for a side without an
// upstream gradient
variable_list rope_backward(const Tensor& gq, const Tensor& gk, const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw,
                            const Tensor& positions, const Tensor& inv_freq, const RopeSettings& s, const bool (&need)[4]) {
  variable_list out(4);
  Tensor q2, k2, g1, g2;
  if (gq.defined() && (need[0] || need[2])) q2 = heads_of(q), g1 = gq.contiguous();
  if (gk.defined() && (need[1] || need[3])) k2 = heads_of(k), g2 = gk.contiguous();
  if (!q2.defined() && !k2.defined()) return out;
  const Tensor w1 = qw.defined() ? qw.contiguous() : Tensor(), w2 = kw.defined() ? kw.contiguous() : Tensor();
  fl_rope_grad_args a = {};
  a.struct_size = sizeof(a);
  a.fwd = rope_args(q2, k2, w1, w2, positions, inv_freq, s);
  const auto like = [](const Tensor& x) { return at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous)); };
  if (q2.defined() && need[0]) out[0] = like(q);
  if (k2.defined() && need[1]) out[1] = like(k);
  if (q2.defined() && need[2]) out[2] = at::empty({a.fwd.dim}, w1.options());
  if (k2.defined() && need[3]) out[3] = at::empty({a.fwd.dim}, w2.options());
  a.grad_q = ptr(g1), a.grad_k = ptr(g2);
  a.fwd.out_q = ptr(out[0]), a.fwd.out_k = ptr(out[1]), a.out_dwq = ptr(out[2]), a.out_dwk = ptr(out[3]);
  Tensor ws;
  if (out[2].defined() || out[3].defined()) {
    size_t n = 0;
    check(L.rope_grad_ws(a.fwd.tokens, a.fwd.dim, &n), "fl_qk_norm_rope_grad_workspace_bytes");
    ws = bytes(n, positions);
    a.workspace = ws.data_ptr(), a.workspace_bytes = static_cast<int64_t>(n);
  }
  const c10::DeviceGuard guard(positions.device());
  check(L.rope_grad(&a, stream_of(positions)), "fl_qk_norm_rope_grad");
  return out;
}

struct Rope : torch::autograd::Function<Rope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const OptTensor& qw, const OptTensor& kw,
                               const Tensor& positions, const Tensor& inv_freq, double eps, double gain, bool norm, bool interleaved) {
    const variable_list out = rope_forward(q, k, qw, kw, positions, inv_freq, {eps, gain, norm, interleaved});
    ctx->set_materialize_grads(false);
    // (a rotation alone needs its inputs' shapes, which its gradients have)
    ctx->save_for_backward({norm ? q : Tensor(), norm ? k : Tensor(), qw ? *qw : Tensor(), kw ? *kw : Tensor(), positions, inv_freq});
    ctx->saved_data["eps"] = eps, ctx->saved_data["gain"] = gain;
    ctx->saved_data["norm"] = norm, ctx->saved_data["interleaved"] = interleaved;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_capture("qk_norm_rope_backward");
    refuse_tangents("qk_norm_rope_backward", grads);
    const auto kept = ctx->get_saved_variables();
    auto& d = ctx->saved_data;
    // (the edges are those of the tensors given)
    const bool has1 = kept[2].defined(), has2 = kept[3].defined();
    const bool need[4] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), has1 && ctx->needs_input_grad(2),
                          has2 && ctx->needs_input_grad(has1 ? 3 : 2)};
    variable_list out;
    {
      const at::NoGradGuard no_grad;
      const bool norm = d["norm"].toBool();
      const Tensor gq = upstream(grads[0]), gk = upstream(grads[1]);
      out = rope_backward(gq, gk, norm ? kept[0] : gq, norm ? kept[1] : gk, kept[2], kept[3], kept[4], kept[5],
                          {d["eps"].toDouble(), d["gain"].toDouble(), norm, d["interleaved"].toBool()}, need);
    }
    out.resize(10);
    return once(std::move(out));
  }
};

// ---------------------------------------------------------------- the paged cache
struct CacheTensors {
  Tensor k, v;
  OptTensor k_scale, v_scale;
};

void set_cache(fl_cache& c, const CacheTensors& t) {
  c.k = t.k.data_ptr(), c.v = t.v.data_ptr();
  c.k_scale = t.k_scale ? ptr<uint8_t>(*t.k_scale) : nullptr, c.v_scale = t.v_scale ? ptr<uint8_t>(*t.v_scale) : nullptr;
  c.pages = t.k.size(0), c.heads = t.k.size(1), c.page_size = t.k.size(2), c.dim = t.k.size(3);
  c.dtype = t.k.scalar_type() == at::kFloat8_e4m3fn ? FL_DTYPE_E4M3 : dtype_of(t.k.scalar_type());
}
void set_rows(fl_cache_rows& r, const Tensor& table, const Tensor& lengths, const OptTensor& starts, int64_t tokens) {
  r.table = ptr<int32_t>(table), r.lengths = ptr<int32_t>(lengths), r.starts = starts ? ptr<int32_t>(*starts) : nullptr;
  r.seqs = lengths.size(0), r.tokens = tokens, r.table_width = table.size(1), r.table_ld = table.stride(0);
}

void cache_call(const CacheTensors& c, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lengths,
                const OptTensor& starts, bool write) {
  const Tensor k2 = write ? heads_of(k) : k, v2 = write ? heads_of(v) : v;
  fl_cache_args a = {};
  a.struct_size = sizeof(a);
  a.dtype = dtype_of(k2.scalar_type());
  set_cache(a.cache, c);
  set_rows(a.rows, table, lengths, starts, k2.size(0));
  a.k = k2.data_ptr(), a.v = v2.data_ptr();
  a.k_ld = k2.stride(0), a.k_hs = k2.stride(1), a.v_ld = v2.stride(0), a.v_hs = v2.stride(1);
  const c10::DeviceGuard guard(k2.device());
  if (write) check(L.cache_write(&a, stream_of(k2)), "fl_cache_write");
  else check(L.cache_read(&a, stream_of(k2)), "fl_cache_read");
}

// out, lse (undefined if not asked for); `into`: where out goes
variable_list attention(const CacheTensors& c, const Tensor& q, const Tensor& table, const Tensor& lengths, const OptTensor& starts,
                        double scale, double softcap, int64_t window, int64_t sinks, const OptTensor& into, bool want_lse) {
  Tensor q2 = heads_of(q);
  const bool odd = reinterpret_cast<uintptr_t>(q2.data_ptr()) % 16 != 0 || (q2.size(0) > 1 && q2.stride(0) % 8 != 0) ||
                   (q2.size(1) > 1 && q2.stride(1) % 8 != 0);
  if (odd) q2 = q2.clone(at::MemoryFormat::Contiguous);
  variable_list out(2);
  out[0] = into ? *into : at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  const Tensor o2 = into ? *into : out[0].view({q2.size(0), q2.size(1), q2.size(2)});
  if (want_lse) out[1] = floats(q.sizes().slice(0, q.dim() - 1), q);
  fl_attn_args a = {};
  a.struct_size = sizeof(a);
  a.dtype = dtype_of(q.scalar_type());
  set_cache(a.cache, c);
  set_rows(a.rows, table, lengths, starts, q2.size(0));
  const auto stride = [](const Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : int64_t{0}; };
  a.q = q2.data_ptr(), a.q_heads = q2.size(1), a.q_ld = stride(q2, 0), a.q_hs = stride(q2, 1);
  a.out = o2.data_ptr(), a.out_ld = stride(o2, 0), a.out_hs = stride(o2, 1);
  a.out_lse = ptr<float>(out[1]);
  a.scale = static_cast<float>(scale), a.softcap = static_cast<float>(softcap), a.window = window, a.sinks = sinks;
  size_t n = 0;
  check(L.attn_ws(&a, &n), "fl_paged_attention_workspace_bytes");
  const c10::DeviceGuard guard(q.device());
  Tensor ws;
  if (n > 0) {
    ws = bytes(n, q);
    a.workspace = ws.data_ptr(), a.workspace_bytes = static_cast<int64_t>(n);
  }
  check(L.attn(&a, stream_of(q)), "fl_paged_attention");
  return out;
}

// Undefined tensors as None
std::vector<OptTensor> or_none(const variable_list& v) {
  std::vector<OptTensor> out;
  for (const Tensor& t : v) out.push_back(t.defined() ? OptTensor(t) : std::nullopt);
  return out;
}
Tensor or_undefined(const OptTensor& t) { return t ? *t : Tensor(); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  using release = py::call_guard<py::gil_scoped_release>;
  m.def("bind", &bind);
  // (differentiable)
  m.def("layer_norm", [](const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
    refuse_tangents("layer_norm", x, w, b);
    return LayerNorm::apply(x, w, b, eps);
  }, release());
  m.def("score", [](const Tensor& x, const OptTensor& t, int64_t k, bool e, bool l, bool r, int64_t ii) {
    refuse_tangents("score_tokens", x);
    return Score::apply(x, t, k, e, l, r, ii);
  }, release());
  m.def("stat", [](const Tensor& x, const Tensor& value, const OptTensor& t, int64_t ii) { return Stat::apply(x, value, t, ii); },
        release());
  m.def("head", [](const Tensor& h, const Tensor& w, const OptTensor& t, bool e, bool l, int64_t ii) {
    refuse_tangents("lm_head_logprobs", h, w);
    return Head::apply(h, w, t, e, l, ii);
  }, release());
  // (the launches alone)
  m.def("norm_forward", [](const Tensor& x, const OptTensor& w, const OptTensor& b, double eps, bool keep) {
    refuse_tangents("layer_norm", x, w, b);
    const at::NoGradGuard no_grad;
    auto [y, stats] = norm_forward(x, w, b, eps, keep);
    return or_none({y, stats});
  }, release());
  m.def("norm_backward", [](const Tensor& g, const Tensor& x, const OptTensor& w, const OptTensor& b, const Tensor& stats, bool nx,
                            bool nw, bool nb) {
    refuse_tangents("layer_norm_backward", g, x, w, stats);
    const at::NoGradGuard no_grad;
    return or_none(norm_backward(g, x, or_undefined(w), stats, nx, nw && w, w ? type_of(w) : type_of(b),
                                 nb ? type_of(b) : std::nullopt));
  }, release());
  m.def("score_forward", [](const Tensor& x, const OptTensor& t, int64_t k, bool e, bool l, bool r, int64_t ii, bool save) {
    refuse_tangents("score_tokens", x);
    const at::NoGradGuard no_grad;
    return or_none(score_forward(x, t, k, e, l, r, ii, save));
  }, release());
  m.def("score_backward", [](const Tensor& x, const OptTensor& t, const Tensor& saved, const OptTensor& ga, const OptTensor& gb,
                             const OptTensor& gc, int64_t ii) {
    refuse_tangents("score_tokens_backward", x, saved, ga, gb, gc);
    const at::NoGradGuard no_grad;
    return score_backward(x, or_undefined(t), saved, or_undefined(ga), or_undefined(gb), or_undefined(gc), ii);
  }, release());
  m.def("head_forward", [](const Tensor& h, const Tensor& w, const OptTensor& t, bool e, bool l, int64_t ii, bool save) {
    refuse_tangents("lm_head_logprobs", h, w);
    const at::NoGradGuard no_grad;
    return or_none(head_forward(h, w, t, e, l, ii, save));
  }, release());
  m.def("head_backward", [](const Tensor& h, const Tensor& w, const OptTensor& t, const Tensor& saved, const OptTensor& ga,
                            const OptTensor& gb, const OptTensor& gc, int64_t ii, bool nh, bool nw) {
    refuse_tangents("lm_head_logprobs_backward", h, w, saved, ga, gb, gc);
    const at::NoGradGuard no_grad;
    return or_none(head_backward(h, w, or_undefined(t), saved, or_undefined(ga), or_undefined(gb), or_undefined(gc), ii, nh, nw));
  }, release());
  m.def("qk_norm_rope", [](const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& inv_freq, const OptTensor& qw,
                           const OptTensor& kw, std::optional<double> eps, bool inter, double gain) -> variable_list {
    const auto [pos, freq] = check_rope(q, k, positions, inv_freq, qw, kw, eps.has_value());
    no_gradient("qk_norm_rope for inv_freq", graded(inv_freq));
    refuse_tangents("qk_norm_rope", q, k, qw, kw, inv_freq);
    if (at::GradMode::is_enabled() && (graded(q) || graded(k) || graded(qw) || graded(kw))) {
      if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
        C10_THROW_ERROR(Error, "qk_norm_rope does not record its autograd graph under stream capture: call it under "
                               "torch.no_grad(), then qk_norm_rope_backward");
      return Rope::apply(q, k, qw, kw, pos, freq, eps.value_or(0.0), gain, eps.has_value(), inter);
    }
    const at::NoGradGuard no_grad;
    return rope_forward(q, k, qw, kw, pos, freq, {eps.value_or(0.0), gain, eps.has_value(), inter});
  }, release());
  m.def("qk_norm_rope_backward", [](const OptTensor& gq, const OptTensor& gk, const Tensor& q, const Tensor& k, const Tensor& positions,
                                    const Tensor& inv_freq, const OptTensor& qw, const OptTensor& kw, std::optional<double> eps,
                                    bool inter, double gain, bool weights) {
    const auto [pos, freq] = check_rope(q, k, positions, inv_freq, qw, kw, eps.has_value());
    check_grad_of(gq, q, "grad_q"), check_grad_of(gk, k, "grad_k");
    refuse_tangents("qk_norm_rope_backward", gq, gk, q, k, qw, kw, inv_freq);
    const at::NoGradGuard no_grad;
    const bool need[4] = {true, true, weights && qw, weights && kw};
    return or_none(rope_backward(or_undefined(gq), or_undefined(gk), q, k, or_undefined(qw), or_undefined(kw), pos, freq,
                                 {eps.value_or(0.0), gain, eps.has_value(), inter}, need));
  }, release());
  m.def("check_cache", &check_cache);
  m.def("cache_write", [](const Tensor& ck, const Tensor& cv, const OptTensor& ks, const OptTensor& vs, const Tensor& k, const Tensor& v,
                          const Tensor& table, const Tensor& lengths, const OptTensor& starts) {
    check_cache(ck, cv, ks, vs);
    VALUE_CHECK(k.dim() >= 3 && k.size(-1) == ck.size(3) && k.size(-2) == ck.size(1) && k.device() == ck.device(), "k must be [..., ",
                ck.size(1), ", ", ck.size(3), "] on ", ck.device(), ", not ", k.sizes(), " on ", k.device());
    VALUE_CHECK(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && v.device() == k.device(),
                "k and v must match in shape, dtype and device");
    SUPPORT_CHECK(is_row_type(k.scalar_type()) && (ck.scalar_type() == at::kFloat8_e4m3fn || k.scalar_type() == ck.scalar_type()),
                  k.scalar_type(), " keys into a ", ck.scalar_type(), " cache");
    check_tokens(ck, table, lengths, starts, lead_rows(k));
    no_gradient("cache_write", graded(k) || graded(v) || graded(ck) || graded(cv));
    refuse_tangents("cache_write", k, v, ck, cv);
    const at::NoGradGuard no_grad;
    cache_call({ck, cv, ks, vs}, k, v, table, lengths, starts, true);
    written(ck), written(cv), written(ks), written(vs);
  }, release());
  m.def("cache_read", [](const Tensor& ck, const Tensor& cv, const OptTensor& ks, const OptTensor& vs, const Tensor& table,
                         const Tensor& lengths, int64_t tokens, const OptTensor& starts, std::optional<at::ScalarType> dtype,
                         const OptTensor& out_k, const OptTensor& out_v) {
    check_cache(ck, cv, ks, vs);
    const auto t = out_k ? out_k->scalar_type() : dtype ? *dtype : ck.scalar_type() == at::kFloat8_e4m3fn ? at::kFloat : ck.scalar_type();
    SUPPORT_CHECK(is_row_type(t), "dtype ", t, " is not supported (float32, bfloat16, float16)");
    VALUE_CHECK(tokens >= 0, "tokens ", tokens, " < 0");
    check_tokens(ck, table, lengths, starts, tokens);
    VALUE_CHECK(!out_k || !dtype || *dtype == t, "out is ", t, ", not dtype ", dtype.value_or(t));
    VALUE_CHECK(out_k.has_value() == out_v.has_value(), "out must be two tensors");
    no_gradient("cache_read", graded(ck) || graded(cv) || graded(out_k) || graded(out_v));
    refuse_tangents("cache_read", ck, cv, out_k, out_v);
    const at::NoGradGuard no_grad;
    const int64_t shape[3] = {tokens, ck.size(1), ck.size(3)};
    for (const OptTensor* o : {&out_k, &out_v})
      VALUE_CHECK(!*o || ((*o)->sizes() == at::IntArrayRef(shape) && (*o)->scalar_type() == t && (*o)->device() == ck.device() &&
                          (*o)->is_contiguous()),
                  "out must be two contiguous ", t, " tensors ", at::IntArrayRef(shape), " on ", ck.device());
    VALUE_CHECK(!out_k || at::get_overlap_status(*out_k, *out_v) == at::MemOverlapStatus::No || tokens == 0,
                "out's two tensors share memory");
    const Tensor k = out_k ? *out_k : at::empty(shape, ck.options().dtype(t)), v = out_v ? *out_v : at::empty(shape, ck.options().dtype(t));
    cache_call({ck, cv, ks, vs}, k, v, table, lengths, starts, false);
    written(out_k), written(out_v);
    return std::make_pair(k, v);
  }, release());
  m.def("attention", [](const Tensor& ck, const Tensor& cv, const OptTensor& ks, const OptTensor& vs, const Tensor& q, const Tensor& table,
                        const Tensor& lengths, const OptTensor& starts, std::optional<double> scale, double softcap,
                        std::optional<int64_t> window, int64_t sinks, const OptTensor& into, bool lse) {
    check_cache(ck, cv, ks, vs);
    VALUE_CHECK(q.dim() >= 3 && q.size(-1) == ck.size(3) && q.device() == ck.device(), "q must be [..., heads, ", ck.size(3), "] on ",
                ck.device(), ", not ", q.sizes(), " on ", q.device());
    SUPPORT_CHECK((q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf) &&
                      (ck.scalar_type() == at::kFloat8_e4m3fn || q.scalar_type() == ck.scalar_type()),
                  q.scalar_type(), " queries over a ", ck.scalar_type(), " cache");
    VALUE_CHECK(q.size(-2) >= 1 && q.size(-2) % ck.size(1) == 0, q.size(-2), " query heads over ", ck.size(1), " cached");
    check_tokens(ck, table, lengths, starts, lead_rows(q));
    VALUE_CHECK(window.value_or(0) >= 0 && sinks >= 0, "window and sinks must be >= 0");
    no_gradient("paged_attention", graded(q) || graded(ck) || graded(cv) || graded(into));
    refuse_tangents("paged_attention", q, ck, cv, into);
    const at::NoGradGuard no_grad;
    OptTensor o;
    if (into) {
      VALUE_CHECK(into->sizes() == q.sizes() && into->scalar_type() == q.scalar_type() && into->device() == q.device(),
                  "out must match q in shape, dtype and device");
      o = into->dim() == 3 ? *into : into->view({-1, q.size(-2), q.size(-1)});
      bool fine = reinterpret_cast<uintptr_t>(o->data_ptr()) % 8 == 0 && o->stride(2) == 1;
      for (int i = 0; i < 2; ++i) fine = fine && (o->size(i) <= 1 || (o->stride(i) % 4 == 0 && o->stride(i) >= q.size(-1)));
      if (o->size(0) > 1 && o->size(1) > 1) {   // (one of tokens and heads inside the other)
        const int in = o->stride(0) < o->stride(1) ? 0 : 1;
        fine = fine && o->stride(1 - in) >= o->stride(in) * (o->size(in) - 1) + o->size(2);
      }
      VALUE_CHECK(fine, "out must be 8-byte aligned, its heads contiguous and apart, strides in multiples of 4 elements");
      VALUE_CHECK(at::get_overlap_status(*into, q) != at::MemOverlapStatus::Partial, "out and q share some of their memory");
    }
    variable_list results = attention({ck, cv, ks, vs}, q, table, lengths, starts,
                                      scale ? *scale : 1.0 / std::sqrt(static_cast<double>(ck.size(3))), softcap, window.value_or(0), sinks,
                                      o, lse);
    written(into);
    return or_none(results);
  }, release());
}
