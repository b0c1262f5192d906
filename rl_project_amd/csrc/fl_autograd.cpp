// score_tokens, layer_norm and lm_head_logprobs as a torch extension over the C
// ABI (include/fl_sampler.h): the launches with their allocations, and the
// autograd nodes.  The kernels are the library's; what is here would cost more
// than the small calls' kernels in Python.  (Host time of layer_norm 255x1025,
// forward and gradients: 110 us with a Python node, which waits for the
// interpreter on the engine's own thread, 73 us so; score_tokens 1x50257 with 5
// alternatives: 20 us over ctypes, 11.6 us so.)
//
// The Python callers have checked every argument; the entry points come from the
// library that Python loaded (bind).
#include <torch/extension.h>

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <optional>
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
} L;

void bind(const std::vector<uintptr_t>& p) {
  TORCH_CHECK(p.size() == 11, "fl_autograd: 11 entry points expected");
  auto at = [&](size_t i, auto& f) { f = reinterpret_cast<std::decay_t<decltype(f)>>(p[i]); };
  at(0, L.last_error), at(1, L.score), at(2, L.score_ws), at(3, L.score_grad), at(4, L.norm), at(5, L.norm_grad),
      at(6, L.norm_ws), at(7, L.head), at(8, L.head_ws), at(9, L.head_grad), at(10, L.head_grad_ws);
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
}
