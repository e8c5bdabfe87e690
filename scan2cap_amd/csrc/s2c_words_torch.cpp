// s2c_words_torch.cpp -- the word operators as differentiable torch functions: argument checks, output and
// scratch tensors, the current stream of the tensors' device, autograd nodes; everything on the device is
// the C ABI of s2c_words.h.  Host code only, built into lib/s2c_words_ext.so.
//
// Why native: a training batch's kernels take 5 - 10 us each, and the same node written as a Python
// autograd.Function over ctypes took 113 us a step at the captioner's batch (its backward runs on the
// engine's thread, where every line of Python costs two to four times what it does on the caller's).
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <sstream>

#include "../../include/s2c_ops.h"
#include "../../include/s2c_words.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

// ---- checks: ValueError for what is wrong with the arguments, RuntimeError for where they live -----------
template <class... A>
void check(bool ok, const A &...what) {
  if (ok) return;
  std::ostringstream s;
  (s << ... << what);
  throw py::value_error(s.str());
}

template <class... A>
void check_place(bool ok, const A &...what) {
  if (ok) return;
  std::ostringstream s;
  (s << ... << what);
  throw std::runtime_error(s.str());
}

int type_code(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return S2C_F32;
    case at::kBFloat16: return S2C_BF16;
    case at::kHalf: return S2C_F16;
    default: return -1;
  }
}

void check_float(const char *name, const Tensor &t) {
  check(type_code(t) >= 0, name, " must be float32, bfloat16 or float16, not ", t.scalar_type());
}

void check_ids(const char *name, const Tensor &t) {
  check(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, name, " must be int64 or int32, not ",
        t.scalar_type());
}

void check_gpu(const char *name, const Tensor &t, const Tensor &like) {
  check_place(t.is_cuda(), name, " must be a GPU tensor: CPU not supported");
  check_place(t.device() == like.device(), name, " is on ", t.device(), ", the other tensors on ", like.device());
}

// values that memory holds as they are (the imaginary part of a conjugated tensor is a view whose sign is
// applied by whoever reads it)
Tensor as_stored(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }

// (the usual case costs no dispatch)
Tensor dense(const Tensor &t, at::ScalarType type) {
  return t.scalar_type() == type && t.is_contiguous() ? as_stored(t) : as_stored(t.to(type).contiguous());
}

Tensor ids64(const Tensor &t) { return dense(t, at::kLong); }

Tensor f32(const Tensor &g) { return dense(g, at::kFloat); }

// a tensor's data, NULL for an undefined one
template <class T>
T *ptr(const Tensor &t) { return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr; }

void *stream_of(const Tensor &t) { return (void *)at::hip::getCurrentHIPStream(t.get_device()).stream(); }

void done(int rc, const char *what) { check_place(rc == 0, what, " failed (rc=", rc, ")"); }

Tensor workspace(long long bytes, const Tensor &like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// ---- logits as the kernels read them -------------------------------------------------------------------------
struct Axes { int n; int64_t size[3], stride[3]; };

// the axes [0, dims) of x as few (size, stride) pairs that step alike; n = 4: more than three
Axes merge_axes(const Tensor &x, int64_t dims) {
  Axes a = {0, {1, 1, 1}, {0, 0, 0}};
  for (int64_t d = 0; d < dims; ++d) {
    const int64_t n = x.size(d), s = x.stride(d);
    if (n == 1) continue;
    if (a.n && a.stride[a.n - 1] == n * s) {
      a.size[a.n - 1] *= n;
      a.stride[a.n - 1] = s;
    } else if (a.n == 3) {
      a.n = 4;
      return a;
    } else {
      a.size[a.n] = n;
      a.stride[a.n++] = s;
    }
  }
  return a;
}

// Up to three leading axes of any strides are read in place (a decoder's word-major logits permuted to
// (B, K, T, V)); more, or words that are not adjacent, are copied first.
Tensor readable(const Tensor &t) {
  const Tensor x = as_stored(t);
  const bool adjacent = x.size(-1) == 1 || x.stride(-1) == 1;
  return adjacent && merge_axes(x, x.dim() - 1).n <= 3 ? x : x.contiguous();
}

s2c_logits logits_of(const Tensor &x, double temperature) {
  const Axes a = merge_axes(x, x.dim() - 1);
  int64_t size[3] = {1, 1, 1}, stride[3] = {0, 0, 0};
  for (int i = 0; i < a.n; ++i) {
    size[3 - a.n + i] = std::max<int64_t>(a.size[i], 1);
    stride[3 - a.n + i] = a.stride[i];
  }
  s2c_logits l;
  l.V = (int)x.size(-1);
  l.rows = (int)(x.numel() / x.size(-1));
  l.dtype = type_code(x);
  l.n1 = (int)size[1];
  l.n2 = (int)size[2];
  l.inv_t = (float)(1.0 / temperature);
  l.s0 = stride[0];
  l.s1 = stride[1];
  l.s2 = stride[2];
  l.x = x.data_ptr();
  return l;
}

void check_logits(const Tensor &x, double temperature) {
  check_float("logits", x);
  check(x.dim() >= 1 && x.size(-1) >= 1, "logits need a vocabulary axis, not shape ", x.sizes());
  check(x.size(-1) < (1LL << 31) && x.numel() / x.size(-1) < (1LL << 31), "logits: more than 2^31 rows or words");
  check(std::isfinite(temperature) && temperature >= 1e-30 && temperature <= 1e30,
        "temperature must be positive and finite, not ", temperature);
}

// The gradients are not differentiable again: where a graph of the backward pass is asked for, one that
// says so is put behind them.
Tensor first_order(const Tensor &g) {
  if (!at::GradMode::is_enabled() || !g.defined()) return g;
  Tensor v = g.detach();
  v.set_requires_grad(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", 1);
  return (*error)({v})[0];
}

// (a forward-mode tangent goes through the autograd node too, which refuses it)
bool wants_grad(const Tensor &t) {
  return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(/*level=*/0).defined();
}

// ---- token_scores ----------------------------------------------------------------------------------------------
struct Scores { Tensor logp, entropy, top_logp, top_ids, stats; };

s2c_token_scores_args scores_args(const Tensor &x, const Tensor &tokens, int64_t k, double temperature,
                                  const std::optional<int64_t> &ignore) {
  s2c_token_scores_args a = {};
  a.lg = logits_of(x, temperature);
  a.k = (int)k;
  a.has_ignore = ignore.has_value();
  a.ignore = ignore.value_or(0);
  a.token = ptr<const long long>(tokens);
  return a;
}

Scores scores_forward(const Tensor &x, const Tensor &tokens, int64_t k, double temperature,
                      const std::optional<int64_t> &ignore, bool stats) {
  const c10::DeviceGuard guard(x.device());
  const auto shape = x.sizes().slice(0, x.dim() - 1);
  const auto opt = x.options().dtype(at::kFloat);
  Scores o;
  if (tokens.defined()) o.logp = at::empty(shape, opt);
  o.entropy = at::empty(shape, opt);
  if (k) {
    std::vector<int64_t> top = shape.vec();
    top.push_back(k);
    o.top_logp = at::empty(top, opt);
    o.top_ids = at::empty(top, opt.dtype(at::kLong));
  }
  s2c_token_scores_args a = scores_args(x, tokens, k, temperature, ignore);
  if (stats) o.stats = at::empty({a.lg.rows, 4}, opt);
  if (a.lg.rows == 0) return o;
  const Tensor ws = workspace(s2c_token_scores_workspace_bytes(a.lg.rows, a.lg.V, a.lg.dtype, a.k), x);
  a.logp = ptr<float>(o.logp);
  a.entropy = ptr<float>(o.entropy);
  a.top_logp = ptr<float>(o.top_logp);
  a.top_ids = ptr<long long>(o.top_ids);
  a.stats = ptr<float>(o.stats);
  a.ws = ptr<void>(ws);
  done(s2c_token_scores_fwd(&a, stream_of(x)), "s2c_token_scores_fwd");
  return o;
}

struct TokenScoresFn : torch::autograd::Function<TokenScoresFn> {
  static variable_list forward(AutogradContext *ctx, const Tensor &logits, const MaybeTensor &words, int64_t k,
                               double temperature, std::optional<int64_t> ignore) {
    const Tensor x = readable(logits), tokens = words.value_or(Tensor());
    const Scores o = scores_forward(x, tokens, k, temperature, ignore, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, tokens, o.top_ids, o.stats});
    ctx->saved_data["k"] = k;
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore"] = ignore;
    if (k) ctx->mark_non_differentiable({o.top_ids});
    // entropy [, logp] [, top_logp, top_ids]: what there is
    variable_list out = {o.entropy};
    if (tokens.defined()) out.push_back(o.logp);
    if (k) {
      out.push_back(o.top_logp);
      out.push_back(o.top_ids);
    }
    return out;
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &g) {
    variable_list out(5);
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0];
    const int64_t k = ctx->saved_data["k"].toInt();
    const size_t words = s[1].defined() ? 1 : 0;
    Tensor grads[3];                              // of logp, entropy, top_logp
    if (words && g[1].defined()) grads[0] = f32(g[1]);
    if (g[0].defined()) grads[1] = f32(g[0]);
    if (k && g[1 + words].defined()) grads[2] = f32(g[1 + words]);
    if (!grads[0].defined() && !grads[1].defined() && !grads[2].defined()) return out;
    const c10::DeviceGuard guard(x.device());
    s2c_token_scores_args a = scores_args(x, s[1], k, ctx->saved_data["temperature"].toDouble(),
                                          ctx->saved_data["ignore"].toOptional<int64_t>());
    a.top_ids = ptr<long long>(s[2]);
    a.stats = ptr<float>(s[3]);
    const Tensor dx = at::empty(x.sizes(), x.options());
    if (a.lg.rows)
      done(s2c_token_scores_bwd(&a, ptr<float>(grads[0]), ptr<float>(grads[1]), ptr<float>(grads[2]), dx.data_ptr(),
                                stream_of(x)),
           "s2c_token_scores_bwd");
    out[0] = first_order(dx);
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> token_scores(const Tensor &logits, const MaybeTensor &tokens, int64_t top_k,
                                                        double temperature, std::optional<int64_t> ignore) {
  check_logits(logits, temperature);
  check(top_k >= 0 && top_k <= std::min<int64_t>(S2C_WORDS_MAX_TOP, logits.size(-1)), "top_k must be in [0, min(",
        S2C_WORDS_MAX_TOP, ", V)], not ", top_k);
  MaybeTensor t;
  if (tokens.has_value()) {
    check_ids("tokens", *tokens);
    check(tokens->sizes() == logits.sizes().slice(0, logits.dim() - 1), "tokens has shape ", tokens->sizes(),
          " for logits of shape ", logits.sizes());
  } else {
    check(!ignore.has_value(), "ignore_index needs tokens");
  }
  check_gpu("logits", logits, logits);
  if (tokens.has_value()) {
    check_gpu("tokens", *tokens, logits);
    t = ids64(*tokens);
  }
  if (!wants_grad(logits)) {
    const Scores o = scores_forward(readable(logits), t.value_or(Tensor()), top_k, temperature, ignore, false);
    return {o.logp, o.entropy, o.top_logp, o.top_ids};
  }
  const variable_list o = TokenScoresFn::apply(logits, t, top_k, temperature, ignore);
  const size_t top = t.has_value() ? 2 : 1;
  return {t.has_value() ? o[1] : Tensor(), o[0], top_k ? o[top] : Tensor(), top_k ? o[top + 1] : Tensor()};
}

// ---- distill_loss ----------------------------------------------------------------------------------------------
s2c_distill_args distill_args(const Tensor &x, const Tensor &ids, const Tensor &teacher, const Tensor &mask,
                              double temperature) {
  s2c_distill_args a = {};
  a.lg = logits_of(x, temperature);
  a.K = (int)ids.size(-1);
  a.teacher_dtype = type_code(teacher);
  a.ids = ptr<const long long>(ids);
  a.teacher = teacher.data_ptr();
  a.mask = ptr<const unsigned char>(mask);
  return a;
}

struct Distilled { Tensor loss, stats; };

Distilled distill_forward(const Tensor &x, const Tensor &ids, const Tensor &teacher, const Tensor &mask,
                          double temperature, bool stats) {
  const c10::DeviceGuard guard(x.device());
  const auto opt = x.options().dtype(at::kFloat);
  Distilled o;
  o.loss = at::empty(x.sizes().slice(0, x.dim() - 1), opt);
  if (x.numel() == 0) return o;
  s2c_distill_args a = distill_args(x, ids, teacher, mask, temperature);
  if (stats) o.stats = at::empty({a.lg.rows, 4}, opt);
  const Tensor ws = workspace(s2c_distill_workspace_bytes(a.lg.rows, a.lg.V, a.lg.dtype), x);
  a.loss = ptr<float>(o.loss);
  a.stats = ptr<float>(o.stats);
  a.ws = ptr<void>(ws);
  done(s2c_distill_fwd(&a, stream_of(x)), "s2c_distill_fwd");
  return o;
}

struct DistillFn : torch::autograd::Function<DistillFn> {
  static Tensor forward(AutogradContext *ctx, const Tensor &logits, const Tensor &ids, const Tensor &teacher,
                        const MaybeTensor &mask, double temperature) {
    const Tensor x = readable(logits);
    const Distilled o = distill_forward(x, ids, teacher, mask.value_or(Tensor()), temperature, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, ids, teacher, o.stats});
    ctx->saved_data["temperature"] = temperature;
    return o.loss;
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &g) {
    variable_list out(5);
    if (!g[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0];
    const c10::DeviceGuard guard(x.device());
    const Tensor dx = at::empty(x.sizes(), x.options());
    if (x.numel()) {
      s2c_distill_args a = distill_args(x, s[1], s[2], Tensor(), ctx->saved_data["temperature"].toDouble());
      a.stats = ptr<float>(s[3]);
      const Tensor up = f32(g[0]);
      done(s2c_distill_bwd(&a, ptr<float>(up), dx.data_ptr(), stream_of(x)), "s2c_distill_bwd");
    }
    out[0] = first_order(dx);
    return out;
  }
};

Tensor distill_loss(const Tensor &logits, const Tensor &ids, const Tensor &teacher, double temperature,
                    const MaybeTensor &mask) {
  check_logits(logits, temperature);
  check(ids.dim() == logits.dim(), "teacher_ids needs the logits' leading axes and a slot axis");
  const int64_t K = ids.size(-1);
  check(K >= 1 && K <= S2C_WORDS_MAX_SLOTS, "1 to ", S2C_WORDS_MAX_SLOTS, " teacher slots a row, not ", K);
  const auto shape = logits.sizes().slice(0, logits.dim() - 1);
  check_ids("teacher_ids", ids);
  check(ids.sizes().slice(0, ids.dim() - 1) == shape, "teacher_ids has shape ", ids.sizes(), " for logits of shape ",
        logits.sizes());
  check_float("teacher_logits", teacher);
  check(teacher.sizes() == ids.sizes(), "teacher_logits has shape ", teacher.sizes(), ", teacher_ids ", ids.sizes());
  check(!wants_grad(teacher), "teacher_logits requires a gradient, which distill_loss does not form: detach it");
  if (mask.has_value())
    check(mask->scalar_type() == at::kBool && mask->sizes() == shape, "mask must be a bool tensor of shape ", shape);
  check_gpu("logits", logits, logits);
  check_gpu("teacher_ids", ids, logits);
  check_gpu("teacher_logits", teacher, logits);
  if (mask.has_value()) check_gpu("mask", *mask, logits);
  const Tensor i = ids64(ids), w = dense(teacher.detach(), teacher.scalar_type());
  const MaybeTensor m = mask.has_value() ? MaybeTensor(mask->contiguous()) : MaybeTensor();
  if (!wants_grad(logits))
    return distill_forward(readable(logits), i, w, m.value_or(Tensor()), temperature, false).loss;
  return DistillFn::apply(logits, i, w, m, temperature);
}

// ---- embed_tokens ----------------------------------------------------------------------------------------------
Tensor embed_forward(const Tensor &tokens, const Tensor &table, double scale, int64_t padding) {
  const c10::DeviceGuard guard(table.device());
  std::vector<int64_t> shape = tokens.sizes().vec();
  shape.push_back(table.size(1));
  const Tensor out = at::empty(shape, table.options());
  if (out.numel())
    done(s2c_embed_fwd(tokens.numel(), (int)table.size(0), (int)table.size(1), type_code(table), table.stride(0),
                       ptr<const long long>(tokens), table.data_ptr(), (float)scale, padding, out.data_ptr(),
                       stream_of(table)),
         "s2c_embed_fwd");
  return out;
}

struct EmbedFn : torch::autograd::Function<EmbedFn> {
  static Tensor forward(AutogradContext *ctx, const Tensor &tokens, const Tensor &table, double scale,
                        int64_t padding) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({tokens});
    ctx->saved_data["V"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embed_forward(tokens, as_stored(table), scale, padding);
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    Tensor g = as_stored(grads[0]);
    const c10::DeviceGuard guard(g.device());
    const Tensor tokens = ctx->get_saved_variables()[0];
    const int64_t N = tokens.numel(), V = ctx->saved_data["V"].toInt(), D = g.size(-1);
    const Tensor d = at::empty({V, D}, g.options());
    if (D) {
      // rows of one stride are read in place
      Axes a = merge_axes(g, g.dim() - 1);
      if (a.n > 1 || (D > 1 && g.stride(-1) != 1)) {
        g = g.contiguous();
        a = merge_axes(g, g.dim() - 1);
      }
      const Tensor ws = workspace(s2c_embed_grad_workspace_bytes(N, (int)V, (int)D), g);
      done(s2c_embed_grad(N, (int)V, (int)D, type_code(g), a.n ? a.stride[0] : D, ptr<const long long>(tokens),
                          g.data_ptr(), (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(),
                          d.data_ptr(), ptr<void>(ws), stream_of(g)),
           "s2c_embed_grad");
    }
    out[1] = first_order(d);
    return out;
  }
};

Tensor embed_tokens(const Tensor &tokens, const Tensor &table, double scale, std::optional<int64_t> padding) {
  check_float("table", table);
  check(table.dim() == 2 && table.size(0) >= 1 && table.size(0) < (1LL << 31) && table.size(1) <= S2C_WORDS_MAX_DIM,
        "table must be (V, D) with 1 <= V and D <= ", S2C_WORDS_MAX_DIM, ", not ", table.sizes());
  check(table.size(1) <= 1 || table.stride(1) == 1, "the table's columns must be adjacent");
  check(std::isfinite(scale) && std::abs(scale) <= 3e38, "scale must be finite, not ", scale);
  check_ids("tokens", tokens);
  check(tokens.numel() < (1LL << 31), "tokens: more than 2^31");
  check_gpu("table", table, table);
  check_gpu("tokens", tokens, table);
  const Tensor t = ids64(tokens);
  check(padding != std::optional<int64_t>(S2C_WORDS_NO_PADDING), "padding_idx cannot be the lowest integer");
  const int64_t pad = padding.value_or(S2C_WORDS_NO_PADDING);
  return wants_grad(table) ? EmbedFn::apply(t, table, scale, pad) : embed_forward(t, as_stored(table), scale, pad);
}

}  // namespace

PYBIND11_MODULE(s2c_words_ext, m) {
  // the argument blocks of the library that is loaded, against those that this file was compiled with
  const long long sizes[] = {sizeof(s2c_logits), sizeof(s2c_token_scores_args), sizeof(s2c_distill_args)};
  for (int i = 0; i < 3; ++i)
    if (s2c_words_args_sizeof(i) != sizes[i])
      throw py::import_error("s2c_words_ext.so and libs2c_hip.so were built from different headers -- run "
                             "`python -m scan2cap_amd.build`");
  m.def("token_scores", &token_scores);
  m.def("distill_loss", &distill_loss);
  m.def("embed_tokens", &embed_tokens);
}
