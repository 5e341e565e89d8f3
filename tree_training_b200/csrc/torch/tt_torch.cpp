// Torch bindings of the layer operators (token log probabilities, rotary
// positions, residual norms, tokens sorted by expert): argument checks, outputs
// and autograd nodes around the C ABI.  A decoder layer makes several of these
// calls for few tokens, where the host decides: a call is 4 to 9 us here, and
// was 10 to 17 through Python (forward and backward of a norm 64, not 113).
//
// No arithmetic is done here.  Every call runs on the current stream of its
// tensors' device; gradients carry no graph (differentiating them again is an
// error).
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <array>
#include <atomic>
#include <optional>
#include <string>

#include "../../../include/tree_training_b200.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

namespace {

// ---- errors and arguments ------------------------------------------------------

// A status of the library other than TT_OK; becomes the package's TTError.
struct Failure : std::runtime_error {
  std::string fn;
  int code;
  Failure(const char* f, int c)
      : std::runtime_error(std::string(f) + " failed: " + tt_status_string(c) + " (status " +
                           std::to_string(c) + ")"),
        fn(f), code(c) {}
};

void check_status(const char* fn, int code) {
  if (code != TT_OK) throw Failure(fn, code);
}

[[noreturn]] void type_error(const std::string& s) { throw py::type_error(s); }
[[noreturn]] void value_error(const std::string& s) { throw py::value_error(s); }

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TT_F32;
    case at::kBFloat16: return TT_BF16;
    case at::kHalf: return TT_F16;
    default: return -1;
  }
}

void need_cuda(const char* op, const char* name, const Tensor& t, const Tensor& first) {
  if (!t.defined()) return;
  if (!t.is_cuda())
    throw std::runtime_error(std::string(op) + ": " + name + " must be a CUDA tensor (no CPU path)");
  if (t.device() != first.device())
    throw std::runtime_error(std::string(op) + ": " + name + " is on " + t.device().str() +
                             ", other tensors on " + first.device().str());
}

void need_int(const char* op, const char* what, const Tensor& t) {
  if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)
    type_error(std::string(op) + ": int64/int32 " + what + " required");
}

// The C ABI's sizes have 32 bits: larger ones are refused, not cut off.
void need_size(const char* op, const char* what, int64_t n) {
  if (n > 0x7fffffff)
    value_error(std::string(op) + ": " + what + " of " + std::to_string(n) +
                " is over the limit of 2^31 - 1");
}

// There are no forward-mode derivatives: a result without its tangent would be
// wrong without a word.  (A tangent counts with gradients turned off, too.)
void no_tangent(const char* op, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined())
      throw std::runtime_error(std::string(op) + ": forward-mode derivatives are not supported");
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// [rows, D] with unit last stride and rows that do not overlap (else a copy).
Tensor rows2d(const Tensor& t) {
  if (t.stride(1) == 1 && (t.stride(0) >= t.size(1) || t.size(0) <= 1)) return t;
  return t.contiguous();
}

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int64_t row_stride(const Tensor& t) { return t.defined() ? t.stride(0) : 0; }

Tensor empty(at::IntArrayRef sizes, const Tensor& like, at::ScalarType type) {
  return at::empty(sizes, like.options().dtype(type).memory_format(at::MemoryFormat::Contiguous)
                              .requires_grad(false));
}

// The device and stream of a call.
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

// The device's status word, which check_device_status reads: asked for once.
std::array<std::atomic<int32_t*>, 64> status_words;

int32_t* status_of(const Tensor& t) {
  const int i = t.device().index();
  TORCH_CHECK(i >= 0 && i < (int)status_words.size(), "device index out of range");
  int32_t* p = status_words[i].load(std::memory_order_acquire);
  if (!p) {
    py::gil_scoped_acquire gil;
    py::object word = py::module_::import("tree_training_b200.attention")
                          .attr("_status_word")(py::cast(t.device()));
    p = word.cast<Tensor>().data_ptr<int32_t>();
    status_words[i].store(p, std::memory_order_release);
  }
  return p;
}

// Gradients that are differentiated again (create_graph) raise there.
variable_list once(const char* op, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(op) + ": its gradients cannot be differentiated again", 1);
  for (auto& g : grads) {
    if (!g.defined()) continue;
    variable_list one{g.detach().requires_grad_(true)};
    g = (*error)(std::move(one))[0];
  }
  return grads;
}

// ---- token log probabilities -----------------------------------------------------

struct Logprobs {
  Tensor logp, ent, top_lp, top_tok, stats;
};

Logprobs logprobs_forward(const Tensor& x, const Tensor& tokens, int64_t k, double temperature,
                          bool keep) {
  const int64_t T = x.size(0), V = x.size(1), M = tokens.size(1);
  Logprobs r;
  r.logp = empty({T, M}, x, at::kFloat);
  r.ent = empty({T}, x, at::kFloat);
  r.top_lp = empty({T, k}, x, at::kFloat);
  r.top_tok = empty({T, k}, x, at::kLong);
  if (keep) r.stats = empty({T, 4}, x, at::kFloat);
  On on(x);
  check_status("tt_token_logprobs_fwd",
               tt_token_logprobs_fwd(dtype_code(x), T, (int32_t)V, ptr(x),
                                     std::max(x.stride(0), V),
                                     (const int64_t*)ptr(tokens), (int32_t)M, (float)temperature,
                                     (int32_t)k, (float*)out(r.logp), (float*)out(r.ent),
                                     (float*)out(r.top_lp), (int64_t*)out(r.top_tok),
                                     (float*)out(r.stats), on.stream));
  return r;
}

struct LogprobsFunction : Function<LogprobsFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& tokens,
                               int64_t k, double temperature) {
    Logprobs r = logprobs_forward(x, tokens, k, temperature, true);
    ctx->save_for_backward({x, tokens, r.top_tok, r.stats});
    ctx->saved_data["temperature"] = temperature;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({r.top_tok});
    return {r.logp, r.ent, r.top_lp, r.top_tok};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return variable_list(4);
    no_tangent("token_logprobs", {&g[0], &g[1], &g[2]});
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &tokens = s[1], &top_tok = s[2], &stats = s[3];
    for (int i = 0; i < 3; ++i)
      if (g[i].defined()) g[i] = g[i].to(at::kFloat).contiguous();
    const int64_t T = x.size(0), V = x.size(1);
    Tensor dx = empty({T, V}, x, x.scalar_type());
    {
      On on(x);
      check_status(
          "tt_token_logprobs_bwd",
          tt_token_logprobs_bwd(dtype_code(x), T, (int32_t)V, ptr(x), std::max(x.stride(0), V),
                                (const int64_t*)ptr(tokens), (int32_t)tokens.size(1),
                                (float)ctx->saved_data["temperature"].toDouble(),
                                (int32_t)top_tok.size(1), (const int64_t*)ptr(top_tok),
                                (const float*)ptr(g[0]), (const float*)ptr(g[1]),
                                (const float*)ptr(g[2]), (const float*)ptr(stats), out(dx),
                                on.stream));
    }
    return once("token_logprobs", {dx, Tensor(), Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits,
                                                          const OptTensor& tokens_, int64_t k,
                                                          double temperature, int64_t max_k) {
  const char* op = "token_logprobs";
  const Tensor tokens = tokens_.value_or(Tensor());
  need_cuda(op, "logits", logits, logits);
  need_cuda(op, "tokens", tokens, logits);
  if (dtype_code(logits) < 0) type_error("token_logprobs: float32/bfloat16/float16 logits required");
  if (logits.dim() != 2 || logits.size(1) < 1)
    value_error("token_logprobs: logits must be [rows, V]");
  const int64_t T = logits.size(0), V = logits.size(1);
  need_size(op, "a vocabulary", V);
  if (k < 0 || k > std::min(max_k, V))
    value_error("token_logprobs: top_k must be in [0, " + std::to_string(std::min(max_k, V)) + "]");
  if (!(temperature >= 1e-20 && temperature <= 1e20))
    value_error("token_logprobs: temperature must be in [1e-20, 1e20]");
  Tensor tok;
  if (tokens.defined()) {
    need_int(op, "tokens", tokens);
    if (tokens.dim() < 1 || tokens.dim() > 2 || tokens.size(0) != T)
      value_error("token_logprobs: tokens must be [rows] or [rows, M]");
    tok = tokens.dim() == 2 ? tokens : tokens.unsqueeze(1);
    need_size(op, "a number of tokens a row", tok.size(1));
    tok = tok.to(at::kLong).contiguous();
  } else {
    tok = empty({T, 0}, logits, at::kLong);
  }
  no_tangent(op, {&logits});
  const Tensor x = rows2d(logits);
  Logprobs r;
  if (wants_grad({&logits})) {
    variable_list v = LogprobsFunction::apply(x, tok, k, temperature);
    r.logp = v[0], r.ent = v[1], r.top_lp = v[2], r.top_tok = v[3];
  } else {
    r = logprobs_forward(x, tok, k, temperature, false);
  }
  if (tokens.defined() && tokens.dim() == 1) r.logp = r.logp.squeeze(1);
  return {r.logp, r.ent, r.top_lp, r.top_tok};
}

// ---- rotary positions --------------------------------------------------------------

std::pair<Tensor, Tensor> turn(Tensor q, Tensor k, const Tensor& pos, const Tensor& table,
                               bool interleaved, bool inverse) {
  const Tensor& first = q.defined() ? q : k;
  const int64_t n = first.size(0), D = first.size(2);
  const int64_t hq = q.defined() ? q.size(1) : 0, hk = k.defined() ? k.size(1) : 0;
  Tensor qo, ko;
  if (q.defined()) {
    if (q.stride(2) != 1) q = q.contiguous();
    qo = empty({n, hq, D}, q, q.scalar_type());
  }
  if (k.defined()) {
    if (k.stride(2) != 1) k = k.contiguous();
    ko = empty({n, hk, D}, k, k.scalar_type());
  }
  if (hq + hk == 0) return {qo, ko};
  int32_t* status = status_of(first);
  On on(first);
  check_status("tt_rotary",
               tt_rotary(dtype_code(first), n, (int32_t)hq, (int32_t)hk, (int32_t)D,
                         (int32_t)table.size(1), interleaved, inverse, hq ? ptr(q) : nullptr,
                         hq ? q.stride(0) : 0, hq ? q.stride(1) : 0, hk ? ptr(k) : nullptr,
                         hk ? k.stride(0) : 0, hk ? k.stride(1) : 0, ptr(pos),
                         pos.scalar_type() == at::kLong, (const float*)ptr(table), table.size(0),
                         hq ? out(qo) : nullptr, hk ? out(ko) : nullptr, status, on.stream));
  return {qo, ko};
}

struct RotaryFunction : Function<RotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k,
                               const Tensor& pos, const Tensor& table, bool interleaved) {
    ctx->save_for_backward({pos, table});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->set_materialize_grads(false);
    auto r = turn(q, k.value_or(Tensor()), pos, table, interleaved, false);
    if (k) return {r.first, r.second};
    return {r.first};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor gk = g.size() > 1 ? g[1] : Tensor();
    variable_list grads(5);
    no_tangent("apply_rotary", {&g[0], &gk});
    if (g[0].defined() || gk.defined()) {
      auto r = turn(g[0], gk, s[0], s[1], ctx->saved_data["interleaved"].toBool(), true);
      grads[0] = r.first, grads[1] = r.second;
    }
    return once("apply_rotary", std::move(grads));
  }
};

std::tuple<Tensor, OptTensor> apply_rotary(const Tensor& q, const OptTensor& k_,
                                           const Tensor& positions, const Tensor& table_,
                                           bool interleaved) {
  const char* op = "apply_rotary";
  const Tensor k = k_.value_or(Tensor());
  need_cuda(op, "q", q, q);
  need_cuda(op, "k", k, q);
  need_cuda(op, "positions", positions, q);
  need_cuda(op, "table", table_, q);
  if (dtype_code(q) < 0 || (k.defined() && k.scalar_type() != q.scalar_type()))
    type_error("apply_rotary: q and k must share one of float32/bfloat16/float16");
  if (q.dim() != 3 ||
      (k.defined() && (k.dim() != 3 || k.size(0) != q.size(0) || k.size(2) != q.size(2))))
    value_error("apply_rotary: q [N, Hq, D] and k [N, Hk, D] required");
  if (table_.scalar_type() != at::kFloat || table_.dim() != 2)
    type_error("apply_rotary: table must be float32 [positions, R] (see rotary_table)");
  need_int(op, "positions", positions);
  if (positions.dim() != 1 || positions.size(0) != q.size(0))
    value_error("apply_rotary: positions must be [N]");
  const int64_t R = table_.size(1);
  if (R < 2 || R % 2 || R > q.size(2))
    value_error("apply_rotary: the table's width must be even and at most the head dim");
  if (q.size(1) < 1) value_error("apply_rotary: q has no heads");
  need_size(op, "a number of heads", q.size(1) + (k.defined() ? k.size(1) : 0));
  need_size(op, "a head dim", q.size(2));
  no_tangent(op, {&q, &k, &table_});
  const Tensor pos = positions.contiguous(), table = table_.contiguous();
  if (wants_grad({&q, &k})) {
    variable_list v = RotaryFunction::apply(q, k_, pos, table, interleaved);
    return {v[0], k_ ? OptTensor(v[1]) : std::nullopt};
  }
  auto r = turn(q, k, pos, table, interleaved, false);
  return {r.first, k_ ? OptTensor(r.second) : std::nullopt};
}

// ---- residual norms ------------------------------------------------------------------

enum Gate { kNone = 0, kChannel = 1, kRow = 2, kFull = 3 };

struct Norm {
  Tensor y, r, stats;
};

Norm norm_forward(const Tensor& x, const Tensor& res, const Tensor& w, const Tensor& post,
                  const Tensor& gate, int64_t mode, double scale, double eps, double offset,
                  bool keep) {
  const int64_t T = x.size(0), D = x.size(1);
  const Tensor& like = res.defined() ? res : x;
  Norm n;
  n.y = empty({T, D}, x, x.scalar_type());
  n.r = empty({T, D}, x, like.scalar_type());
  if (keep) n.stats = empty({T, 2}, x, at::kFloat);
  int32_t* status = status_of(x);
  On on(x);
  check_status(
      "tt_residual_norm_fwd",
      tt_residual_norm_fwd(dtype_code(x), dtype_code(like), T, (int32_t)D, ptr(x), x.stride(0),
                           ptr(res), row_stride(res), ptr(w), ptr(post),
                           w.scalar_type() == at::kFloat, (float)offset, ptr(gate),
                           row_stride(gate), (int)mode, (float)scale, (float)eps, out(n.y),
                           out(n.r), (float*)out(n.stats), status, on.stream));
  return n;
}

struct NormFunction : Function<NormFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& res_,
                               const Tensor& w, const OptTensor& post_, const OptTensor& gate_,
                               int64_t mode, double scale, double eps, double offset) {
    const Tensor res = res_.value_or(Tensor()), post = post_.value_or(Tensor()),
                 gate = gate_.value_or(Tensor());
    Norm n = norm_forward(x, res, w, post, gate, mode, scale, eps, offset, true);
    ctx->save_for_backward({x, res, w, post, gate, n.stats});
    ctx->saved_data["mode"] = mode;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["offset"] = offset;
    ctx->set_materialize_grads(false);
    return {n.y, n.r};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list grads(9);
    if (!g[0].defined() && !g[1].defined()) return grads;
    no_tangent("residual_norm", {&g[0], &g[1]});
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &res = s[1], &w = s[2], &post = s[3], &gate = s[4], &stats = s[5];
    const int64_t mode = ctx->saved_data["mode"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    const double offset = ctx->saved_data["offset"].toDouble();
    const int64_t T = x.size(0), D = x.size(1);
    const at::ScalarType rt = res.defined() ? res.scalar_type() : x.scalar_type();
    // (inputs that are not there have no number)
    int input = 0;
    auto needs = [&](const Tensor& t) { return t.defined() && ctx->needs_input_grad(input++); };
    const bool need_x = needs(x), need_res = needs(res), need_w = needs(w), need_post = needs(post),
               need_gate = needs(gate);
    // the same array where nothing stands between the two
    const bool same = !post.defined() && mode == kNone && scale == 1.0 && rt == x.scalar_type();
    auto vector = [&](const Tensor& like) {
      Tensor t = empty(like.sizes(), like, like.scalar_type());
      return T ? t : t.zero_();
    };
    Tensor dx, dres, dw, dpost, dgate;
    if (need_res || (same && need_x)) dres = empty({T, D}, x, rt);
    if (need_x && !same) dx = empty({T, D}, x, x.scalar_type());
    if (need_w) dw = vector(w);
    if (need_post) dpost = vector(post);
    if (need_gate) dgate = vector(gate);
    const Tensor dy = g[0].defined() ? rows2d(g[0]) : g[0];
    const Tensor dr = g[1].defined() ? rows2d(g[1]) : g[1];
    const int blocks = tt_residual_norm_bwd_blocks(T, (int32_t)D);
    const Tensor part = empty({3, blocks, D}, x, at::kFloat);
    int32_t* status = status_of(x);
    {
      On on(x);
      check_status(
          "tt_residual_norm_bwd",
          tt_residual_norm_bwd(dtype_code(x), rt == at::kFloat ? TT_F32 : dtype_code(x), T,
                               (int32_t)D, ptr(x), x.stride(0), ptr(res), row_stride(res), ptr(w),
                               ptr(post), w.scalar_type() == at::kFloat, (float)offset, ptr(gate),
                               row_stride(gate), (int)mode, (float)scale,
                               (const float*)ptr(stats), ptr(dy), row_stride(dy), ptr(dr),
                               row_stride(dr), out(dx), out(dres), out(dgate), out(dw),
                               out(dpost), (float*)out(part), blocks, status, on.stream));
    }
    if (need_x) grads[0] = same ? dres : dx;
    if (need_res) grads[1] = dres;
    grads[2] = dw, grads[3] = dpost, grads[4] = dgate;
    return once("residual_norm", std::move(grads));
  }
};

std::tuple<Tensor, Tensor> residual_norm(const Tensor& x, const OptTensor& residual_,
                                         const Tensor& weight, const OptTensor& post_,
                                         const OptTensor& gate_, double scale, double eps,
                                         double offset, int64_t max_dim) {
  const char* op = "residual_norm";
  const Tensor residual = residual_.value_or(Tensor()), post = post_.value_or(Tensor()),
               gate = gate_.value_or(Tensor());
  need_cuda(op, "x", x, x);
  need_cuda(op, "residual", residual, x);
  need_cuda(op, "weight", weight, x);
  need_cuda(op, "post_weight", post, x);
  need_cuda(op, "gate", gate, x);
  if (dtype_code(x) < 0) type_error("residual_norm: float32/bfloat16/float16 x required");
  if (residual.defined() && residual.scalar_type() != x.scalar_type() &&
      residual.scalar_type() != at::kFloat)
    type_error("residual_norm: residual must have x's type or float32");
  if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > max_dim)
    value_error("residual_norm: x must be [..., D] with 1 <= D <= " + std::to_string(max_dim));
  if (residual.defined() && residual.sizes() != x.sizes())
    value_error("residual_norm: residual must have x's shape");
  const int64_t D = x.size(-1);
  auto check_weight = [&](const char* name, const Tensor& w) {
    if (!w.defined()) return;
    if (w.dim() != 1 || w.size(0) != D)
      value_error(std::string("residual_norm: ") + name + " must be [" + std::to_string(D) + "]");
    if ((w.scalar_type() != x.scalar_type() && w.scalar_type() != at::kFloat) ||
        w.scalar_type() != weight.scalar_type())
      type_error(std::string("residual_norm: ") + name +
                 " must be float32 or x's type, like weight");
  };
  check_weight("weight", weight);
  check_weight("post_weight", post);
  int64_t mode = kNone;
  if (gate.defined()) {
    if (gate.scalar_type() != x.scalar_type())
      type_error("residual_norm: gate must have x's type");
    auto row_shape = x.sizes().vec();
    row_shape.back() = 1;
    if (gate.dim() == 1 && gate.size(0) == D && (x.dim() > 1 || D > 1))
      mode = kChannel;
    else if (gate.sizes() == x.sizes())
      mode = kFull;
    else if (gate.sizes() == at::IntArrayRef(row_shape))
      mode = kRow;
    else
      value_error("residual_norm: gate must be [D], [..., 1] or [..., D]");
  }
  no_tangent(op, {&x, &residual, &weight, &post, &gate});
  const bool two = x.dim() == 2;
  auto flat = [&](const Tensor& t) {
    if (!t.defined()) return t;
    return rows2d(two ? t : t.reshape({-1, t.size(-1)}));
  };
  const Tensor x2 = flat(x), r2 = flat(residual);
  const Tensor g2 = mode == kChannel ? gate.contiguous() : flat(gate);
  const Tensor w2 = weight.contiguous(), p2 = post.defined() ? post.contiguous() : post;
  auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
  Tensor y, r;
  if (wants_grad({&x, &residual, &weight, &post, &gate})) {
    variable_list v = NormFunction::apply(x2, opt(r2), w2, opt(p2), opt(g2), mode, scale, eps,
                                          offset);
    y = v[0], r = v[1];
  } else {
    Norm n = norm_forward(x2, r2, w2, p2, g2, mode, scale, eps, offset, false);
    y = n.y, r = n.r;
  }
  if (two) return {y, r};
  return {y.view(x.sizes()), r.view(x.sizes())};
}

// ---- tokens sorted by expert -------------------------------------------------------------

std::tuple<Tensor, Tensor, Tensor> expert_plan(const Tensor& expert_ids, int64_t E,
                                               int64_t max_experts, int64_t max_choices) {
  const char* op = "expert_plan";
  need_cuda(op, "expert_ids", expert_ids, expert_ids);
  need_int(op, "expert ids", expert_ids);
  if (expert_ids.dim() != 2) value_error("expert_plan: expert_ids must be [T, k]");
  if (E < 1 || E > max_experts)
    value_error("expert_plan: n_experts must be in [1, " + std::to_string(max_experts) + "]");
  const int64_t T = expert_ids.size(0), k = expert_ids.size(1), n = T * k;
  if (k > max_choices)
    value_error("expert_plan: at most " + std::to_string(max_choices) + " choices a token");
  if (n > 0x7fffffff) value_error("expert_plan: more than 2^31 - 1 choices");
  const Tensor ids = expert_ids.contiguous();
  const int64_t ws = tt_moe_plan_workspace_size(n, (int32_t)E);
  const Tensor slots = empty({T, k}, ids, at::kInt), entries = empty({n}, ids, at::kInt);
  const Tensor offsets = empty({E + 1}, ids, at::kInt);
  const Tensor work = ws > 0 ? empty({ws / 4}, ids, at::kInt) : Tensor();
  On on(ids);
  check_status("tt_moe_plan",
               tt_moe_plan(ptr(ids), ids.scalar_type() == at::kLong, n, (int32_t)E,
                           (int32_t*)out(slots), (int32_t*)out(entries), (int32_t*)out(offsets),
                           out(work), ws, on.stream));
  return {slots, entries, offsets};
}

// What the calls take of a plan.
struct Plan {
  const Tensor &slots, &offsets;
  int64_t T, k, E;
  Plan(const Tensor& s, const Tensor& o)
      : slots(s), offsets(o), T(s.size(0)), k(s.size(1)), E(o.size(0) - 1) {}
};

Tensor dispatch_rows(const Tensor& x, const Plan& p) {
  const int64_t H = x.size(1);
  Tensor xs = empty({p.T * p.k, H}, x, x.scalar_type());
  On on(x);
  check_status("tt_moe_dispatch",
               tt_moe_dispatch(dtype_code(x), p.T, (int32_t)p.k, (int32_t)H, (int32_t)p.E,
                               (const int32_t*)ptr(p.slots), (const int32_t*)ptr(p.offsets),
                               ptr(x), out(xs), on.stream));
  return xs;
}

Tensor collect_rows(const Tensor& dxs, const Plan& p) {
  const int64_t H = dxs.size(1);
  Tensor dx = empty({p.T, H}, dxs, dxs.scalar_type());
  On on(dxs);
  check_status("tt_moe_collect",
               tt_moe_collect(dtype_code(dxs), p.T, (int32_t)p.k, (int32_t)H, (int32_t)p.E,
                              (const int32_t*)ptr(p.slots), (const int32_t*)ptr(p.offsets),
                              ptr(dxs), out(dx), on.stream));
  return dx;
}

Tensor combine_rows(const Tensor& ys, const Tensor& w, const Plan& p) {
  const int64_t H = ys.size(1);
  Tensor y = empty({p.T, H}, ys, ys.scalar_type());
  On on(ys);
  check_status("tt_moe_combine",
               tt_moe_combine(dtype_code(ys), dtype_code(w), p.T, (int32_t)p.k, (int32_t)H,
                              (int32_t)p.E, (const int32_t*)ptr(p.slots),
                              (const int32_t*)ptr(p.offsets), ptr(ys), ptr(w), out(y),
                              on.stream));
  return y;
}

struct DispatchFunction : Function<DispatchFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& slots,
                        const Tensor& offsets) {
    ctx->save_for_backward({slots, offsets});
    return dispatch_rows(x, Plan(slots, offsets));
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    no_tangent("expert_dispatch", {&g[0]});
    return once("expert_dispatch",
                {collect_rows(g[0].contiguous(), Plan(s[0], s[1])), Tensor(), Tensor()});
  }
};

struct CombineFunction : Function<CombineFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ys, const Tensor& w,
                        const Tensor& slots, const Tensor& offsets) {
    ctx->save_for_backward({ys, w, slots, offsets});
    return combine_rows(ys, w, Plan(slots, offsets));
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &ys = s[0], &w = s[1];
    const Plan p(s[2], s[3]);
    no_tangent("expert_combine", {&g[0]});
    const Tensor dy = g[0].contiguous();
    Tensor dys = empty(ys.sizes(), ys, ys.scalar_type()), dw = empty(w.sizes(), w, w.scalar_type());
    {
      On on(ys);
      check_status("tt_moe_spread",
                   tt_moe_spread(dtype_code(ys), dtype_code(w), p.T, (int32_t)p.k,
                                 (int32_t)ys.size(1), (int32_t)p.E, (const int32_t*)ptr(p.slots),
                                 (const int32_t*)ptr(p.offsets), ptr(dy), ptr(ys), ptr(w),
                                 out(dys), out(dw), on.stream));
    }
    return once("expert_combine", {dys, dw, Tensor(), Tensor()});
  }
};

// A plan may be the caller's own: what its arrays hold is checked by the kernels,
// which take a slot outside the sorted rows as a dropped choice.
void check_plan(const char* op, const Tensor& slots, const Tensor& offsets) {
  const std::string name = std::string(op) + ": ";
  if (slots.scalar_type() != at::kInt || offsets.scalar_type() != at::kInt)
    type_error(name + "the plan's slots and offsets must be int32");
  if (slots.dim() != 2 || offsets.dim() != 1 || offsets.size(0) < 2)
    value_error(name + "the plan's slots must be [T, k] and its offsets [experts + 1]");
  if (slots.numel() > 0x7fffffff) value_error(name + "more than 2^31 - 1 choices");
}

void check_rows(const char* op, const char* name, const Tensor& t, int64_t rows,
                const Tensor& slots, const Tensor& offsets) {
  need_cuda(op, name, t, t);
  need_cuda(op, "plan.slots", slots, t);
  need_cuda(op, "plan.offsets", offsets, t);
  if (dtype_code(t) < 0)
    type_error(std::string(op) + ": float32/bfloat16/float16 " + name + " required");
  if (t.dim() != 2 || t.size(0) != rows || t.size(1) < 1)
    value_error(std::string(op) + ": " + name + " must be [" + std::to_string(rows) + ", H]");
  need_size(op, "a row's width", t.size(1));
}

Tensor expert_dispatch(const Tensor& x_, const Tensor& slots_, const Tensor& offsets_) {
  const char* op = "expert_dispatch";
  check_plan(op, slots_, offsets_);
  check_rows(op, "x", x_, slots_.size(0), slots_, offsets_);
  no_tangent(op, {&x_});
  const Tensor x = x_.contiguous(), slots = slots_.contiguous(), offsets = offsets_.contiguous();
  if (wants_grad({&x})) return DispatchFunction::apply(x, slots, offsets);
  return dispatch_rows(x, Plan(slots, offsets));
}

Tensor expert_combine(const Tensor& ys_, const Tensor& weights, const Tensor& slots_,
                      const Tensor& offsets_) {
  const char* op = "expert_combine";
  check_plan(op, slots_, offsets_);
  const Tensor slots = slots_.contiguous(), offsets = offsets_.contiguous();
  check_rows(op, "ys", ys_, slots.size(0) * slots.size(1), slots, offsets);
  need_cuda(op, "weights", weights, ys_);
  if (dtype_code(weights) < 0)
    type_error("expert_combine: float32/bfloat16/float16 weights required");
  if (weights.sizes() != slots.sizes())
    value_error("expert_combine: weights must be [" + std::to_string(slots.size(0)) + ", " +
                std::to_string(slots.size(1)) + "]");
  no_tangent(op, {&ys_, &weights});
  const Tensor ys = ys_.contiguous(), w = weights.contiguous();
  if (wants_grad({&ys, &w})) return CombineFunction::apply(ys, w, slots, offsets);
  return combine_rows(ys, w, Plan(slots, offsets));
}

}  // namespace

PYBIND11_MODULE(_tt_torch, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Failure& e) {
      py::object cls = py::module_::import("tree_training_b200._lib").attr("TTError");
      PyErr_SetObject(cls.ptr(), cls(e.fn, e.code).ptr());
    }
  });
  using Unlocked = py::call_guard<py::gil_scoped_release>;
  m.def("token_logprobs", &token_logprobs, Unlocked());
  m.def("apply_rotary", &apply_rotary, Unlocked());
  m.def("residual_norm", &residual_norm, Unlocked());
  m.def("expert_plan", &expert_plan, Unlocked());
  m.def("expert_dispatch", &expert_dispatch, Unlocked());
  m.def("expert_combine", &expert_combine, Unlocked());
}
