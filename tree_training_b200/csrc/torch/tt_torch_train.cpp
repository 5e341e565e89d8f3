// Torch bindings of the operators at the ends and in the middle of a training
// step (embedding rows, the gated feed-forward product, the LM head's loss, the
// gradients' norm), as in tt_torch.cpp.
#include "tt_torch.h"

#include <algorithm>
#include <cmath>
#include <vector>

namespace {

using namespace tt_torch;

Tensor bytes(int64_t n, const Tensor& like) {
  return empty({std::max<int64_t>(n, 16)}, like, at::kByte);
}

int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }

// [rows, n] with unit last stride whose rows the tensor cores' copies can read: on
// 16-byte boundaries (else padded copies, all by one launch).  fp32 rows as they are.
template <size_t N>
std::array<Tensor, N> rows16(const std::array<const Tensor*, N>& ts) {
  std::array<Tensor, N> r, copy;
  int64_t rows[N], cols[N], ld[N], to_ld[N];
  const void* src[N];
  void* dst[N];
  int32_t n = 0;
  for (size_t i = 0; i < N; ++i) {
    const Tensor& t = r[i] = rows2d(*ts[i]);
    if (t.scalar_type() == at::kFloat) continue;
    if ((reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0 &&
        (t.stride(0) % 8 == 0 || (t.size(0) == 1 && t.size(1) % 8 == 0)))
      continue;
    copy[i] = empty({t.size(0), pad8(t.size(1))}, t, t.scalar_type());
    rows[n] = t.size(0), cols[n] = t.size(1), ld[n] = std::max(t.stride(0), t.size(1));
    to_ld[n] = pad8(t.size(1)), src[n] = ptr(t), dst[n++] = out(copy[i]);
  }
  if (n == 0) return r;
  On on(r[0]);
  check_status("tt_align_rows_of",
               tt_align_rows_of(n, rows, cols, src, ld, dst, to_ld, on.stream));
  at::NoGradGuard no_grad;
  for (size_t i = 0; i < N; ++i)
    if (copy[i].defined()) r[i] = copy[i].narrow(1, 0, r[i].size(1));
  return r;
}

// The stride of rows (of one row: its own width, rounded up).
int64_t ld_of(const Tensor& t) {
  return t.size(0) == 1 ? pad8(t.size(1)) : t.stride(0);
}

// ---- embedding -------------------------------------------------------------------

Tensor embed_rows(const Tensor& ids, const Tensor& w, double scale) {
  const int64_t n = ids.numel(), V = w.size(0), H = w.size(1);
  auto sizes = ids.sizes().vec();
  sizes.push_back(H);
  Tensor y = empty(sizes, w, w.scalar_type());
  int32_t* status = status_of(w);
  On on(w);
  check_status("tt_embedding_fwd",
               tt_embedding_fwd(dtype_code(w), n, V, (int32_t)H, ptr(ids),
                                ids.scalar_type() == at::kLong, ptr(w), std::max(w.stride(0), H),
                                (float)scale, out(y), status, on.stream));
  return y;
}

struct EmbeddingFunction : Function<EmbeddingFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& w, const Tensor& ids, double scale,
                        int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["V"] = w.size(0);
    return embed_rows(ids, w, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_tangent("embedding", {&g[0]});
    const Tensor ids = ctx->get_saved_variables()[0];
    const int64_t V = ctx->saved_data["V"].toInt(), H = g[0].size(-1), n = ids.numel();
    const Tensor dy = rows2d(g[0].reshape({n, H}));
    Tensor dw = empty({V, H}, dy, dy.scalar_type());
    {
      On on(dy);
      const int64_t size = tt_embedding_bwd_workspace_size(n, V, (int32_t)H);
      const Tensor ws = bytes(size, dy);
      check_status("tt_embedding_bwd",
                   tt_embedding_bwd(dtype_code(dy), n, V, (int32_t)H, ptr(ids),
                                    ids.scalar_type() == at::kLong, ptr(dy),
                                    std::max(dy.stride(0), H),
                                    (float)ctx->saved_data["scale"].toDouble(),
                                    ctx->saved_data["padding"].toInt(), out(dw), out(ws), size,
                                    on.stream));
    }
    return once("embedding", {dw, Tensor(), Tensor(), Tensor()});
  }
};

Tensor embedding(const Tensor& ids_, const Tensor& w_, double scale,
                 std::optional<int64_t> padding_) {
  const char* op = "embedding";
  need_cuda(op, "weight", w_, w_);
  need_cuda(op, "ids", ids_, w_);
  need_int(op, "ids", ids_);
  if (dtype_code(w_) < 0) type_error("embedding: float32/bfloat16/float16 weight required");
  if (w_.dim() != 2 || w_.size(0) < 1 || w_.size(1) < 1)
    value_error("embedding: weight must be [V, H]");
  const int64_t V = w_.size(0);
  need_size(op, "a vocabulary", V);
  if (w_.size(1) > (1 << 22)) value_error("embedding: a row's width is limited to 2^22");
  need_size(op, "a number of tokens", ids_.numel());
  int64_t padding = -1;
  if (padding_) {
    padding = *padding_ < 0 ? *padding_ + V : *padding_;
    if (padding < 0 || padding >= V)
      value_error("embedding: padding_idx is outside the vocabulary");
  }
  if (!std::isfinite((float)scale)) value_error("embedding: scale must be finite");
  no_tangent(op, {&w_});
  const Tensor ids = ids_.contiguous(), w = rows2d(w_);
  if (wants_grad({&w})) return EmbeddingFunction::apply(w, ids, scale, padding);
  return embed_rows(ids, w, scale);
}

// ---- the gated half of a feed-forward block -------------------------------------------

struct Gated {
  Tensor h, g, u;
};

Gated gated_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t act, bool keep) {
  const int64_t T = x.size(0), H = x.size(1), F = wg.size(0), ld = pad8(F);
  Gated r;
  r.h = empty({T, F}, x, x.scalar_type());
  if (keep || x.scalar_type() == at::kFloat) {
    r.g = empty({T, ld}, x, at::kFloat);
    r.u = empty({T, ld}, x, at::kFloat);
  }
  int32_t* status = status_of(x);
  On on(x);
  const int64_t size =
      tt_gated_linear_fwd_workspace_size(dtype_code(x), T, (int32_t)H, (int32_t)F);
  const Tensor ws = size ? bytes(size, x) : Tensor();
  check_status("tt_gated_linear_fwd",
               tt_gated_linear_fwd(dtype_code(x), T, (int32_t)H, (int32_t)F, ptr(x), ld_of(x),
                                   ptr(wg), ld_of(wg), ptr(wu), ld_of(wu), (int)act, out(r.h),
                                   (float*)out(r.g), (float*)out(r.u), ld, out(ws), size, status,
                                   on.stream));
  return r;
}

struct GatedFunction : Function<GatedFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu,
                        int64_t act) {
    const auto [x2, g2, u2] = rows16<3>({&x, &wg, &wu});
    Gated r = gated_forward(x2, g2, u2, act, true);
    // (with odd widths the copies that were made)
    ctx->save_for_backward({x2, g2, u2, r.g, r.u});
    ctx->saved_data["act"] = act;
    return r.h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    no_tangent("gated_linear", {&grad[0]});
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &wg = s[1], &wu = s[2], &g = s[3], &u = s[4];
    const int64_t T = x.size(0), H = x.size(1), F = wg.size(0);
    const Tensor dh = rows2d(grad[0]);
    Tensor dx, dwg, dwu;
    auto like = [&](int64_t n) {
      Tensor t = empty({n, H}, x, x.scalar_type());
      return T ? t : t.zero_();
    };
    if (ctx->needs_input_grad(0)) dx = like(T);
    if (ctx->needs_input_grad(1)) dwg = like(F);
    if (ctx->needs_input_grad(2)) dwu = like(F);
    int32_t* status = status_of(x);
    {
      On on(x);
      const int64_t size =
          tt_gated_linear_bwd_workspace_size(dtype_code(x), T, (int32_t)H, (int32_t)F);
      const Tensor ws = bytes(size, x);
      check_status(
          "tt_gated_linear_bwd",
          tt_gated_linear_bwd(dtype_code(x), T, (int32_t)H, (int32_t)F, ptr(x), ld_of(x), ptr(wg),
                              ld_of(wg), ptr(wu), ld_of(wu), (int)ctx->saved_data["act"].toInt(),
                              (const float*)ptr(g), (const float*)ptr(u), pad8(F), ptr(dh),
                              std::max(dh.stride(0), F), out(dx), out(dwg), out(dwu), out(ws), size,
                              status, on.stream));
    }
    return once("gated_linear", {dx, dwg, dwu, Tensor()});
  }
};

Tensor gated_linear(const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t act) {
  const char* op = "gated_linear";
  need_cuda(op, "x", x, x);
  need_cuda(op, "w_gate", wg, x);
  need_cuda(op, "w_up", wu, x);
  if (dtype_code(x) < 0 || wg.scalar_type() != x.scalar_type() ||
      wu.scalar_type() != x.scalar_type())
    type_error("gated_linear: x, w_gate and w_up must share one of float32/bfloat16/float16");
  if (x.dim() < 1 || x.size(-1) < 1) value_error("gated_linear: x must be [..., H]");
  const int64_t H = x.size(-1);
  if (wg.dim() != 2 || wg.size(0) < 1 || wg.size(1) != H)
    value_error("gated_linear: w_gate must be [F, " + std::to_string(H) + "]");
  if (wu.sizes() != wg.sizes()) value_error("gated_linear: w_up must have w_gate's shape");
  need_size(op, "a row's width", H + 257);
  if (wg.size(0) > (1 << 30) - 256)
    value_error("gated_linear: the number of features is limited to 2^30 - 256");
  const int64_t T = x.numel() / H;
  need_size(op, "a number of rows", T + 256);
  no_tangent(op, {&x, &wg, &wu});
  const Tensor x2 = x.dim() == 2 ? x : x.reshape({T, H});
  Tensor h;
  if (wants_grad({&x, &wg, &wu}))
    h = GatedFunction::apply(x2, wg, wu, act);
  else {
    const auto [xr, gr, ur] = rows16<3>({&x2, &wg, &wu});
    h = gated_forward(xr, gr, ur, act, false).h;
  }
  if (x.dim() == 2) return h;
  auto sizes = x.sizes().vec();
  sizes.back() = wg.size(0);
  return h.view(sizes);
}

// ---- the LM head's loss ------------------------------------------------------------------

struct CE {
  Tensor losses, lse, kept;
};

// (flat: losses [T] of one label a row)
CE ce_forward(const Tensor& x, const Tensor& w, const Tensor& labels, double scale, bool flat,
              bool keep) {
  const int64_t T = x.size(0), H = x.size(1), V = w.size(0), M = labels.size(1);
  CE r{flat ? empty({T}, x, at::kFloat) : empty({T, M}, x, at::kFloat),
       empty({T}, x, at::kFloat), Tensor()};
  const int64_t ld = keep ? tt_linear_ce_kept_ld(dtype_code(x), T, (int32_t)H, V) : 0;
  if (ld) r.kept = empty({T, ld}, x, at::kFloat);
  int32_t* status = status_of(x);
  On on(x);
  const int64_t size = tt_linear_ce_fwd_workspace_size(dtype_code(x), T, (int32_t)H, V, M);
  const Tensor ws = bytes(size, x);
  check_status("tt_linear_ce_fwd",
               tt_linear_ce_fwd(dtype_code(x), T, (int32_t)H, V, M, ptr(x), ld_of(x), ptr(w),
                                ld_of(w), (const int64_t*)ptr(labels), (float)scale,
                                (float*)out(r.losses), (float*)out(r.lse), (float*)out(r.kept),
                                out(ws), size, status, on.stream));
  return r;
}

struct LinearCEFunction : Function<LinearCEFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w,
                               const Tensor& labels, double scale, bool flat) {
    const auto [x2, w2] = rows16<2>({&x, &w});
    CE r = ce_forward(x2, w2, labels, scale, flat, true);
    // (with odd widths the copies that were made)
    ctx->save_for_backward({x2, w2, labels, r.lse, r.kept});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return {r.losses, r.lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list grads(5);
    if (!g[0].defined() && !g[1].defined()) return grads;
    no_tangent("linear_cross_entropy", {&g[0], &g[1]});
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &labels = s[2], &lse = s[3], &kept = s[4];
    const int64_t T = x.size(0), H = x.size(1), V = w.size(0), M = labels.size(1);
    for (int i = 0; i < 2; ++i)
      if (g[i].defined()) g[i] = g[i].resolve_neg().to(at::kFloat).contiguous();
    auto like = [&](int64_t n) {
      Tensor t = empty({n, H}, x, x.scalar_type());
      return T ? t : t.zero_();
    };
    Tensor dx, dw;
    if (ctx->needs_input_grad(0)) dx = like(T);
    if (ctx->needs_input_grad(1)) dw = like(V);
    int32_t* status = status_of(x);
    {
      On on(x);
      const int64_t size = tt_linear_ce_bwd_workspace_size(dtype_code(x), T, (int32_t)H, V, M);
      const Tensor ws = bytes(size, x);
      check_status("tt_linear_ce_bwd",
                   tt_linear_ce_bwd(dtype_code(x), T, (int32_t)H, V, M, ptr(x), ld_of(x), ptr(w),
                                    ld_of(w), (const int64_t*)ptr(labels),
                                    (float)ctx->saved_data["scale"].toDouble(),
                                    (const float*)ptr(lse), (const float*)ptr(kept),
                                    (const float*)ptr(g[0]), (const float*)ptr(g[1]), out(dx),
                                    out(dw), out(ws), size, status, on.stream));
    }
    return once("linear_cross_entropy", {dx, dw, Tensor(), Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor> linear_cross_entropy(const Tensor& x_, const Tensor& w,
                                                const Tensor& labels_, double scale) {
  const char* op = "linear_cross_entropy";
  need_cuda(op, "hidden", x_, x_);
  need_cuda(op, "weight", w, x_);
  need_cuda(op, "labels", labels_, x_);
  if (dtype_code(x_) < 0 || w.scalar_type() != x_.scalar_type())
    type_error("linear_cross_entropy: hidden and weight must share one of "
               "float32/bfloat16/float16");
  need_int(op, "labels", labels_);
  if (x_.dim() != 2 || x_.size(1) < 1)
    value_error("linear_cross_entropy: hidden must be [rows, H]");
  const int64_t T = x_.size(0), H = x_.size(1);
  if (w.dim() != 2 || w.size(0) < 1 || w.size(1) != H)
    value_error("linear_cross_entropy: weight must be [V, " + std::to_string(H) + "]");
  if (labels_.dim() < 1 || labels_.dim() > 2 || labels_.size(0) != T)
    value_error("linear_cross_entropy: labels must be [rows] or [rows, M]");
  need_size(op, "a row's width", H + 257);
  need_size(op, "a vocabulary", w.size(0) + 256);
  need_size(op, "a number of rows", T + 256);
  if (!std::isfinite((float)scale)) value_error("linear_cross_entropy: scale must be finite");
  const Tensor labels =
      (labels_.dim() == 2 ? labels_ : labels_.unsqueeze(1)).to(at::kLong).contiguous();
  need_size(op, "a number of labels a row", labels.size(1));
  no_tangent(op, {&x_, &w});
  Tensor losses, lse;
  if (wants_grad({&x_, &w})) {
    variable_list v = LinearCEFunction::apply(x_, w, labels, scale, labels_.dim() == 1);
    losses = v[0], lse = v[1];
  } else {
    const auto [x, wr] = rows16<2>({&x_, &w});
    CE r = ce_forward(x, wr, labels, scale, labels_.dim() == 1, false);
    losses = r.losses, lse = r.lse;
  }
  return {losses, lse};
}

// ---- the norm of many tensors ----------------------------------------------------------------

struct List {
  std::vector<Tensor> hold;                // dense copies of what is not dense
  std::vector<int32_t> dtypes;
  std::vector<int64_t> sizes;
  std::vector<void*> data;

  List(const char* op, const char* name, const std::vector<Tensor>& ts, bool written) {
    for (const Tensor& t : ts) {
      need_cuda(op, name, t, ts[0]);
      if (dtype_code(t) < 0)
        type_error(std::string(op) + ": " + name + " must be float32/bfloat16/float16");
      if (t.is_sparse()) type_error(std::string(op) + ": " + name + " must be dense tensors");
      if (written && t.is_neg())
        value_error(std::string(op) + ": " + name + " keeps its sign beside its memory "
                                                    "(resolve_neg)");
      no_tangent(op, {&t});
      const bool dense = t.is_non_overlapping_and_dense();
      if (written && !dense)
        value_error(std::string(op) + ": a tensor that is written must fill its memory without "
                                      "gaps or overlaps");
      hold.push_back(dense ? t : t.contiguous());  // (a norm does not ask for signs)
      dtypes.push_back(dtype_code(t));
      sizes.push_back(t.numel());
      data.push_back(const_cast<void*>(hold.back().const_data_ptr()));
    }
  }
  int32_t count() const { return (int32_t)sizes.size(); }
};

int64_t end_of(const List& l, size_t i) {
  return (int64_t)(uintptr_t)l.data[i] + l.sizes[i] * (l.dtypes[i] == TT_F32 ? 4 : 2);
}

// No byte is written twice, and none that another tensor of the call is read from.
void no_overlap(const char* op, const List& src, const List& dst) {
  std::vector<size_t> order;
  for (size_t i = 0; i < dst.sizes.size(); ++i)
    if (dst.sizes[i]) order.push_back(i);
  auto at = [](const List& l, size_t i) { return (int64_t)(uintptr_t)l.data[i]; };
  std::sort(order.begin(), order.end(),
            [&](size_t a, size_t b) { return at(dst, a) < at(dst, b); });
  for (size_t k = 1; k < order.size(); ++k)
    if (end_of(dst, order[k - 1]) > at(dst, order[k]))
      value_error(std::string(op) + ": two tensors that are written share memory");
  for (size_t i = 0; i < src.sizes.size(); ++i) {
    if (!src.sizes[i] || (src.data[i] == dst.data[i])) continue;
    const int64_t b = at(src, i), e = end_of(src, i);
    auto k = std::upper_bound(order.begin(), order.end(), b,
                              [&](int64_t v, size_t j) { return v < end_of(dst, j); });
    if (k != order.end() && at(dst, *k) < e)
      value_error(std::string(op) + ": a tensor shares memory with another one's output");
  }
}

double norm_type_of(const char* op, double p) {
  if (!(p == 1.0 || p == 2.0 || (std::isinf(p) && p > 0)))
    value_error(std::string(op) + ": norm_type must be 1, 2 or inf");
  return p;
}

Tensor grad_norm(const std::vector<Tensor>& grads, double norm_type) {
  const char* op = "grad_norm";
  norm_type_of(op, norm_type);
  if (grads.empty()) value_error("grad_norm: no tensors");
  torch::NoGradGuard no_grad;
  const List l(op, "a tensor", grads, false);
  Tensor norm = empty({}, grads[0], at::kFloat);
  On on(grads[0]);
  const int64_t size = tt_grad_norm_workspace_size(l.count());
  const Tensor ws = bytes(size, grads[0]);
  check_status("tt_grad_norm",
               tt_grad_norm(l.count(), l.dtypes.data(), l.sizes.data(), l.data.data(), norm_type,
                            (float*)out(norm), out(ws), size, on.stream));
  return norm;
}

Tensor clip_grad_norm(const std::vector<Tensor>& grads, double max_norm, double norm_type,
                      double eps, const OptTensor& norm_,
                      const std::optional<std::vector<Tensor>>& out_) {
  const char* op = "clip_grad_norm";
  norm_type_of(op, norm_type);
  if (grads.empty()) value_error("clip_grad_norm: no tensors");
  if (!(max_norm >= 0)) value_error("clip_grad_norm: max_norm must be at least 0");
  if (!(eps >= 0 && std::isfinite(eps))) value_error("clip_grad_norm: eps must be at least 0");
  torch::NoGradGuard no_grad;
  const std::vector<Tensor>& outs = out_ ? *out_ : grads;
  if (outs.size() != grads.size())
    value_error("clip_grad_norm: out must have one tensor for each gradient");
  for (size_t i = 0; i < grads.size(); ++i) {
    if (outs[i].sizes() != grads[i].sizes() || outs[i].scalar_type() != grads[i].scalar_type())
      value_error("clip_grad_norm: each tensor of out must have its gradient's shape and type");
    if (outs[i].strides() != grads[i].strides() && grads[i].numel() > 1 &&
        !(outs[i].is_contiguous() && grads[i].is_contiguous()))
      value_error("clip_grad_norm: each tensor of out must have its gradient's strides");
  }
  const List src(op, "a gradient", grads, true), dst(op, "a tensor of out", outs, true);
  if (outs[0].device() != grads[0].device())
    throw std::runtime_error("clip_grad_norm: out is on another device than the gradients");
  no_overlap(op, src, dst);
  Tensor norm = empty({}, grads[0], at::kFloat), given;
  if (norm_ && norm_->defined()) {
    need_cuda(op, "norm", *norm_, grads[0]);
    if (norm_->numel() != 1 || norm_->scalar_type() != at::kFloat)
      type_error("clip_grad_norm: norm must be one float32");
    given = *norm_;
    // (every block reads it, others may have written by then)
    const int64_t at = (int64_t)(uintptr_t)given.const_data_ptr();
    for (size_t i = 0; i < dst.sizes.size(); ++i)
      if (dst.sizes[i] && at + 4 > (int64_t)(uintptr_t)dst.data[i] && at < end_of(dst, i))
        value_error("clip_grad_norm: norm is a part of a tensor that is written");
  }
  // what is written has a new version: autograd refuses what it saved of it (and
  // inference tensors are not written outside inference mode)
  for (const Tensor& t : outs) t.unsafeGetTensorImpl()->bump_version();
  On on(grads[0]);
  const int64_t size = tt_grad_norm_workspace_size(src.count());
  const Tensor ws = bytes(size, grads[0]);
  check_status("tt_clip_grad_norm",
               tt_clip_grad_norm(src.count(), src.dtypes.data(), src.sizes.data(),
                                 src.data.data(), dst.data.data(), norm_type,
                                 (const float*)ptr(given), (float)max_norm, (float)eps,
                                 (float*)out(norm), out(ws), size, on.stream));
  return norm;
}

}  // namespace

void bind_train_ops(py::module_& m) {
  using Unlocked = py::call_guard<py::gil_scoped_release>;
  m.def("embedding", &embedding, Unlocked());
  m.def("gated_linear", &gated_linear, Unlocked());
  m.def("linear_cross_entropy", &linear_cross_entropy, Unlocked());
  m.def("grad_norm", &grad_norm, Unlocked());
  m.def("clip_grad_norm", &clip_grad_norm, Unlocked());
}
