// The torch.library operators around the attention: a block's residual and norms, 8-bit tokens and products, the optimiser's step.
#include <algorithm>

#include "helpers.h"

namespace {

// ------------------------------------------------------------------------------------------------
// residual and norms.  x, y [batch, tokens, channels] contiguous; gate [batch, 1 | tokens, 1] or [batch, 1, channels]
// ------------------------------------------------------------------------------------------------
struct NormShape {
  bool norm, post;
  int64_t kind;
  double eps, post_eps;
};

s3r_residual_norm norm_args(const Tensor& x, const optional<Tensor>& y, const optional<Tensor>& weight, const optional<Tensor>& bias,
                            const optional<Tensor>& scale, const optional<Tensor>& gate, const optional<Tensor>& post_weight,
                            const optional<Tensor>& post_bias, const NormShape& n) {
  need_cuda(x, "x");
  TORCH_CHECK(x.dim() == 3 && x.is_contiguous(), "residual_norm: x must be a contiguous [batch, tokens, channels]");
  s3r_residual_norm a = {};
  a.batch = x.size(0);
  a.tokens = x.size(1);
  TORCH_CHECK(x.size(2) >= 1 && x.size(2) <= 8192, "residual_norm: ", x.size(2), " channels (1 to 8192)");
  a.channels = static_cast<int>(x.size(2));
  a.kind = static_cast<int>(n.kind);
  a.post = n.post;
  a.eps = static_cast<float>(n.eps);
  a.post_eps = static_cast<float>(n.post_eps);
  a.x_type = a.y_type = a.h_type = type_of(x, "x");
  a.x = x.data_ptr();
  if (y.has_value()) {
    TORCH_CHECK(y->device() == x.device() && y->sizes() == x.sizes() && y->is_contiguous(), "residual_norm: y must be like x, contiguous");
    a.y = y->data_ptr();
    a.y_type = type_of(*y, "y");
  }
  a.param_type = -1;
  auto param = [&](const optional<Tensor>& t, const char* name) -> const void* {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->device() == x.device() && t->dim() == 1 && t->size(0) == x.size(2) && t->is_contiguous(), "residual_norm: ", name,
                " must be a contiguous [channels] on x's device");
    const int type = type_of(*t, name);
    TORCH_CHECK(a.param_type < 0 || a.param_type == type, "residual_norm: parameters of one type");
    a.param_type = type;
    return t->data_ptr();
  };
  a.weight = param(weight, "weight");
  a.bias = param(bias, "bias");
  a.scale = param(scale, "scale");
  a.post_weight = param(post_weight, "post_weight");
  a.post_bias = param(post_bias, "post_bias");
  if (a.param_type < 0) a.param_type = S3R_F32;
  if (gate.has_value()) {
    const Tensor& g = *gate;
    TORCH_CHECK(g.device() == x.device() && g.dim() == 3 && g.size(0) == x.size(0), "residual_norm: gate must have x's batch");
    a.gate = g.data_ptr();
    a.gate_type = type_of(g, "gate");
    if (g.size(2) == 1) {
      TORCH_CHECK(g.size(1) == 1 || g.size(1) == x.size(1), "residual_norm: gate has ", g.size(1), " tokens");
      a.gate_mode = S3R_GATE_ROW;
      a.gate_stride_b = g.stride(0);
      a.gate_stride_t = g.size(1) == 1 ? 0 : g.stride(1);
    } else {
      TORCH_CHECK(g.size(1) == 1 && g.size(2) == x.size(2) && g.stride(2) == 1, "residual_norm: a gate per channel is [batch, 1, channels]");
      a.gate_mode = S3R_GATE_CHANNEL;
      a.gate_stride_b = g.stride(0);
    }
  }
  return a;
}

struct NormInputs {
  Tensor x;
  optional<Tensor> y, w, b, s, g, pw, pb;
};

// (r, h, stats), undefined where there is nothing to compute or to keep
std::tuple<Tensor, Tensor, Tensor> run_norm_fwd(const NormInputs& in, const NormShape& n, at::ScalarType h_type, bool keep) {
  const Tensor& x = in.x;
  s3r_residual_norm a = norm_args(x, in.y, in.w, in.b, in.s, in.g, in.pw, in.pb, n);
  c10::cuda::CUDAGuard guard(x.device());
  Tensor r, h, stats;
  if (in.y.has_value()) r = fresh_like(x);
  if (n.norm) h = fresh(x.sizes(), x, h_type), a.h_type = type_of(h, "the norm's result");
  if (keep) stats = fresh({4, a.batch * a.tokens}, x, at::kFloat);
  if (x.numel()) {
    a.r = pointer(r);
    a.h = pointer(h);
    a.stats = keep ? f32(stats) : nullptr;
    check(s3r_residual_norm_fwd(&a, stream()), "s3r_residual_norm_fwd");
  }
  return {r, h, stats};
}
std::tuple<Tensor, Tensor, Tensor> residual_norm_fwd(const Tensor& x, const optional<Tensor>& y, const optional<Tensor>& weight,
                                                     const optional<Tensor>& bias, const optional<Tensor>& scale,
                                                     const optional<Tensor>& gate, const optional<Tensor>& post_weight,
                                                     const optional<Tensor>& post_bias, bool norm, bool post, int64_t kind, double eps,
                                                     double post_eps, at::ScalarType h_type, bool keep) {
  auto [r, h, stats] = run_norm_fwd({x, y, weight, bias, scale, gate, post_weight, post_bias}, {norm, post, kind, eps, post_eps}, h_type, keep);
  return {r.defined() ? r : none(x), h.defined() ? h : fresh({0}, x, h_type), stats.defined() ? stats : fresh({0, x.size(0) * x.size(1)}, x, at::kFloat)};
}

std::tuple<Tensor, Tensor, Tensor> residual_norm_int8(const Tensor& x, const optional<Tensor>& y, const optional<Tensor>& weight,
                                                      const optional<Tensor>& bias, const optional<Tensor>& scale,
                                                      const optional<Tensor>& gate, const optional<Tensor>& post_weight,
                                                      const optional<Tensor>& post_bias, bool post, int64_t kind, double eps,
                                                      double post_eps) {
  s3r_residual_norm a = norm_args(x, y, weight, bias, scale, gate, post_weight, post_bias, {true, post, kind, eps, post_eps});
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = a.batch * a.tokens, pitch = (a.channels + 15) / 16 * 16;
  Tensor r = y.has_value() ? fresh_like(x) : none(x), q = fresh({a.batch, a.tokens, pitch}, x, at::kChar).narrow(2, 0, a.channels);
  Tensor s = fresh({a.batch, a.tokens}, x, at::kFloat);
  if (rows) {
    a.r = y.has_value() ? r.data_ptr() : nullptr;
    a.q = static_cast<int8_t*>(q.data_ptr());
    a.q_pitch = pitch;
    a.q_scale = f32(s);
    check(s3r_residual_norm_fwd(&a, stream()), "s3r_residual_norm_fwd");
  }
  return {r, q, s};
}

// Gradients of (x, y, weight, bias, scale, gate, post_weight, post_bias); those that `want` (a bit each) does not name are undefined (from the
// operator: without elements).
enum { kX = 1, kY = 2, kWeight = 4, kBias = 8, kScale = 16, kGate = 32, kPostWeight = 64, kPostBias = 128 };
std::vector<Tensor> run_norm_bwd(const Tensor& r, const optional<Tensor>& y, const optional<Tensor>& weight, const optional<Tensor>& scale,
                                 const optional<Tensor>& gate, const optional<Tensor>& post_weight, const optional<Tensor>& post_bias,
                                 const Tensor& stats, const optional<Tensor>& dr, const optional<Tensor>& dh, optional<at::ScalarType> branch,
                                 bool post, int64_t kind, int64_t want, at::ScalarType param_type) {
  s3r_residual_norm f = norm_args(r, y, weight, {}, scale, gate, post_weight, post_bias, {true, post, kind, 0., 0.});
  TORCH_CHECK(y.has_value() || !post, "residual_norm: the branch of a post norm is missing");
  c10::cuda::CUDAGuard guard(r.device());
  f.r = r.data_ptr();
  if (!y.has_value() && branch.has_value()) {                   // there was a branch, of this type, that is not read any more
    TORCH_CHECK(!(want & (kScale | kGate)), "residual_norm: the branch is missing");
    f.y = f.r;
    f.y_type = type_of(at::empty({0}, at::TensorOptions().dtype(*branch)), "the branch");
  }
  f.stats = f32(stats);
  f.param_type = type_of(at::empty({0}, at::TensorOptions().dtype(param_type)), "parameters");
  const int64_t rows = f.batch * f.tokens;
  auto incoming = [&](const optional<Tensor>& t, const char* name) {
    if (!t.has_value()) return;
    TORCH_CHECK(t->device() == r.device() && t->sizes() == r.sizes() && t->is_contiguous(), "residual_norm: ", name, " must be like x, contiguous");
  };
  incoming(dr, "the gradient of the sum");
  incoming(dh, "the gradient of the norm");
  TORCH_CHECK(!dr.has_value() || dr->scalar_type() == r.scalar_type(), "residual_norm: the gradient of the sum has another type than the sum");
  if (dh.has_value()) f.h_type = type_of(*dh, "the gradient of the norm");
  if (!dh.has_value()) want &= ~(kWeight | kBias);
  auto channels = [&](int64_t bit) { return want & bit ? fresh({r.size(2)}, r, param_type) : Tensor(); };
  Tensor dx = fresh_like(r), dy = want & kY && branch.has_value() ? fresh(r.sizes(), r, *branch) : Tensor();
  Tensor dw = channels(kWeight), db = channels(kBias), ds = channels(kScale), dpw = channels(kPostWeight), dpb = channels(kPostBias);
  Tensor dg, dg_row;
  s3r_residual_norm_grad g = {};
  if (want & kGate) {
    if (f.gate_mode == S3R_GATE_ROW) {
      dg_row = fresh({f.batch, f.tokens, 1}, r, at::kFloat);
      g.d_gate_row = f32(dg_row);
    } else {
      dg = fresh({f.batch, 1, r.size(2)}, r, gate->scalar_type());
      g.d_gate_channel = dg.data_ptr();
    }
  }
  if (rows == 0) {
    for (Tensor* t : {&dw, &db, &ds, &dg, &dpw, &dpb})
      if (t->defined()) t->zero_();
  } else {
    g.dr = pointer(dr);
    g.dh = pointer(dh);
    g.dx = dx.data_ptr();
    g.dy = pointer(dy);
    g.d_weight = pointer(dw);
    g.d_bias = pointer(db);
    g.d_scale = pointer(ds);
    g.d_post_weight = pointer(dpw);
    g.d_post_bias = pointer(dpb);
    int sums = 0;
    for (const Tensor* t : {&dw, &db, &ds, &dpw, &dpb, &dg}) sums += t->defined();
    Tensor ws;
    if (sums) {
      g.workspace_bytes = s3r_residual_norm_bwd_workspace_bytes(f.batch, f.tokens, f.channels, f.gate_mode) / 6 * sums;
      ws = fresh({static_cast<int64_t>(g.workspace_bytes)}, r, at::kByte);
      g.workspace = ws.data_ptr();
    }
    check(s3r_residual_norm_bwd(&f, &g, stream()), "s3r_residual_norm_bwd");
  }
  if (dg_row.defined()) dg = (gate->size(1) == 1 ? dg_row.sum(1, true) : dg_row).to(gate->scalar_type());
  return {dx, dy, dw, db, ds, dg, dpw, dpb};
}

std::vector<Tensor> residual_norm_bwd(const Tensor& r, const optional<Tensor>& y, const optional<Tensor>& weight,
                                      const optional<Tensor>& scale, const optional<Tensor>& gate, const optional<Tensor>& post_weight,
                                      const optional<Tensor>& post_bias, const Tensor& stats, const optional<Tensor>& dr,
                                      const optional<Tensor>& dh, optional<at::ScalarType> branch, bool post, int64_t kind, int64_t want,
                                      at::ScalarType param_type) {
  auto g = run_norm_bwd(r, y, weight, scale, gate, post_weight, post_bias, stats, dr, dh, branch, post, kind, want, param_type);
  for (Tensor& t : g)
    if (!t.defined()) t = none(r);
  return g;
}

std::tuple<Tensor, Tensor, Tensor> call_norm_fwd(const Tensor& x, const optional<Tensor>& y, const optional<Tensor>& w, const optional<Tensor>& b,
                                                 const optional<Tensor>& s, const optional<Tensor>& g, const optional<Tensor>& pw,
                                                 const optional<Tensor>& pb, const NormShape& n, at::ScalarType h_type, bool keep) {
  S3R_DISPATCHED(residual_norm_fwd)(x, y, w, b, s, g, pw, pb, n.norm, n.post, n.kind, n.eps, n.post_eps, h_type, keep);
}
std::vector<Tensor> call_norm_bwd(const Tensor& r, const optional<Tensor>& y, const optional<Tensor>& w, const optional<Tensor>& s,
                                  const optional<Tensor>& g, const optional<Tensor>& pw, const optional<Tensor>& pb, const Tensor& stats,
                                  const optional<Tensor>& dr, const optional<Tensor>& dh, optional<at::ScalarType> branch, bool post,
                                  int64_t kind, int64_t want, at::ScalarType param_type) {
  S3R_DISPATCHED(residual_norm_bwd)(r, y, w, s, g, pw, pb, stats, dr, dh, branch, post, kind, want, param_type);
}

std::tuple<Tensor, Tensor, Tensor> call_norm_int8(const NormInputs& in, bool post, int64_t kind, double eps, double post_eps) {
  S3R_DISPATCHED(residual_norm_int8)(in.x, in.y, in.w, in.b, in.s, in.g, in.pw, in.pb, post, kind, eps, post_eps);
}

struct NormNode : torch::autograd::Function<NormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& y, const optional<Tensor>& w,
                               const optional<Tensor>& b, const optional<Tensor>& s, const optional<Tensor>& g, const optional<Tensor>& pw,
                               const optional<Tensor>& pb, bool norm, bool post, int64_t kind, double eps, double post_eps, int64_t h_type) {
    at::AutoDispatchBelowADInplaceOrView below;
    const bool branch = y.has_value();
    const NormShape shape = {norm, post, kind, eps, post_eps};
    const auto type = static_cast<at::ScalarType>(h_type);
    auto [r, h, stats] = plain(x) ? run_norm_fwd({x, y, w, b, s, g, pw, pb}, shape, type, true) : call_norm_fwd(x, y, w, b, s, g, pw, pb, shape, type, true);
    // the branch itself is needed for the gradients of what multiplies it
    const bool needs_y = branch && (post || (s.has_value() && s->requires_grad()) || (g.has_value() && g->requires_grad()));
    at::ScalarType param = at::kFloat;
    int64_t present = 1, bit = 2;                 // which of the eight tensors are there: only they have an edge
    for (const auto* t : {&y, &w, &b, &s, &g, &pw, &pb}) {
      if (t->has_value()) present |= bit;
      if (t->has_value() && t != &y && t != &g) param = (*t)->scalar_type();
      bit *= 2;
    }
    ctx->save_for_backward({branch ? r : x, needs_y ? *y : Tensor(), value(w), value(s), value(g), value(pw), value(pb), stats});
    ctx->saved_data["ints"] = std::vector<int64_t>{present, branch, static_cast<int64_t>(branch ? y->scalar_type() : x.scalar_type()), post, kind,
                                                  static_cast<int64_t>(param)};
    ctx->set_materialize_grads(false);
    variable_list out;
    if (branch) out.push_back(r);
    if (norm) out.push_back(h);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return once(g, [&] { return gradients(ctx, g); });
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& incoming) {
    variable_list out(14);
    const auto s = ctx->get_saved_variables();
    const auto ints = ctx->saved_data["ints"].toIntVector();
    const int64_t present = ints[0];
    const bool branch = ints[1], post = ints[3];
    auto given = [](const Tensor& t) { return t.defined() ? optional<Tensor>(t.contiguous()) : optional<Tensor>(); };
    const optional<Tensor> dr = branch ? given(incoming[0]) : optional<Tensor>();
    const optional<Tensor> dh = incoming.size() > (branch ? 1u : 0u) ? given(incoming.back()) : optional<Tensor>();
    if (!dr.has_value() && !dh.has_value()) return out;
    int64_t want = 0;
    for (int i = 0, edge = 0; i < 8; ++i)
      if (present >> i & 1 && ctx->needs_input_grad(edge++)) want |= int64_t{1} << i;
    if (!branch) want &= kX | kWeight | kBias;
    // a branch that nothing is multiplied with is not kept, only its type
    optional<at::ScalarType> branch_type;
    if (branch) branch_type = static_cast<at::ScalarType>(ints[2]);
    const auto& backward = plain(s[0]) ? run_norm_bwd : call_norm_bwd;
    const auto g = backward(s[0], maybe(s[1]), maybe(s[2]), maybe(s[3]), maybe(s[4]), maybe(s[5]), maybe(s[6]), s[7], dr, dh, branch_type, post, ints[4],
                                 want, static_cast<at::ScalarType>(ints[5]));
    for (int i = 0; i < 8; ++i)
      if (want >> i & 1 && g[i].defined() && (dh.has_value() || !(i == 2 || i == 3))) out[i] = g[i];
    return out;
  }
};

// [.., tokens, channels] as a contiguous [batch, tokens, channels], which begins anywhere: the kernels look at addresses themselves
Tensor as_rows(const Tensor& t) {
  const int64_t d = t.dim(), tokens = d > 1 ? t.size(d - 2) : 1;
  int64_t batch = 1;
  if (d == 3) return t.contiguous();
  for (int64_t i = 0; i + 2 < d; ++i) batch *= t.size(i);
  return t.contiguous().view({batch, tokens, t.size(d - 1)});
}
optional<Tensor> gate_of(const optional<Tensor>& gate, const Tensor& x) {
  if (!gate.has_value()) return {};
  const Tensor& g = *gate;
  TORCH_CHECK(g.dim() == x.dim(), "residual_norm: gate must have as many dimensions as x");
  const int64_t d = x.dim(), tokens = d > 1 ? g.size(d - 2) : 1, channels = g.size(d - 1);
  TORCH_CHECK((channels == 1 && (tokens == 1 || tokens == (d > 1 ? x.size(d - 2) : 1))) || (channels == x.size(d - 1) && tokens == 1),
              "residual_norm: gate must be [.., tokens or 1, 1] or [.., 1, channels], got ", g.sizes(), " for ", x.sizes());
  std::vector<int64_t> whole(g.sizes().begin(), g.sizes().end());
  int64_t batch = 1;
  for (int64_t i = 0; i + 2 < d; ++i) {
    TORCH_CHECK(g.size(i) == 1 || g.size(i) == x.size(i), "residual_norm: gate of ", g.sizes(), " for ", x.sizes());
    whole[i] = x.size(i);
    batch *= x.size(i);
  }
  const Tensor rows = g.expand(whole).reshape({batch, tokens, channels});
  return channels > 1 && rows.stride(2) != 1 ? rows.contiguous() : rows;
}
NormInputs norm_inputs(const Tensor& x, const optional<Tensor>& y, const optional<Tensor>& w, const optional<Tensor>& b, const optional<Tensor>& s,
                       const optional<Tensor>& gate, const optional<Tensor>& pw, const optional<Tensor>& pb, bool norm, bool post, int64_t kind) {
  TORCH_CHECK(x.dim() >= 1, "residual_norm: x needs a dimension");
  TORCH_CHECK(kind == S3R_NORM_LAYER || kind == S3R_NORM_RMS, "residual_norm: kind ", kind);
  TORCH_CHECK(norm || (!w.has_value() && !b.has_value()), "residual_norm: weight and bias belong to a norm");
  TORCH_CHECK(post || (!pw.has_value() && !pb.has_value()), "residual_norm: post_weight and post_bias belong to a post norm");
  TORCH_CHECK(y.has_value() || (!s.has_value() && !gate.has_value() && !post), "residual_norm: scale, gate and post_norm need a branch y");
  TORCH_CHECK(y.has_value() || norm, "residual_norm: nothing to compute without a branch and without a norm");
  TORCH_CHECK(!y.has_value() || y->sizes() == x.sizes(), "residual_norm: y ", y.has_value() ? y->sizes() : x.sizes(), " is not like x ", x.sizes());
  NormInputs in = {as_rows(x), {}, w, b, s, gate_of(gate, x), pw, pb};
  if (y.has_value()) in.y = as_rows(*y);
  of_one_type({&in.w, &in.b, &in.s, &in.pw, &in.pb});
  return in;
}

// (r, h); what is not computed - r without a branch, h without a norm - is x
std::tuple<Tensor, Tensor> residual_norm(const Tensor& x, const optional<Tensor>& y, const optional<Tensor>& w, const optional<Tensor>& b,
                                         const optional<Tensor>& s, const optional<Tensor>& gate, const optional<Tensor>& pw,
                                         const optional<Tensor>& pb, bool norm, bool post, int64_t kind, double eps, double post_eps,
                                         at::ScalarType h_type) {
  const NormInputs in = norm_inputs(x, y, w, b, s, gate, pw, pb, norm, post, kind);
  if (wants_grad(x, value(y), value(w), value(b), value(s), value(gate), value(pw), value(pb))) {
    const auto out = NormNode::apply(in.x, in.y, in.w, in.b, in.s, in.g, in.pw, in.pb, norm, post, kind, eps, post_eps,
                                     static_cast<int64_t>(h_type));
    return {y.has_value() ? in_shape(out[0], x.sizes()) : x, norm ? in_shape(out.back(), x.sizes()) : x};
  }
  const NormShape shape = {norm, post, kind, eps, post_eps};
  auto [r, h, stats] = plain(x) ? run_norm_fwd(in, shape, h_type, false)
                                : call_norm_fwd(in.x, in.y, in.w, in.b, in.s, in.g, in.pw, in.pb, shape, h_type, false);
  return {y.has_value() ? in_shape(r, x.sizes()) : x, norm ? in_shape(h, x.sizes()) : x};
}

std::tuple<Tensor, Tensor, Tensor> residual_norm_to_int8(const Tensor& x, const optional<Tensor>& y, const optional<Tensor>& w,
                                                         const optional<Tensor>& b, const optional<Tensor>& s, const optional<Tensor>& gate,
                                                         const optional<Tensor>& pw, const optional<Tensor>& pb, bool post, int64_t kind,
                                                         double eps, double post_eps) {
  TORCH_CHECK(!wants_grad(x, value(y), value(w), value(b), value(s), value(gate), value(pw), value(pb)),
              "residual_norm_int8 is forward-only: call it under torch.no_grad()");
  const NormInputs in = norm_inputs(x, y, w, b, s, gate, pw, pb, true, post, kind);
  auto [r, q, qs] = plain(x) ? residual_norm_int8(in.x, in.y, in.w, in.b, in.s, in.g, in.pw, in.pb, post, kind, eps, post_eps)
                             : call_norm_int8(in, post, kind, eps, post_eps);
  return {y.has_value() ? in_shape(r, x.sizes()) : x, in_shape(q, x.sizes()), in_shape(qs, x.sizes().slice(0, x.dim() - 1))};
}

// ------------------------------------------------------------------------------------------------
// 8-bit tokens and products
// ------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x) {
  need_cuda(x, "x");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "quantize_tokens: x needs channels");
  const int type = type_of(x, "x");
  TORCH_CHECK(x.size(-1) < (int64_t{1} << 31), "quantize_tokens: ", x.size(-1), " channels");
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t K = x.size(-1), pitch = (K + 15) / 16 * 16, rows = x.numel() / K;
  Tensor in = x.reshape({rows, K});
  if (in.stride(1) != 1 || (rows > 1 && in.stride(0) < K)) in = in.contiguous();
  Tensor q = fresh({rows, pitch}, x, at::kChar).narrow(1, 0, K), s = fresh(x.sizes().slice(0, x.dim() - 1), x, at::kFloat);
  if (rows)
    check(s3r_quantize_rows(in.data_ptr(), type, rows > 1 ? in.stride(0) : K, static_cast<int8_t*>(q.data_ptr()), pitch, f32(s), rows, static_cast<int>(K),
                            stream()), "s3r_quantize_rows");
  return {q.view(x.sizes()), s};
}

// [.., K] bytes as rows whose base and pitch are multiples of 16
Tensor byte_rows(const Tensor& t, int64_t rows, int64_t K) {
  Tensor r = t.reshape({rows, K});
  const bool fits = (K == 1 || r.stride(1) == 1) && (rows <= 1 || (r.stride(0) >= K && r.stride(0) % 16 == 0)) &&
                    reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0;
  if (fits) return r;                        // a single row has no pitch
  if (K > 1 && r.stride(1) != 1) r = r.contiguous();
  const int64_t pitch = (K + 15) / 16 * 16;
  Tensor whole = fresh({rows, pitch}, t, at::kChar);
  check(s3r_pad_rows(static_cast<const int8_t*>(r.data_ptr()), rows > 1 ? r.stride(0) : K, static_cast<int8_t*>(whole.data_ptr()), pitch, rows,
                     static_cast<int>(K), stream()), "s3r_pad_rows");
  return whole.narrow(1, 0, K);
}

Tensor int8_product(const Tensor& q, const Tensor& q_scale, const Tensor& weight, const Tensor& weight_scale, const optional<Tensor>& bias,
                   at::ScalarType out_type) {
  need_cuda(q, "q");
  TORCH_CHECK(q.scalar_type() == at::kChar && weight.scalar_type() == at::kChar, "int8_linear: q and weight must be int8");
  TORCH_CHECK(q.dim() >= 1 && weight.dim() == 2 && q.size(-1) == weight.size(1), "int8_linear: q [.., K] and weight [N, K], got ", q.sizes(), " and ", weight.sizes());
  const int64_t K = weight.size(1), N = weight.size(0);
  TORCH_CHECK(K >= 1 && K <= 65536, "int8_linear: K = ", K, " (1 to 65536)");
  TORCH_CHECK(N >= 1 && N < (int64_t{1} << 30), "int8_linear: N = ", N);
  const int64_t M = q.numel() / K;
  TORCH_CHECK(q_scale.scalar_type() == at::kFloat && q_scale.numel() == M, "int8_linear: one fp32 scale per token, got ", q_scale.sizes(), " of ", q_scale.scalar_type());
  TORCH_CHECK(weight_scale.scalar_type() == at::kFloat && weight_scale.dim() == 1 && weight_scale.size(0) == N, "int8_linear: one fp32 scale per channel, got ",
              weight_scale.sizes(), " of ", weight_scale.scalar_type());
  TORCH_CHECK(!bias.has_value() || (bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == N), "int8_linear: bias must be fp32 [N]");
  for (const Tensor* t : {&q_scale, &weight, &weight_scale}) TORCH_CHECK(t->device() == q.device(), "int8_linear: tensors of one device");
  TORCH_CHECK(!bias.has_value() || bias->device() == q.device(), "int8_linear: tensors of one device");
  c10::cuda::CUDAGuard guard(q.device());
  std::vector<int64_t> shape(q.sizes().begin(), q.sizes().end());
  shape.back() = N;
  Tensor out = fresh(shape, q, out_type);
  const int type = type_of(out, "the result");
  if (M == 0) return out;
  const Tensor a = byte_rows(q, M, K), b = byte_rows(weight, N, K), as = q_scale.contiguous(), bs = weight_scale.contiguous();
  const Tensor add = bias.has_value() ? bias->contiguous() : Tensor();
  const int64_t whole = (K + 15) / 16 * 16;
  check(s3r_int8_linear(static_cast<const int8_t*>(a.data_ptr()), M > 1 ? a.stride(0) : whole, f32(as), static_cast<const int8_t*>(b.data_ptr()),
                        N > 1 ? b.stride(0) : whole, f32(bs), add.defined() ? f32(add) : nullptr, out.data_ptr(), type, M, static_cast<int>(N),
                        static_cast<int>(K), stream()), "s3r_int8_linear");
  return out;
}

// ------------------------------------------------------------------------------------------------
// the optimiser
// ------------------------------------------------------------------------------------------------
Tensor norm_of(at::TensorList tensors) {
  TORCH_CHECK(!tensors.empty(), "grad_norm: no tensors");
  std::vector<Tensor> kept;
  std::vector<const void*> ptr;
  std::vector<int64_t> counts;
  std::vector<int> types;
  for (const Tensor& t : tensors) {
    need_cuda(t, "a gradient");
    TORCH_CHECK(t.device() == tensors[0].device(), "grad_norm: tensors of one device");
    kept.push_back(t.contiguous());
    ptr.push_back(kept.back().data_ptr());
    counts.push_back(t.numel());
    types.push_back(type_of(t, "a gradient"));
  }
  c10::cuda::CUDAGuard guard(tensors[0].device());
  const int n = static_cast<int>(ptr.size());
  const size_t bytes = s3r_grad_norm_workspace_bytes(n, counts.data());
  const Tensor ws = fresh({static_cast<int64_t>(bytes)}, tensors[0], at::kByte);
  Tensor norm = fresh({}, tensors[0], at::kFloat);
  check(s3r_grad_norm(n, ptr.data(), counts.data(), types.data(), f32(norm), ws.data_ptr(), bytes, stream()), "s3r_grad_norm");
  return norm;
}

void need_states(const Tensor& p, const Tensor& m, const Tensor& v, const Tensor* e) {
  const at::ScalarType type = e ? at::kByte : at::kFloat;
  for (const Tensor* t : {&m, &v})
    TORCH_CHECK(t->device() == p.device() && t->scalar_type() == type && t->sizes() == p.sizes() && t->is_contiguous(),
                "adamw: a state must be contiguous ", type, " of its parameter's shape ", p.sizes(), ", got ", t->scalar_type(), " ", t->sizes());
  if (e)
    TORCH_CHECK(e->device() == p.device() && e->scalar_type() == at::kByte && e->dim() == 2 && e->size(0) == 2 && e->size(1) == (p.numel() + 255) / 256 &&
                    (e->numel() == 0 || e->stride(1) == 1), "adamw: scales of ", p.numel(), " elements must be uint8 [2, ", (p.numel() + 255) / 256, "], got ", e->sizes());
}

// scales: those of the 8-bit states, one behind the other.  A list with gaps (Tensor?[]) cannot be declared as written: tracers
// take none of its gaps, and a list that is not declared is read again from before the step.
void adamw_update(at::TensorList params, at::TensorList grads, at::TensorList exp_avg, at::TensorList exp_avg_sq, const Tensor& step,
                at::TensorList scales, double lr, const optional<Tensor>& lr_tensor, double beta1, double beta2, double eps,
                double weight_decay, const optional<Tensor>& norm, double max_norm, int64_t seed, at::OptionalIntArrayRef numbers) {
  const size_t n = params.size();
  TORCH_CHECK(n > 0, "adamw: no tensors");
  TORCH_CHECK(grads.size() == n && exp_avg.size() == n && exp_avg_sq.size() == n, "adamw: ", n, " parameters, ", grads.size(), " gradients, ",
              exp_avg.size(), " and ", exp_avg_sq.size(), " states");
  const at::Device device = params[0].device();
  TORCH_CHECK(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "adamw: betas are in [0, 1)");
  TORCH_CHECK(eps >= 0 && weight_decay >= 0, "adamw: eps and weight_decay are not negative");
  TORCH_CHECK(step.device() == device && step.scalar_type() == at::kLong && step.numel() == 1, "adamw: step must be one int64 on the parameters' device");
  for (const auto* t : {&norm, &lr_tensor})
    TORCH_CHECK(!t->has_value() || ((*t)->device() == device && (*t)->scalar_type() == at::kFloat && (*t)->numel() == 1),
                "adamw: grad_norm and lr as tensors must be one fp32 on the parameters' device");
  TORCH_CHECK(max_norm <= 0 || norm.has_value(), "adamw: max_norm needs grad_norm");
  std::vector<uint32_t> number_of;
  if (numbers.has_value()) {
    TORCH_CHECK(numbers->size() == n, "adamw: ", n, " parameters, ", numbers->size(), " numbers");
    for (const int64_t i : *numbers) {
      TORCH_CHECK(i >= 0 && i < (1 << 24), "adamw: numbers are 0 to 2^24 - 1, got ", i);
      number_of.push_back(static_cast<uint32_t>(i));
    }
  }
  std::vector<Tensor> kept;
  std::vector<void*> p(n), m(n), v(n);
  std::vector<const void*> g(n);
  std::vector<uint8_t*> me(n, nullptr), ve(n, nullptr);
  std::vector<int64_t> counts(n);
  std::vector<int> p_types(n), g_types(n);
  size_t scale_of = 0;
  for (size_t i = 0; i < n; ++i) {
    need_cuda(params[i], "a parameter");
    TORCH_CHECK(params[i].device() == device && grads[i].device() == device, "adamw: tensors of one device");
    TORCH_CHECK(params[i].is_contiguous(), "adamw: parameters must be contiguous");
    TORCH_CHECK(grads[i].sizes() == params[i].sizes(), "adamw: gradient ", grads[i].sizes(), " of parameter ", params[i].sizes());
    const Tensor* scale = nullptr;
    if (exp_avg[i].scalar_type() == at::kByte) {
      TORCH_CHECK(scale_of < scales.size(), "adamw: an 8-bit state has no scales");
      scale = &scales[scale_of++];
    }
    need_states(params[i], exp_avg[i], exp_avg_sq[i], scale);
    if (scale) {
      me[i] = static_cast<uint8_t*>(scale->data_ptr());
      ve[i] = me[i] + scale->stride(0);
    }
    kept.push_back(grads[i].contiguous());
    g[i] = kept.back().data_ptr();
    p[i] = params[i].data_ptr();
    m[i] = exp_avg[i].data_ptr();
    v[i] = exp_avg_sq[i].data_ptr();
    counts[i] = params[i].numel();
    p_types[i] = type_of(params[i], "a parameter");
    g_types[i] = type_of(grads[i], "a gradient");
  }
  TORCH_CHECK(scale_of == scales.size(), "adamw: scales for a state that is not in 8 bits");
  // memory that is listed twice, as a whole or in part, would be updated by two warps at once
  std::vector<std::pair<const char*, const char*>> ranges;
  auto apart = [&](const auto& list, auto&& bytes) {
    ranges.clear();
    for (size_t i = 0; i < n; ++i)
      if (counts[i] && list[i]) ranges.emplace_back(reinterpret_cast<const char*>(list[i]), reinterpret_cast<const char*>(list[i]) + bytes(i));
    std::sort(ranges.begin(), ranges.end());
    for (size_t i = 1; i < ranges.size(); ++i)
      TORCH_CHECK(ranges[i - 1].second <= ranges[i].first, "adamw: a parameter or state is listed twice, as a whole or in part");
  };
  apart(p, [&](size_t i) { return counts[i] * params[i].element_size(); });
  for (const auto* list : {&m, &v}) apart(*list, [&](size_t i) { return counts[i] * exp_avg[i].element_size(); });
  for (const auto* list : {&me, &ve}) apart(*list, [&](size_t i) { return (counts[i] + 255) / 256; });
  c10::cuda::CUDAGuard guard(device);
  const Tensor ws = fresh({256}, params[0], at::kByte);
  s3r_adamw a = {};
  a.n = static_cast<int>(n);
  a.params = p.data();
  a.grads = g.data();
  a.m = m.data();
  a.v = v.data();
  a.m_exponents = me.data();
  a.v_exponents = ve.data();
  a.counts = counts.data();
  a.param_types = p_types.data();
  a.grad_types = g_types.data();
  a.step = static_cast<int64_t*>(step.data_ptr());
  a.lr = lr_tensor.has_value() ? f32(*lr_tensor) : nullptr;
  a.lr_host = lr;
  a.beta1 = beta1;
  a.beta2 = beta2;
  a.eps = eps;
  a.weight_decay = weight_decay;
  a.norm = norm.has_value() ? f32(*norm) : nullptr;
  a.max_norm = max_norm;
  a.seed = seed;
  a.workspace = ws.data_ptr();
  check(s3r_adamw_step_numbered(&a, number_of.empty() ? nullptr : number_of.data(), stream()), "s3r_adamw_step");
}

void adamw_values(at::TensorList exp_avg, at::TensorList exp_avg_sq, at::TensorList scales, at::TensorList m_out, at::TensorList v_out) {
  const size_t n = exp_avg.size();
  TORCH_CHECK(exp_avg_sq.size() == n && scales.size() == n && m_out.size() == n && v_out.size() == n, "adamw_state: lists of one length");
  if (n == 0) return;
  std::vector<const void*> m(n), v(n);
  std::vector<const uint8_t*> me(n), ve(n);
  std::vector<float*> mo(n), vo(n);
  std::vector<int64_t> counts(n);
  for (size_t i = 0; i < n; ++i) {
    need_cuda(exp_avg[i], "a state");
    TORCH_CHECK(exp_avg[i].device() == exp_avg[0].device(), "adamw_state: tensors of one device");
    need_states(exp_avg[i], exp_avg[i], exp_avg_sq[i], &scales[i]);
    for (const Tensor* t : {&m_out[i], &v_out[i]})
      TORCH_CHECK(t->device() == exp_avg[i].device() && t->scalar_type() == at::kFloat && t->sizes() == exp_avg[i].sizes() && t->is_contiguous(),
                  "adamw_state: results must be contiguous fp32 of the states' shapes");
    me[i] = static_cast<const uint8_t*>(scales[i].data_ptr());
    ve[i] = me[i] + scales[i].stride(0);
    m[i] = exp_avg[i].data_ptr();
    v[i] = exp_avg_sq[i].data_ptr();
    mo[i] = f32(m_out[i]);
    vo[i] = f32(v_out[i]);
    counts[i] = exp_avg[i].numel();
  }
  c10::cuda::CUDAGuard guard(exp_avg[0].device());
  check(s3r_adamw_state(static_cast<int>(n), m.data(), v.data(), me.data(), ve.data(), mo.data(), vo.data(), counts.data(), stream()), "s3r_adamw_state");
}

// What autograd has saved of these tensors is not what they hold any more (the dispatcher's own path counts by the schema).
void written(at::TensorList list) {
  for (const Tensor& t : list)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ------------------------------------------------------------------------------------------------
// The operators that have no gradient, as they are called: on ordinary tensors straight into the base operator.  Through the dispatcher
// each of them passed PyTorch's boxed autograd fallback, which looks at every tensor of every list.
// ------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> quantize_tokens(const Tensor& x) {
  no_tangents(x);
  if (plain(x)) return quantize_rows(x);
  S3R_DISPATCHED(quantize_rows)(x);
}
Tensor int8_linear(const Tensor& q, const Tensor& q_scale, const Tensor& weight, const Tensor& weight_scale, const optional<Tensor>& bias,
                   at::ScalarType out_type) {
  no_tangents(q_scale, weight_scale, bias);
  if (plain(q)) return int8_product(q, q_scale, weight, weight_scale, bias, out_type);
  S3R_DISPATCHED(int8_product)(q, q_scale, weight, weight_scale, bias, out_type);
}
Tensor grad_norm(at::TensorList tensors) {
  TORCH_CHECK(!tensors.empty(), "grad_norm: no tensors");
  no_tangents(tensors);
  if (plain(tensors[0])) return norm_of(tensors);
  S3R_DISPATCHED(norm_of)(tensors);
}
void adamw_step(at::TensorList params, at::TensorList grads, at::TensorList exp_avg, at::TensorList exp_avg_sq, const Tensor& step,
                const c10::List<optional<Tensor>>& scales, double lr, const optional<Tensor>& lr_tensor, double beta1, double beta2, double eps,
                double weight_decay, const optional<Tensor>& norm, double max_norm, int64_t seed, at::OptionalIntArrayRef numbers) {
  TORCH_CHECK(!params.empty(), "adamw: no tensors");
  no_tangents(params, grads, exp_avg, exp_avg_sq, lr_tensor, norm);
  std::vector<Tensor> held;
  if (!scales.empty()) {
    TORCH_CHECK(scales.size() == params.size() && exp_avg.size() == params.size(), "adamw: ", params.size(), " parameters, ", exp_avg.size(), " states, ",
                scales.size(), " scales");
    held.reserve(scales.size());
    for (size_t i = 0; i < exp_avg.size(); ++i) {
      optional<Tensor> scale = scales.get(i);
      TORCH_CHECK(scale.has_value() == (exp_avg[i].scalar_type() == at::kByte), "adamw: scales belong to a state of uint8 codes and only to one, got ",
                  scale.has_value() ? "scales" : "none", " for a state of ", exp_avg[i].scalar_type());
      if (scale.has_value()) held.push_back(*std::move(scale));
    }
  }
  if (plain(params[0])) {
    adamw_update(params, grads, exp_avg, exp_avg_sq, step, held, lr, lr_tensor, beta1, beta2, eps, weight_decay, norm, max_norm, seed, numbers);
    for (const auto list : {params, exp_avg, exp_avg_sq, at::TensorList(held), at::TensorList(step)}) written(list);
    return;
  }
  S3R_DISPATCHED(adamw_update)(params, grads, exp_avg, exp_avg_sq, step, held, lr, lr_tensor, beta1, beta2, eps, weight_decay, norm, max_norm, seed, numbers);
}
void adamw_state(at::TensorList exp_avg, at::TensorList exp_avg_sq, at::TensorList scales, at::TensorList m_out, at::TensorList v_out) {
  no_tangents(m_out, v_out);
  if (exp_avg.empty() || plain(exp_avg[0])) {
    adamw_values(exp_avg, exp_avg_sq, scales, m_out, v_out);
    written(m_out);
    return written(v_out);
  }
  S3R_DISPATCHED(adamw_values)(exp_avg, exp_avg_sq, scales, m_out, v_out);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(speed3r_b200, m) {
  m.def("residual_norm_fwd(Tensor x, Tensor? y, Tensor? weight, Tensor? bias, Tensor? scale, Tensor? gate, Tensor? post_weight, "
        "Tensor? post_bias, bool norm, bool post, int kind, float eps, float post_eps, ScalarType h_type, bool keep) -> (Tensor, Tensor, Tensor)");
  m.def("residual_norm_bwd(Tensor r, Tensor? y, Tensor? weight, Tensor? scale, Tensor? gate, Tensor? post_weight, Tensor? post_bias, "
        "Tensor stats, Tensor? dr, Tensor? dh, ScalarType? branch, bool post, int kind, int want, ScalarType param_type) -> Tensor[]");
  m.def("residual_norm_int8(Tensor x, Tensor? y, Tensor? weight, Tensor? bias, Tensor? scale, Tensor? gate, Tensor? post_weight, "
        "Tensor? post_bias, bool post, int kind, float eps, float post_eps) -> (Tensor, Tensor, Tensor)");
  m.def("residual_norm(Tensor x, Tensor? y, Tensor? weight, Tensor? bias, Tensor? scale, Tensor? gate, Tensor? post_weight, "
        "Tensor? post_bias, bool norm, bool post, int kind, float eps, float post_eps, ScalarType h_type) -> (Tensor, Tensor)", &residual_norm);
  m.def("residual_norm_to_int8(Tensor x, Tensor? y, Tensor? weight, Tensor? bias, Tensor? scale, Tensor? gate, Tensor? post_weight, "
        "Tensor? post_bias, bool post, int kind, float eps, float post_eps) -> (Tensor, Tensor, Tensor)", &residual_norm_to_int8);
  m.def("quantize_rows(Tensor x) -> (Tensor, Tensor)");
  m.def("int8_product(Tensor q, Tensor q_scale, Tensor weight, Tensor weight_scale, Tensor? bias, ScalarType out_type) -> Tensor");
  m.def("norm_of(Tensor[] tensors) -> Tensor");
  m.def("adamw_update(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avg, Tensor(c!)[] exp_avg_sq, Tensor(d!) step, Tensor(e!)[] scales, float lr, "
        "Tensor? lr_tensor, float beta1, float beta2, float eps, float weight_decay, Tensor? norm, float max_norm, int seed, int[]? numbers=None) -> ()");
  m.def("adamw_values(Tensor[] exp_avg, Tensor[] exp_avg_sq, Tensor[] scales, Tensor(a!)[] m_out, Tensor(b!)[] v_out) -> ()");
  m.def("quantize_tokens(Tensor x) -> (Tensor, Tensor)", &quantize_tokens);
  m.def("int8_linear(Tensor q, Tensor q_scale, Tensor weight, Tensor weight_scale, Tensor? bias, ScalarType out_type) -> Tensor", &int8_linear);
  m.def("grad_norm(Tensor[] tensors) -> Tensor", &grad_norm);
  m.def("adamw_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avg, Tensor(c!)[] exp_avg_sq, Tensor(d!) step, Tensor(e!)?[] scales, float lr, "
        "Tensor? lr_tensor, float beta1, float beta2, float eps, float weight_decay, Tensor? norm, float max_norm, int seed, int[]? numbers=None) -> ()", &adamw_step);
  m.def("adamw_state(Tensor[] exp_avg, Tensor[] exp_avg_sq, Tensor[] scales, Tensor(a!)[] m_out, Tensor(b!)[] v_out) -> ()", &adamw_state);
}

#define S3R_BLOCK_OPS(m)                              \
  m.impl("residual_norm_fwd", &residual_norm_fwd);    \
  m.impl("residual_norm_bwd", &residual_norm_bwd);    \
  m.impl("residual_norm_int8", &residual_norm_int8);  \
  m.impl("quantize_rows", &quantize_rows);        \
  m.impl("int8_product", &int8_product);                \
  m.impl("norm_of", &norm_of);                    \
  m.impl("adamw_update", &adamw_update);                  \
  m.impl("adamw_values", &adamw_values)

TORCH_LIBRARY_IMPL(speed3r_b200, CUDA, m) { S3R_BLOCK_OPS(m); }
TORCH_LIBRARY_IMPL(speed3r_b200, CPU, m) { S3R_BLOCK_OPS(m); }      // every one of them refuses CPU tensors
