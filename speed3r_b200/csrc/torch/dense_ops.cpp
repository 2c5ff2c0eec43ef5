// The torch.library operators of the dense half of a block: Linear layers with their epilogue, the norms and rotation of q and k.
#include "helpers.h"

namespace {

// ------------------------------------------------------------------------------------------------
// residual + act(x W^T + bias) * scale
// ------------------------------------------------------------------------------------------------
// The tensor itself where its rows of K 16-bit elements lie one behind the other at multiples of 16 bytes (a view takes a microsecond), else [rows, K]
// whose base and rows begin at such
Tensor half_rows(const Tensor& t, int64_t rows, int64_t K) {
  if (K % 8 == 0 && t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) return t;
  Tensor r = t.reshape({rows, K});
  const bool fits = (K == 1 || r.stride(1) == 1) && (rows <= 1 || (r.stride(0) >= K && r.stride(0) % 8 == 0)) &&
                    reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0;
  if (fits) return r;
  if (K > 1 && r.stride(1) != 1) r = r.contiguous();
  const int64_t pitch = (K + 7) / 8 * 8;
  Tensor whole = fresh({rows, pitch}, t, t.scalar_type());
  check(s3r_pad_rows(static_cast<const int8_t*>(r.data_ptr()), 2 * (rows > 1 ? r.stride(0) : K), static_cast<int8_t*>(whole.data_ptr()), 2 * pitch, rows,
                     static_cast<int>(2 * K), stream()), "s3r_pad_rows");
  return whole.narrow(1, 0, K);
}
int64_t pitch_of(const Tensor& t, int64_t K) { return t.dim() == 2 && t.size(0) > 1 ? t.stride(0) : (K + 7) / 8 * 8; }

struct LinearSizes {
  int64_t M, N, K;
};
LinearSizes linear_sizes(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, const optional<Tensor>& scale) {
  need_cuda(x, "x");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "linear: x must be bf16 or fp16, got ", x.scalar_type());
  TORCH_CHECK(weight.scalar_type() == x.scalar_type(), "linear: x and weight must be of one type, got ", x.scalar_type(), " and ", weight.scalar_type());
  TORCH_CHECK(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(1), "linear: x [.., K] and weight [N, K], got ", x.sizes(), " and ", weight.sizes());
  const int64_t K = weight.size(1), N = weight.size(0);
  TORCH_CHECK(K >= 1 && K < (int64_t{1} << 30), "linear: K = ", K);
  TORCH_CHECK(N >= 1 && N < (int64_t{1} << 30), "linear: N = ", N);
  const int64_t M = x.numel() / K;
  TORCH_CHECK(M < (int64_t{1} << 31) - 512, "linear: ", M, " rows");
  TORCH_CHECK(weight.device() == x.device(), "linear: tensors of one device");
  for (const auto* t : {&bias, &scale})
    TORCH_CHECK(!t->has_value() || ((*t)->device() == x.device() && (*t)->dim() == 1 && (*t)->size(0) == N), "linear: bias and scale must be [N] on x's device");
  return {M, N, K};
}

s3r_linear linear_args(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& scale, const LinearSizes& n, int64_t act, at::ScalarType out_type) {
  TORCH_CHECK(act >= S3R_ACT_NONE && act <= S3R_ACT_SILU, "linear: activation ", act);
  s3r_linear a = {};
  a.M = n.M;
  a.N = static_cast<int>(n.N);
  a.K = static_cast<int>(n.K);
  a.type = type_of(x, "x");
  a.x = x.data_ptr();
  a.x_pitch = pitch_of(x, n.K);
  a.weight = weight.data_ptr();
  a.w_pitch = pitch_of(weight, n.K);
  if (bias.defined()) a.bias = bias.data_ptr(), a.bias_type = type_of(bias, "bias");
  if (scale.defined()) a.scale = scale.data_ptr(), a.scale_type = type_of(scale, "scale");
  a.act = static_cast<int>(act);
  a.out_type = out_type == at::kFloat ? S3R_F32 : out_type == at::kBFloat16 ? S3R_BF16 : S3R_F16;
  TORCH_CHECK(out_type == at::kFloat || out_type == at::kBFloat16 || out_type == at::kHalf, "linear: the result must be fp32, bf16 or fp16, got ", out_type);
  return a;
}
// for the parts of a long sum of few rows
Tensor workspace(const Tensor& like, int64_t M, int64_t N, int64_t K) {
  const size_t bytes = s3r_linear_workspace_bytes(M, N, K);
  return bytes ? fresh({static_cast<int64_t>(bytes)}, like, at::kByte) : Tensor();
}
Tensor dense(const optional<Tensor>& t) { return t.has_value() ? t->contiguous() : Tensor(); }

Tensor linear_fwd(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, const optional<Tensor>& scale, const optional<Tensor>& residual,
                  int64_t act, at::ScalarType out_type) {
  const LinearSizes n = linear_sizes(x, weight, bias, scale);
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n.N;
  if (residual.has_value()) {
    TORCH_CHECK(residual->device() == x.device() && residual->sizes() == at::IntArrayRef(shape), "linear: residual must be ", at::IntArrayRef(shape), " on x's device, got ",
                residual->sizes());
    type_of(*residual, "residual");
  }
  c10::cuda::CUDAGuard guard(x.device());
  Tensor out = fresh(shape, x, out_type);
  if (n.M == 0) return out;
  const Tensor a = half_rows(x, n.M, n.K), w = half_rows(weight, n.N, n.K), b = dense(bias), s = dense(scale), r = dense(residual);
  s3r_linear f = linear_args(a, w, b, s, n, act, out_type);
  if (r.defined()) f.residual = r.data_ptr(), f.residual_type = type_of(r, "residual");
  f.out = out.data_ptr();
  const Tensor ws = workspace(x, n.M, n.N, n.K);
  f.workspace = pointer(ws);
  f.workspace_bytes = ws.defined() ? ws.numel() : 0;
  check(s3r_linear_fwd(&f, stream()), "s3r_linear_fwd");
  return out;
}

// Gradients of (x, weight, bias, scale); those that `want` (a bit each) does not name are undefined (from the operator: without elements).
enum { kX = 1, kWeight = 2, kBias = 4, kScale = 8 };
std::vector<Tensor> run_linear_bwd(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, const optional<Tensor>& scale, const Tensor& dy, int64_t act,
                                   int64_t want) {
  const LinearSizes n = linear_sizes(x, weight, bias, scale);
  TORCH_CHECK(dy.device() == x.device() && dy.numel() == n.M * n.N && dy.is_contiguous(), "linear: the gradient must be like the result, contiguous");
  TORCH_CHECK((bias.has_value() || !(want & kBias)) && (scale.has_value() || !(want & kScale)), "linear: a gradient of what is not there");
  c10::cuda::CUDAGuard guard(x.device());
  auto like = [](const Tensor& t) { return fresh(t.sizes(), t, t.scalar_type()); };
  Tensor dx = want & kX ? like(x) : Tensor(), dw = want & kWeight ? like(weight) : Tensor();
  Tensor db = want & kBias ? like(*bias) : Tensor(), ds = want & kScale ? like(*scale) : Tensor();
  if (n.M == 0) {
    for (Tensor* t : {&dw, &db, &ds})
      if (t->defined()) t->zero_();
    return {dx, dw, db, ds};
  }
  const Tensor a = half_rows(x, n.M, n.K), w = half_rows(weight, n.N, n.K), b = dense(bias), s = dense(scale);
  const s3r_linear f = linear_args(a, w, b, s, n, act, dy.scalar_type());
  // dz is dy itself where nothing stands between them
  const bool same = act == S3R_ACT_NONE && !scale.has_value() && dy.scalar_type() == x.scalar_type() && n.N % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16 == 0;
  const bool products = want & (kX | kWeight);
  const int64_t pitch = (n.N + 7) / 8 * 8;
  const Tensor dz = !products ? Tensor() : same ? dy : fresh({n.M, pitch}, x, x.scalar_type());
  s3r_linear_grad g = {};
  g.dy = dy.data_ptr();
  g.dz = dz.defined() && !same ? dz.data_ptr() : nullptr;
  g.dz_pitch = pitch;
  g.d_bias = pointer(db);
  g.d_scale = pointer(ds);
  Tensor ws;
  if (const int sums = db.defined() + ds.defined()) {
    g.workspace_bytes = s3r_linear_bwd_workspace_bytes(n.M, static_cast<int>(n.N)) * sums;
    ws = fresh({static_cast<int64_t>(g.workspace_bytes)}, x, at::kByte);
    g.workspace = ws.data_ptr();
  }
  check(s3r_linear_bwd(&f, &g, stream()), "s3r_linear_bwd");
  auto product = [&](bool turned, const Tensor& other, Tensor& out, int64_t rows, int64_t sum) {
    const Tensor parts = workspace(x, rows, n.K, sum);
    check(s3r_product(dz.data_ptr(), pitch, turned, other.data_ptr(), pitch_of(other, n.K), 1, f.type, out.data_ptr(), rows, static_cast<int>(n.K), sum, pointer(parts),
                      parts.defined() ? parts.numel() : 0, stream()), "s3r_product");
  };
  if (dx.defined()) product(false, w, dx, n.M, n.N);
  if (dw.defined()) product(true, a, dw, n.N, n.M);
  return {dx, dw, db, ds};
}
std::vector<Tensor> linear_bwd(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, const optional<Tensor>& scale, const Tensor& dy, int64_t act,
                               int64_t want) {
  auto g = run_linear_bwd(x, weight, bias, scale, dy, act, want);
  for (Tensor& t : g)
    if (!t.defined()) t = none(x);
  return g;
}

Tensor call_linear_fwd(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, const optional<Tensor>& scale, const optional<Tensor>& residual,
                       int64_t act, at::ScalarType out_type) {
  if (plain(x)) return linear_fwd(x, weight, bias, scale, residual, act, out_type);
  S3R_DISPATCHED(linear_fwd)(x, weight, bias, scale, residual, act, out_type);
}
std::vector<Tensor> call_linear_bwd(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, const optional<Tensor>& scale, const Tensor& dy,
                                    int64_t act, int64_t want) {
  if (plain(x)) return run_linear_bwd(x, weight, bias, scale, dy, act, want);
  S3R_DISPATCHED(linear_bwd)(x, weight, bias, scale, dy, act, want);
}

// a residual of x's leading dimensions as rows
Tensor as_result(const Tensor& residual, const Tensor& x, const LinearSizes& n) {
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = n.N;
  TORCH_CHECK(residual.device() == x.device() && residual.sizes() == at::IntArrayRef(shape), "linear: residual must be ", at::IntArrayRef(shape), " on x's device, got ", residual.sizes());
  return residual.reshape({n.M, n.N});
}

struct LinearNode : torch::autograd::Function<LinearNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, const optional<Tensor>& scale,
                        const optional<Tensor>& residual, int64_t act, int64_t out_type) {
    at::AutoDispatchBelowADInplaceOrView below;
    int64_t present = 3;                          // which of the five tensors are there: only they have an edge
    if (bias.has_value()) present |= 4;
    if (scale.has_value()) present |= 8;
    if (residual.has_value()) present |= 16;
    const int64_t kept = residual.has_value() ? static_cast<int64_t>(residual->scalar_type()) : 0;
    ctx->saved_data["ints"] = std::vector<int64_t>{present, act, kept};
    ctx->set_materialize_grads(false);
    if (!plain(x)) {
      ctx->save_for_backward({x, weight, value(bias), value(scale)});
      return call_linear_fwd(x, weight, bias, scale, residual, act, static_cast<at::ScalarType>(out_type));
    }
    // what is laid out anew is kept that way; a view made here does not count its owner's changes, so the owner is kept in its place
    const LinearSizes n = linear_sizes(x, weight, bias, scale);
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor a = n.M ? half_rows(x, n.M, n.K) : x, w = n.M ? half_rows(weight, n.N, n.K) : weight;
    ctx->save_for_backward({a.is_alias_of(x) ? x : a, w.is_alias_of(weight) ? weight : w, value(bias), value(scale)});
    ctx->saved_data["shape"] = x.sizes().vec();
    const bool rows = a.sizes() != x.sizes();
    Tensor out = linear_fwd(a, w, bias, scale, rows && residual.has_value() ? optional<Tensor>(as_result(*residual, x, n)) : residual, act, static_cast<at::ScalarType>(out_type));
    if (!rows) return out;
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = n.N;
    return in_shape(out, shape);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return once(g, [&] { return gradients(ctx, g); });
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& incoming) {
    variable_list out(7);
    if (!incoming[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const auto ints = ctx->saved_data["ints"].toIntVector();
    int64_t want = 0;
    for (int i = 0, edge = 0; i < 5; ++i)
      if (ints[0] >> i & 1 && ctx->needs_input_grad(edge++)) want |= int64_t{1} << i;
    if (want & 16) out[4] = incoming[0].to(static_cast<at::ScalarType>(ints[2]));
    if (want & 15) {
      const auto g = call_linear_bwd(s[0], s[1], maybe(s[2]), maybe(s[3]), incoming[0].contiguous(), ints[1], want & 15);
      for (int i = 0; i < 4; ++i)
        if (want >> i & 1) out[i] = g[i];
      if (out[0].defined() && ctx->saved_data.count("shape")) out[0] = in_shape(out[0], ctx->saved_data["shape"].toIntVector());
    }
    return out;
  }
};

Tensor linear(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, const optional<Tensor>& scale, const optional<Tensor>& residual, int64_t act,
              at::ScalarType out_type) {
  if (wants_grad(x, weight, value(bias), value(scale), value(residual)))
    return LinearNode::apply(x, weight, bias, scale, residual, act, static_cast<int64_t>(out_type));
  return call_linear_fwd(x, weight, bias, scale, residual, act, out_type);
}

// ------------------------------------------------------------------------------------------------
// q, k and v of the packed projection
// ------------------------------------------------------------------------------------------------
struct RopeShape {
  int64_t heads, kv_heads;
  bool q_normed, k_normed;
  int64_t kind;
  double q_eps, k_eps;
};

s3r_qkv_norm_rope rope_args(const Tensor& qkv, const optional<Tensor>& pos, const optional<Tensor>& cos, const optional<Tensor>& sin, const optional<Tensor>& qw,
                            const optional<Tensor>& qb, const optional<Tensor>& kw, const optional<Tensor>& kb, const RopeShape& n) {
  need_cuda(qkv, "qkv");
  TORCH_CHECK(qkv.dim() == 3 && (qkv.size(2) == 1 || qkv.stride(2) == 1), "qkv_norm_rope: qkv must be [batch, tokens, channels] with contiguous channels");
  TORCH_CHECK(n.heads >= 1 && n.kv_heads >= 1 && n.heads <= 4096 && n.kv_heads <= 4096, "qkv_norm_rope: ", n.heads, " heads and ", n.kv_heads, " (1 to 4096)");
  const int64_t all = n.heads + 2 * n.kv_heads, d = qkv.size(2) / all;
  TORCH_CHECK(qkv.size(2) == d * all, "qkv_norm_rope: ", qkv.size(2), " channels for ", n.heads, " + 2 * ", n.kv_heads, " heads");
  TORCH_CHECK(d >= 2 && d <= 256 && d % 2 == 0, "qkv_norm_rope: heads of ", d, " channels (even, 2 to 256)");
  TORCH_CHECK(qkv.size(0) * qkv.size(1) < (int64_t{1} << 31) - 1024, "qkv_norm_rope: too many tokens");
  s3r_qkv_norm_rope a = {};
  a.batch = qkv.size(0);
  a.tokens = qkv.size(1);
  a.heads = static_cast<int>(n.heads);
  a.kv_heads = static_cast<int>(n.kv_heads);
  a.head_dim = static_cast<int>(d);
  a.kind = static_cast<int>(n.kind);
  a.q_normed = n.q_normed;
  a.k_normed = n.k_normed;
  a.q_eps = static_cast<float>(n.q_eps);
  a.k_eps = static_cast<float>(n.k_eps);
  a.type = type_of(qkv, "qkv");
  a.stride_b = qkv.stride(0);
  a.stride_t = qkv.stride(1);
  a.qkv = qkv.data_ptr();
  if (pos.has_value()) {
    TORCH_CHECK(cos.has_value() && sin.has_value(), "qkv_norm_rope: positions need cos and sin");
    TORCH_CHECK(pos->device() == qkv.device() && pos->scalar_type() == at::kLong && pos->dim() == 3 && pos->size(0) == a.batch && pos->size(1) == a.tokens &&
                    pos->size(2) >= 1 && (pos->size(2) == 1 || pos->stride(2) == 1), "qkv_norm_rope: pos must be int64 [batch, tokens, axes] on qkv's device, got ",
                pos->scalar_type(), " ", pos->sizes());
    for (const auto* t : {&cos, &sin})
      TORCH_CHECK((*t)->device() == qkv.device() && (*t)->dim() == 2 && (*t)->sizes() == cos->sizes() && (*t)->scalar_type() == cos->scalar_type() &&
                      ((*t)->size(1) <= 1 || (*t)->stride(1) == 1), "qkv_norm_rope: cos and sin must be [rows, pairs] of one type on qkv's device");
    TORCH_CHECK(cos->size(0) >= 1 && cos->size(1) >= 1 && cos->size(0) < (int64_t{1} << 31) && 2 * cos->size(1) * pos->size(2) <= d,
                "qkv_norm_rope: tables ", cos->sizes(), " and ", pos->size(2), " axes for heads of ", d, " channels");
    a.axes = static_cast<int>(pos->size(2));
    a.pairs = static_cast<int>(cos->size(1));
    a.rows = static_cast<int>(cos->size(0));
    a.pos = static_cast<const int64_t*>(pos->data_ptr());
    a.pos_stride_b = pos->stride(0);
    a.pos_stride_t = pos->stride(1);
    a.cos = cos->data_ptr();
    a.sin = sin->data_ptr();
    a.cos_pitch = cos->stride(0);
    a.sin_pitch = sin->stride(0);
    a.table_type = type_of(*cos, "cos");
  }
  a.param_type = -1;
  auto param = [&](const optional<Tensor>& t, const char* name) -> const void* {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->device() == qkv.device() && t->dim() == 1 && t->size(0) == d && t->is_contiguous(), "qkv_norm_rope: ", name, " must be a contiguous [", d, "] on qkv's device");
    const int type = type_of(*t, name);
    TORCH_CHECK(a.param_type < 0 || a.param_type == type, "qkv_norm_rope: parameters of one type");
    a.param_type = type;
    return t->data_ptr();
  };
  a.q_weight = param(qw, "q_norm's weight");
  a.q_bias = param(qb, "q_norm's bias");
  a.k_weight = param(kw, "k_norm's weight");
  a.k_bias = param(kb, "k_norm's bias");
  if (a.param_type < 0) a.param_type = S3R_F32;
  return a;
}

std::tuple<Tensor, Tensor, Tensor> qkv_norm_rope_fwd(const Tensor& qkv, const optional<Tensor>& pos, const optional<Tensor>& cos, const optional<Tensor>& sin,
                                                     const optional<Tensor>& qw, const optional<Tensor>& qb, const optional<Tensor>& kw, const optional<Tensor>& kb,
                                                     int64_t heads, int64_t kv_heads, bool q_normed, bool k_normed, int64_t kind, double q_eps, double k_eps) {
  s3r_qkv_norm_rope a = rope_args(qkv, pos, cos, sin, qw, qb, kw, kb, {heads, kv_heads, q_normed, k_normed, kind, q_eps, k_eps});
  c10::cuda::CUDAGuard guard(qkv.device());
  auto made = [&](int64_t h) { return fresh({a.batch, h, a.tokens, a.head_dim}, qkv, qkv.scalar_type()); };
  Tensor q = made(heads), k = made(kv_heads), v = made(kv_heads);
  if (qkv.numel()) {
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    check(s3r_qkv_norm_rope_fwd(&a, stream()), "s3r_qkv_norm_rope_fwd");
  }
  return {q, k, v};
}

// Gradients of (qkv, q_norm's weight and bias, k_norm's); those that `want` (a bit each) does not name are undefined (from the operator: without elements).
std::vector<Tensor> run_rope_bwd(const Tensor& qkv, const optional<Tensor>& pos, const optional<Tensor>& cos, const optional<Tensor>& sin, const optional<Tensor>& qw,
                                 const optional<Tensor>& kw, const optional<Tensor>& dq, const optional<Tensor>& dk, const optional<Tensor>& dv, int64_t heads,
                                 int64_t kv_heads, bool q_normed, bool k_normed, int64_t kind, double q_eps, double k_eps, int64_t want, at::ScalarType param_type) {
  s3r_qkv_norm_rope f = rope_args(qkv, pos, cos, sin, qw, {}, kw, {}, {heads, kv_heads, q_normed, k_normed, kind, q_eps, k_eps});
  f.param_type = type_of(at::empty({0}, at::TensorOptions().dtype(param_type)), "parameters");
  c10::cuda::CUDAGuard guard(qkv.device());
  s3r_qkv_norm_rope_grad g = {};
  auto incoming = [&](const optional<Tensor>& t, int64_t h, const void** p, int64_t* strides) {
    if (!t.has_value()) return;
    TORCH_CHECK(t->device() == qkv.device() && t->scalar_type() == qkv.scalar_type() && t->sizes() == at::IntArrayRef({f.batch, h, f.tokens, f.head_dim}) &&
                    t->stride(3) == 1, "qkv_norm_rope: gradients must be like q, k and v");
    *p = t->data_ptr();
    for (int i = 0; i < 3; ++i) strides[i] = t->stride(i);
  };
  incoming(dq, heads, &g.dq, g.dq_strides);
  incoming(dk, kv_heads, &g.dk, g.dk_strides);
  incoming(dv, kv_heads, &g.dv, g.dv_strides);
  Tensor d_qkv = fresh(qkv.sizes(), qkv, qkv.scalar_type());
  std::vector<Tensor> sums(4);
  for (int i = 0; i < 4; ++i)
    if (want >> (i + 1) & 1) sums[i] = fresh({f.head_dim}, qkv, param_type);
  if (qkv.numel()) {
    g.d_qkv = d_qkv.data_ptr();
    g.d_q_weight = pointer(sums[0]);
    g.d_q_bias = pointer(sums[1]);
    g.d_k_weight = pointer(sums[2]);
    g.d_k_bias = pointer(sums[3]);
    Tensor ws;
    if (want & ~1) {
      g.workspace_bytes = s3r_qkv_norm_rope_bwd_workspace_bytes(f.batch, f.tokens, f.heads, f.kv_heads, f.head_dim);
      ws = fresh({static_cast<int64_t>(g.workspace_bytes)}, qkv, at::kByte);
      g.workspace = ws.data_ptr();
    }
    check(s3r_qkv_norm_rope_bwd(&f, &g, stream()), "s3r_qkv_norm_rope_bwd");
  } else {
    for (Tensor& t : sums)
      if (t.defined()) t.zero_();
  }
  return {d_qkv, sums[0], sums[1], sums[2], sums[3]};
}
std::vector<Tensor> qkv_norm_rope_bwd(const Tensor& qkv, const optional<Tensor>& pos, const optional<Tensor>& cos, const optional<Tensor>& sin, const optional<Tensor>& qw,
                                      const optional<Tensor>& kw, const optional<Tensor>& dq, const optional<Tensor>& dk, const optional<Tensor>& dv, int64_t heads,
                                      int64_t kv_heads, bool q_normed, bool k_normed, int64_t kind, double q_eps, double k_eps, int64_t want,
                                      at::ScalarType param_type) {
  auto g = run_rope_bwd(qkv, pos, cos, sin, qw, kw, dq, dk, dv, heads, kv_heads, q_normed, k_normed, kind, q_eps, k_eps, want, param_type);
  for (Tensor& t : g)
    if (!t.defined()) t = fresh({0}, qkv, param_type);
  return g;
}

struct RopeInputs {
  Tensor qkv;
  optional<Tensor> pos, cos, sin, qw, qb, kw, kb;
};
std::tuple<Tensor, Tensor, Tensor> call_rope_fwd(const RopeInputs& in, const RopeShape& n) {
  if (plain(in.qkv)) return qkv_norm_rope_fwd(in.qkv, in.pos, in.cos, in.sin, in.qw, in.qb, in.kw, in.kb, n.heads, n.kv_heads, n.q_normed, n.k_normed, n.kind, n.q_eps, n.k_eps);
  S3R_DISPATCHED(qkv_norm_rope_fwd)(in.qkv, in.pos, in.cos, in.sin, in.qw, in.qb, in.kw, in.kb, n.heads, n.kv_heads, n.q_normed, n.k_normed, n.kind, n.q_eps, n.k_eps);
}
std::vector<Tensor> call_rope_bwd(const Tensor& qkv, const optional<Tensor>& pos, const optional<Tensor>& cos, const optional<Tensor>& sin, const optional<Tensor>& qw,
                                  const optional<Tensor>& kw, const optional<Tensor>& dq, const optional<Tensor>& dk, const optional<Tensor>& dv, int64_t heads,
                                  int64_t kv_heads, bool q_normed, bool k_normed, int64_t kind, double q_eps, double k_eps, int64_t want, at::ScalarType param_type) {
  S3R_DISPATCHED(qkv_norm_rope_bwd)(qkv, pos, cos, sin, qw, kw, dq, dk, dv, heads, kv_heads, q_normed, k_normed, kind, q_eps, k_eps, want, param_type);
}

struct RopeNode : torch::autograd::Function<RopeNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& qkv, const optional<Tensor>& qw, const optional<Tensor>& qb, const optional<Tensor>& kw,
                               const optional<Tensor>& kb, const optional<Tensor>& pos, const optional<Tensor>& cos, const optional<Tensor>& sin, int64_t heads,
                               int64_t kv_heads, bool q_normed, bool k_normed, int64_t kind, double q_eps, double k_eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    int64_t present = 1, bit = 2;                 // which of the five tensors are there: only they have an edge
    at::ScalarType param = at::kFloat;
    for (const auto* t : {&qw, &qb, &kw, &kb}) {
      if (t->has_value()) present |= bit, param = (*t)->scalar_type();
      bit *= 2;
    }
    ctx->save_for_backward({qkv, value(qw), value(kw), value(pos), value(cos), value(sin)});
    ctx->saved_data["ints"] = std::vector<int64_t>{present, heads, kv_heads, q_normed, k_normed, kind, static_cast<int64_t>(param)};
    ctx->saved_data["eps"] = std::vector<double>{q_eps, k_eps};
    ctx->set_materialize_grads(false);
    auto [q, k, v] = call_rope_fwd({qkv, pos, cos, sin, qw, qb, kw, kb}, {heads, kv_heads, q_normed, k_normed, kind, q_eps, k_eps});
    return {q, k, v};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return once(g, [&] { return gradients(ctx, g); });
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& incoming) {
    variable_list out(15);
    if (!incoming[0].defined() && !incoming[1].defined() && !incoming[2].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const auto ints = ctx->saved_data["ints"].toIntVector();
    const auto eps = ctx->saved_data["eps"].toDoubleVector();
    int64_t want = 0;
    for (int i = 0, edge = 0; i < 5; ++i)
      if (ints[0] >> i & 1) {
        if (ctx->needs_input_grad(edge)) want |= int64_t{1} << i;
        ++edge;
      }
    auto given = [](const Tensor& t) { return !t.defined() ? optional<Tensor>() : optional<Tensor>(t.stride(3) == 1 ? t : t.contiguous()); };
    const auto& backward = plain(s[0]) ? run_rope_bwd : call_rope_bwd;
    const auto g = backward(s[0], maybe(s[3]), maybe(s[4]), maybe(s[5]), maybe(s[1]), maybe(s[2]), given(incoming[0]), given(incoming[1]), given(incoming[2]), ints[1],
                            ints[2], ints[3], ints[4], ints[5], eps[0], eps[1], want, static_cast<at::ScalarType>(ints[6]));
    for (int i = 0; i < 5; ++i)
      if (want >> i & 1) out[i] = g[i];
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor> qkv_norm_rope(const Tensor& qkv, const optional<Tensor>& pos, const optional<Tensor>& cos, const optional<Tensor>& sin,
                                                 const optional<Tensor>& qw, const optional<Tensor>& qb, const optional<Tensor>& kw, const optional<Tensor>& kb,
                                                 int64_t heads, int64_t kv_heads, bool q_normed, bool k_normed, int64_t kind, double q_eps, double k_eps) {
  TORCH_CHECK(kind == S3R_NORM_LAYER || kind == S3R_NORM_RMS, "qkv_norm_rope: kind ", kind);
  TORCH_CHECK((q_normed || (!qw.has_value() && !qb.has_value())) && (k_normed || (!kw.has_value() && !kb.has_value())), "qkv_norm_rope: weight and bias belong to a norm");
  TORCH_CHECK(qkv.dim() == 3, "qkv_norm_rope: qkv must be [batch, tokens, channels], got ", qkv.sizes());
  RopeInputs in = {qkv.size(2) > 1 && qkv.stride(2) != 1 ? qkv.contiguous() : qkv, pos, cos, sin, qw, qb, kw, kb};
  TORCH_CHECK(pos.has_value() == cos.has_value() && pos.has_value() == sin.has_value(), "qkv_norm_rope: pos, cos and sin come together or not at all");
  if (pos.has_value()) {
    TORCH_CHECK(!at::GradMode::is_enabled() || !(cos->requires_grad() || sin->requires_grad()), "qkv_norm_rope: cos and sin have no gradients here");
    TORCH_CHECK(pos->scalar_type() == at::kLong || pos->scalar_type() == at::kInt, "qkv_norm_rope: pos must be int64 or int32, got ", pos->scalar_type());
    TORCH_CHECK((pos->dim() == 3 || pos->dim() == 2) && pos->size(pos->dim() - 2) == qkv.size(1) && (pos->dim() == 2 || pos->size(0) == 1 || pos->size(0) == qkv.size(0)),
                "qkv_norm_rope: pos must be [batch or 1, tokens, axes] or [tokens, axes], got ", pos->sizes(), " for ", qkv.sizes());
    // calls that would change nothing are left out: each takes up to a microsecond
    Tensor p = pos->scalar_type() == at::kLong ? *pos : pos->to(at::kLong);
    if (p.size(-1) > 1 && p.stride(-1) != 1) p = p.contiguous();
    in.pos = p.dim() == 3 && p.size(0) == qkv.size(0) ? p : p.expand({qkv.size(0), qkv.size(1), p.size(-1)});
    const bool mixed = cos->scalar_type() != sin->scalar_type();
    for (optional<Tensor>* t : {&in.cos, &in.sin}) {
      if (mixed) **t = (*t)->to(at::kFloat);
      if ((*t)->dim() == 2 && (*t)->size(1) > 1 && (*t)->stride(1) != 1) **t = (*t)->contiguous();
    }
  }
  const RopeShape n = {heads, kv_heads, q_normed, k_normed, kind, q_eps, k_eps};
  of_one_type({&in.qw, &in.qb, &in.kw, &in.kb});
  no_tangents(cos, sin);
  if (wants_grad(qkv, value(qw), value(qb), value(kw), value(kb))) {
    const auto out = RopeNode::apply(in.qkv, in.qw, in.qb, in.kw, in.kb, in.pos, in.cos, in.sin, heads, kv_heads, q_normed, k_normed, kind, q_eps, k_eps);
    return {out[0], out[1], out[2]};
  }
  return call_rope_fwd(in, n);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(speed3r_b200, m) {
  m.def("linear_fwd(Tensor x, Tensor weight, Tensor? bias, Tensor? scale, Tensor? residual, int act, ScalarType out_type) -> Tensor");
  m.def("linear_bwd(Tensor x, Tensor weight, Tensor? bias, Tensor? scale, Tensor dy, int act, int want) -> Tensor[]");
  m.def("linear(Tensor x, Tensor weight, Tensor? bias, Tensor? scale, Tensor? residual, int act, ScalarType out_type) -> Tensor", &linear);
  m.def("qkv_norm_rope_fwd(Tensor qkv, Tensor? pos, Tensor? cos, Tensor? sin, Tensor? q_weight, Tensor? q_bias, Tensor? k_weight, Tensor? k_bias, int heads, "
        "int kv_heads, bool q_normed, bool k_normed, int kind, float q_eps, float k_eps) -> (Tensor, Tensor, Tensor)");
  m.def("qkv_norm_rope_bwd(Tensor qkv, Tensor? pos, Tensor? cos, Tensor? sin, Tensor? q_weight, Tensor? k_weight, Tensor? dq, Tensor? dk, Tensor? dv, int heads, "
        "int kv_heads, bool q_normed, bool k_normed, int kind, float q_eps, float k_eps, int want, ScalarType param_type) -> Tensor[]");
  m.def("qkv_norm_rope(Tensor qkv, Tensor? pos, Tensor? cos, Tensor? sin, Tensor? q_weight, Tensor? q_bias, Tensor? k_weight, Tensor? k_bias, int heads, "
        "int kv_heads, bool q_normed, bool k_normed, int kind, float q_eps, float k_eps) -> (Tensor, Tensor, Tensor)", &qkv_norm_rope);
}

#define S3R_DENSE_OPS(m)                            \
  m.impl("linear_fwd", &linear_fwd);                \
  m.impl("linear_bwd", &linear_bwd);                \
  m.impl("qkv_norm_rope_fwd", &qkv_norm_rope_fwd);  \
  m.impl("qkv_norm_rope_bwd", &qkv_norm_rope_bwd)

TORCH_LIBRARY_IMPL(speed3r_b200, CUDA, m) { S3R_DENSE_OPS(m); }
TORCH_LIBRARY_IMPL(speed3r_b200, CPU, m) { S3R_DENSE_OPS(m); }      // every one of them refuses CPU tensors
