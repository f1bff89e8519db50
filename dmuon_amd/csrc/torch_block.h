// The autograd operators of a block's attention and of the token lookup; part of torch_binding.cpp, whose
// helpers it uses.
#pragma once

namespace {

// ---- attention over heads -----------------------------------------------------------------------

// [batch][tokens][heads][dim] or [tokens][heads][dim] as the kernels read it: whole 16-byte chunks and, of
// keys and values, rows that do not overlap. Others are copied.
struct HeadsView {
  Tensor t;
  int64_t batch, token, head;
  HeadsView(const Tensor& x, bool keys, int64_t group) {
    if (!fits(x, keys, group)) t = x.resolve_neg().clone(at::MemoryFormat::Contiguous);
    else t = x;
    set(t);
  }

 private:
  void set(const Tensor& x) {
    const int64_t n = x.dim(), d = x.size(n - 1), h = x.size(n - 2);
    auto stride = [&](int64_t i, int64_t dense) { return x.size(i) > 1 ? x.stride(i) : dense; };
    head = stride(n - 2, d);
    token = stride(n - 3, h * d);
    batch = n == 4 ? stride(0, x.size(1) * h * d) : 0;
  }
  bool fits(const Tensor& x, bool keys, int64_t group) {
    if (x.is_neg() || x.stride(-1) != 1 || reinterpret_cast<uintptr_t>(ptr(x)) % 16) return false;
    set(x);
    if (batch % 8 || token % 8 || head % 8) return false;
    if (keys) return token >= x.size(-1) && token < (1 << 24);
    return 65 * token + group * head < (1 << 30);
  }
};

struct AttentionCall {
  bool causal = true, packed = false;
  int64_t window = 0, batch = 0, group = 1;
  double scale = 0.;

  dmuon_attention_args describe(const HeadsView& q, const HeadsView& k, const HeadsView& v,
                                const Tensor& lengths, const Tensor& q_starts, const Tensor& kv_starts) const {
    dmuon_attention_args a{};
    a.q = ptr(q.t);
    a.k = ptr(k.t);
    a.v = ptr(v.t);
    a.kv_lengths = static_cast<const int64_t*>(ptr(lengths));
    a.q_starts = static_cast<const int64_t*>(ptr(q_starts));
    a.kv_starts = static_cast<const int64_t*>(ptr(kv_starts));
    a.batch = batch;
    a.q_len = q.t.size(-3);
    a.kv_len = k.t.size(-3);
    a.heads = q.t.size(-2);
    a.kv_heads = k.t.size(-2);
    a.dim = q.t.size(-1);
    a.window = window;
    a.q_batch = q.batch; a.q_token = q.token; a.q_head = q.head;
    a.k_batch = k.batch; a.k_token = k.token; a.k_head = k.head;
    a.v_batch = v.batch; a.v_token = v.token; a.v_head = v.head;
    a.scale = (float)scale;
    a.causal = causal;
    a.dtype = code(q.t.scalar_type());
    return a;
  }

  Tensor forward(const HeadsView& q, const HeadsView& k, const HeadsView& v, const Tensor& lengths,
                 const Tensor& q_starts, const Tensor& kv_starts, Tensor* lse, Tensor* rest) const {
    const c10::DeviceGuard guard(q.t.device());
    auto a = describe(q, k, v, lengths, q_starts, kv_starts);
    Tensor out = at::empty(q.t.sizes(), q.t.options());
    a.out = ptr(out);
    if (lse) {
      *lse = at::empty(q.t.sizes().slice(0, q.t.dim() - 1), q.t.options().dtype(at::kFloat));
      a.lse = static_cast<float*>(ptr(*lse));
      *rest = at::empty(q.t.sizes(), q.t.options());
      a.rest = ptr(*rest);
    }
    int64_t need = 0;
    call(dmuon_attention_workspace_size(&a, &need));
    const Tensor ws = workspace(need, q.t);
    call(dmuon_attention(&a, ws.data_ptr(), need, stream_of(q.t)));
    return out;
  }
};

struct Attend : torch::autograd::Function<Attend> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const OptTensor& lengths, const OptTensor& q_starts, const OptTensor& kv_starts,
                        const AttentionCall& c) {
    const HeadsView qv(q, false, c.group), kv(k, true, c.group), vv(v, true, c.group);
    Tensor lse, rest;
    const Tensor n = lengths.value_or(Tensor()), qs = q_starts.value_or(Tensor()),
                 ks = kv_starts.value_or(Tensor());
    const Tensor out = c.forward(qv, kv, vv, n, qs, ks, &lse, &rest);
    ctx->saved_data["causal"] = c.causal;
    ctx->saved_data["packed"] = c.packed;
    ctx->saved_data["window"] = c.window;
    ctx->saved_data["batch"] = c.batch;
    ctx->saved_data["group"] = c.group;
    ctx->saved_data["scale"] = c.scale;
    ctx->save_for_backward({qv.t, kv.t, vv.t, out, lse, n, qs, ks, rest});
    return out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("attention");
    const auto s = ctx->get_saved_variables();
    AttentionCall c;
    c.causal = ctx->saved_data["causal"].toBool();
    c.packed = ctx->saved_data["packed"].toBool();
    c.window = ctx->saved_data["window"].toInt();
    c.batch = ctx->saved_data["batch"].toInt();
    c.group = ctx->saved_data["group"].toInt();
    c.scale = ctx->saved_data["scale"].toDouble();
    const c10::DeviceGuard guard(s[0].device());
    const HeadsView q(s[0], false, c.group), k(s[1], true, c.group), v(s[2], true, c.group);
    const HeadsView d(grads[0], false, c.group);
    auto a = c.describe(q, k, v, s[5], s[6], s[7]);
    a.out = ptr(s[3]);
    a.rest = ptr(s[8]);
    a.lse = static_cast<float*>(ptr(s[4]));
    a.dout = ptr(d.t);
    a.do_batch = d.batch;
    a.do_token = d.token;
    a.do_head = d.head;
    variable_list out(7);
    void** place[3] = {&a.dq, &a.dk, &a.dv};
    for (int i = 0; i < 3; ++i) {
      if (!ctx->needs_input_grad(i)) continue;
      out[i] = at::empty(s[i].sizes(), s[i].options());
      *place[i] = ptr(out[i]);
    }
    int64_t need = 0;
    call(dmuon_attention_grad_workspace_size(&a, &need));
    const Tensor ws = workspace(need, s[0]);
    call(dmuon_attention_grad(&a, ws.data_ptr(), need, stream_of(s[0])));
    return out;
  }
};

// Integers of the shape [n] on the operands' device, as 64-bit ones.
Tensor integers(const char* who, const char* name, const Tensor& t, int64_t n, const Tensor& like) {
  no_tangent(who, t);
  TORCH_CHECK_VALUE(at::isIntegralType(t.scalar_type(), false), who, ": ", name, " must be integers, got ",
                    t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 1 && (n < 0 ? t.size(0) >= 1 : t.size(0) == n), who, ": ", name,
                    " must have one value for each sequence", n < 0 ? " and one more" : "", ", got ",
                    t.sizes());
  TORCH_CHECK(t.device() == like.device(), who, ": ", name, " must live on ", like.device());
  return dense(t.to(at::kLong));
}

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, bool causal,
                 const std::optional<int64_t>& window, const std::optional<double>& scale,
                 const OptTensor& kv_lengths, const OptTensor& q_starts, const OptTensor& kv_starts) {
  const char* who = "attention";
  untraced(who);
  for (const Tensor* t : {&q, &k, &v}) no_tangent(who, *t);
  TORCH_CHECK_VALUE(live(q_starts) == live(kv_starts), who, ": q_starts and kv_starts come together");
  AttentionCall c;
  c.packed = live(q_starts);
  TORCH_CHECK_VALUE(!c.packed || !live(kv_lengths), who, ": kv_lengths are of sequences that are not packed");
  const int64_t dims = c.packed ? 3 : 4;
  TORCH_CHECK_VALUE(q.dim() == dims && k.dim() == dims && v.sizes() == k.sizes() &&
                        k.size(-1) == q.size(-1) && (c.packed || k.size(0) == q.size(0)),
                    who, c.packed ? ": packed q [tokens, heads, dim] and k, v [tokens, kv_heads, dim]"
                                  : ": q [batch, tokens, heads, dim] and k, v [batch, tokens, kv_heads, dim]",
                    " do not fit: ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  const int64_t d = q.size(-1), heads = q.size(-2), kv_heads = k.size(-2);
  TORCH_CHECK_VALUE(d >= 8 && d <= 128 && d % 8 == 0, who, ": dim must be a multiple of 8 and 8 .. 128, got ",
                    d);
  TORCH_CHECK_VALUE(kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0, who,
                    ": heads must be a multiple of kv_heads, got ", heads, " and ", kv_heads);
  TORCH_CHECK_VALUE((q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf) &&
                        k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                    who, ": q, k and v must all be bfloat16 or float16, got ", q.scalar_type(), ", ",
                    k.scalar_type(), " and ", v.scalar_type());
  TORCH_CHECK_VALUE(!window.has_value() || (*window >= 1 && causal), who,
                    ": window must be positive, and needs causal");
  c.scale = scale.value_or(1. / std::sqrt((double)d));
  // a normal fp32 number: the kernels multiply by it in fp32
  TORCH_CHECK_VALUE(c.scale >= 0x1p-126 && c.scale < 0x1p127, who,
                    ": scale must be positive and within fp32, got ", c.scale);
  TORCH_CHECK(q.is_cuda() && k.device() == q.device() && v.device() == q.device(), who,
              ": tensors must live on one GPU (HIP kernel only)");
  c.causal = causal;
  c.window = window.value_or(0);
  c.group = heads / kv_heads;
  OptTensor n, qs, ks;
  if (c.packed) {
    qs = integers(who, "q_starts", *q_starts, -1, q);
    ks = integers(who, "kv_starts", *kv_starts, qs->size(0), q);
    c.batch = qs->size(0) - 1;
  } else {
    c.batch = q.size(0);
    if (live(kv_lengths)) n = integers(who, "kv_lengths", *kv_lengths, c.batch, q);
  }
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return Attend::apply(q, k, v, n, qs, ks, c);
  const HeadsView qv(q, false, c.group), kv(k, true, c.group), vv(v, true, c.group);
  return c.forward(qv, kv, vv, n.value_or(Tensor()), qs.value_or(Tensor()), ks.value_or(Tensor()), nullptr, nullptr);
}

// ---- the heads' norms and rotation --------------------------------------------------------------

// [..., heads, dim] with one stride from token to token.
struct TokensView {
  Tensor t;
  int64_t tokens, token, head;
  explicit TokensView(const Tensor& x) : t(x) {
    const int64_t n = x.dim(), h = x.size(n - 2), d = x.size(n - 1);
    tokens = 1;
    for (int64_t i = 0; i < n - 2; ++i) tokens *= x.size(i);
    if (x.is_neg() || x.stride(n - 1) != 1 || !even()) {
      t = dense(x);
      token = h * d;
      head = d;
    }
    ptr(t);                               // refuses tensors without memory
  }

 private:
  bool even() {
    const int64_t n = t.dim();
    head = t.size(n - 2) > 1 ? t.stride(n - 2) : t.size(n - 1);
    token = t.size(n - 2) * t.size(n - 1);
    int64_t next = -1;                    // what the dimension outside must step by
    for (int64_t i = n - 3; i >= 0; --i) {
      if (t.size(i) <= 1) continue;
      if (next < 0) token = t.stride(i);
      else if (t.stride(i) != next) return false;
      next = t.stride(i) * t.size(i);
    }
    return true;
  }
};

dmuon_rotary_heads_args describe_heads(const TokensView& q, const TokensView& k, const Tensor& positions,
                                       const Tensor& inv_freq, const Tensor& wq, const Tensor& wk, double eps,
                                       bool interleaved) {
  dmuon_rotary_heads_args a{};
  a.q = ptr(q.t);
  a.k = ptr(k.t);
  a.positions = static_cast<const int64_t*>(ptr(positions));
  a.inv_freq = ptr(inv_freq);
  a.q_weight = ptr(wq);
  a.k_weight = ptr(wk);
  if (wq.defined()) a.q_weight_dtype = code(wq.scalar_type());
  if (wk.defined()) a.k_weight_dtype = code(wk.scalar_type());
  a.tokens = q.tokens;
  a.period = positions.numel();
  a.heads = q.t.size(-2);
  a.kv_heads = k.t.size(-2);
  a.dim = q.t.size(-1);
  a.rotary_dim = 2 * inv_freq.numel();
  a.q_token = q.token; a.q_head = q.head;
  a.k_token = k.token; a.k_head = k.head;
  a.eps = (float)eps;
  a.interleaved = interleaved;
  a.inv_freq_double = inv_freq.scalar_type() == at::kDouble;
  a.dtype = code(q.t.scalar_type());
  return a;
}

variable_list heads_forward(const TokensView& q, const TokensView& k, const Tensor& positions,
                            const Tensor& inv_freq, const Tensor& wq, const Tensor& wk, double eps,
                            bool interleaved) {
  const c10::DeviceGuard guard(q.t.device());
  auto a = describe_heads(q, k, positions, inv_freq, wq, wk, eps, interleaved);
  Tensor qo = at::empty(q.t.sizes(), q.t.options()), ko = at::empty(k.t.sizes(), k.t.options());
  a.q_out = ptr(qo);
  a.k_out = ptr(ko);
  call(dmuon_rotary_heads(&a, stream_of(q.t)));
  return {qo, ko};
}

struct RotaryHeads : torch::autograd::Function<RotaryHeads> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const OptTensor& wq,
                               const OptTensor& wk, const Tensor& positions, const Tensor& inv_freq,
                               double eps, bool interleaved) {
    const TokensView qv(q), kv(k);
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->save_for_backward({qv.t, kv.t, wq.value_or(Tensor()), wk.value_or(Tensor()), positions, inv_freq});
    ctx->set_materialize_grads(false);
    return heads_forward(qv, kv, positions, inv_freq, wq.value_or(Tensor()), wk.value_or(Tensor()), eps,
                         interleaved);
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("rotary_heads");
    const auto s = ctx->get_saved_variables();
    const c10::DeviceGuard guard(s[0].device());
    const TokensView q(s[0]), k(s[1]);
    auto a = describe_heads(q, k, s[4], s[5], s[2], s[3], ctx->saved_data["eps"].toDouble(),
                            ctx->saved_data["interleaved"].toBool());
    std::optional<TokensView> dq, dk;
    if (grads[0].defined()) {
      dq.emplace(grads[0]);
      a.dq_out = ptr(dq->t);
      a.dq_out_token = dq->token;
      a.dq_out_head = dq->head;
    }
    if (grads[1].defined()) {
      dk.emplace(grads[1]);
      a.dk_out = ptr(dk->t);
      a.dk_out_token = dk->token;
      a.dk_out_head = dk->head;
    }
    variable_list out(8);
    void** place[4] = {&a.dq, &a.dk, &a.d_q_weight, &a.d_k_weight};
    // the operands that are there count as the graph's inputs, in their order
    for (int i = 0, input = 0; i < 4; ++i) {
      if (!s[i].defined()) continue;
      if (!ctx->needs_input_grad(input++)) continue;
      out[i] = at::empty(s[i].sizes(), s[i].options());
      *place[i] = ptr(out[i]);
    }
    int64_t need = 0;
    call(dmuon_rotary_heads_grad_workspace_size(&a, &need));
    const Tensor ws = workspace(need, s[0]);
    call(dmuon_rotary_heads_grad(&a, ws.data_ptr(), need, stream_of(s[0])));
    return out;
  }
};

std::tuple<Tensor, Tensor> rotary_heads(const Tensor& q, const Tensor& k, const Tensor& positions,
                                        const Tensor& inv_freq, const OptTensor& wq, const OptTensor& wk,
                                        double eps, bool interleaved) {
  const char* who = "rotary_heads";
  untraced(who);
  for (const Tensor* t : {&q, &k, &positions, &inv_freq}) no_tangent(who, *t);
  for (const OptTensor* t : {&wq, &wk})
    if (live(*t)) no_tangent(who, **t);
  TORCH_CHECK_VALUE(q.dim() >= 2 && k.dim() == q.dim() && k.size(-1) == q.size(-1) &&
                        q.sizes().slice(0, q.dim() - 2) == k.sizes().slice(0, q.dim() - 2) &&
                        q.size(-2) >= 1 && k.size(-2) >= 1,
                    who, ": q [..., heads, dim] and k [..., kv_heads, dim] do not fit: ", q.sizes(), ", ",
                    k.sizes());
  const int64_t dim = q.size(-1);
  TORCH_CHECK_VALUE(dim >= 2 && dim <= 512 && dim % 2 == 0, who, ": dim must be even and 2 .. 512, got ", dim);
  TORCH_CHECK_VALUE(code(q.scalar_type()) >= 0 && k.scalar_type() == q.scalar_type(), who,
                    ": q and k must have one dtype, float32, bfloat16 or float16, got ", q.scalar_type(),
                    " and ", k.scalar_type());
  TORCH_CHECK_VALUE(at::isIntegralType(positions.scalar_type(), false), who,
                    ": positions must be integers, got ", positions.scalar_type());
  // the trailing part of the leading shape, behind any ones
  const auto lead = q.sizes().slice(0, q.dim() - 2);
  auto shape = positions.sizes();
  while (!shape.empty() && shape[0] == 1 && (shape.size() > lead.size() ||
         shape != lead.slice(lead.size() - shape.size()))) shape = shape.slice(1);
  TORCH_CHECK_VALUE(shape.size() <= lead.size() && shape == lead.slice(lead.size() - shape.size()), who,
                    ": positions ", positions.sizes(), " do not fit the leading shape ", lead);
  TORCH_CHECK_VALUE((inv_freq.scalar_type() == at::kFloat || inv_freq.scalar_type() == at::kDouble) &&
                        inv_freq.dim() == 1 && inv_freq.size(0) >= 1 && 2 * inv_freq.size(0) <= dim,
                    who, ": inv_freq must be float32 or float64 with 1 .. dim / 2 values, got ",
                    inv_freq.scalar_type(), " ", inv_freq.sizes());
  TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && inv_freq.requires_grad()), who,
                    ": inv_freq has no gradient");
  const char* names[2] = {"q_weight", "k_weight"};
  const OptTensor* weights[2] = {&wq, &wk};
  for (int i = 0; i < 2; ++i) {
    if (!live(*weights[i])) continue;
    const Tensor& w = **weights[i];
    TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == dim, who, ": ", names[i], " must be [", dim, "], got ",
                      w.sizes());
    TORCH_CHECK_VALUE(w.scalar_type() == q.scalar_type() || w.scalar_type() == at::kFloat, who, ": ", names[i],
                      " must be ", q.scalar_type(), " or Float, got ", w.scalar_type());
  }
  auto here = [&](const OptTensor& t) { return !live(t) || t->device() == q.device(); };
  TORCH_CHECK(q.is_cuda() && k.device() == q.device() && positions.device() == q.device() &&
                  inv_freq.device() == q.device() && here(wq) && here(wk), who,
              ": tensors must live on one GPU (HIP kernel only)");
  const Tensor p = dense(positions.to(at::kLong)), f = dense(inv_freq);
  OptTensor a, b;
  if (live(wq)) a = dense(*wq);
  if (live(wk)) b = dense(*wk);
  const bool grad = q.requires_grad() || k.requires_grad() || (live(a) && a->requires_grad()) ||
                    (live(b) && b->requires_grad());
  const variable_list out =
      at::GradMode::is_enabled() && grad
          ? RotaryHeads::apply(q, k, a, b, p, f, eps, interleaved)
          : heads_forward(TokensView(q), TokensView(k), p, f, a.value_or(Tensor()), b.value_or(Tensor()), eps,
                          interleaved);
  return {out[0], out[1]};
}

// ---- token lookup -------------------------------------------------------------------------------

struct EmbeddingCall {
  int64_t padding = -1;
  double scale = 1.;
};

Tensor lookup(const Tensor& weight, const Tensor& tokens, const EmbeddingCall& c) {
  const c10::DeviceGuard guard(weight.device());
  const Tensor w = dense_rows(weight);
  auto shape = tokens.sizes().vec();
  shape.push_back(weight.size(1));
  Tensor out = at::empty(shape, weight.options());
  dmuon_embedding_args a{};
  a.tokens = static_cast<const int64_t*>(ptr(tokens));
  a.weight = ptr(w);
  a.out = ptr(out);
  a.tokens_n = tokens.numel();
  a.vocab = weight.size(0);
  a.dim = weight.size(1);
  a.ld_weight = pitch(w);
  a.padding_idx = c.padding;
  a.scale = (float)c.scale;
  a.dtype = code(weight.scalar_type());
  call(dmuon_embedding(&a, stream_of(weight)));
  return out;
}

struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& tokens,
                        const EmbeddingCall& c) {
    ctx->saved_data["padding"] = c.padding;
    ctx->saved_data["scale"] = c.scale;
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->save_for_backward({tokens});
    return lookup(weight, tokens, c);
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("embedding");
    const Tensor tokens = ctx->get_saved_variables()[0];
    const Tensor dy = rows_of(grads[0]);
    const c10::DeviceGuard guard(dy.device());
    Tensor dw = at::empty({ctx->saved_data["vocab"].toInt(), dy.size(1)}, dy.options());
    dmuon_embedding_args a{};
    a.tokens = static_cast<const int64_t*>(ptr(tokens));
    a.dy = ptr(dy);
    a.d_weight = ptr(dw);
    a.tokens_n = tokens.numel();
    a.vocab = dw.size(0);
    a.dim = dw.size(1);
    a.ld_dy = pitch(dy);
    a.padding_idx = ctx->saved_data["padding"].toInt();
    a.scale = (float)ctx->saved_data["scale"].toDouble();
    a.dtype = code(dy.scalar_type());
    int64_t need = 0;
    call(dmuon_embedding_grad_workspace_size(&a, &need));
    const Tensor ws = workspace(need, dy);
    call(dmuon_embedding_grad(&a, ws.data_ptr(), need, stream_of(dy)));
    return {dw, Tensor(), Tensor()};
  }
};

Tensor embedding(const Tensor& tokens, const Tensor& weight, double scale,
                 const std::optional<int64_t>& padding_idx) {
  const char* who = "embedding";
  untraced(who);
  no_tangent(who, weight);
  no_tangent(who, tokens);
  TORCH_CHECK_VALUE(at::isIntegralType(tokens.scalar_type(), false), who, ": tokens must be integers, got ",
                    tokens.scalar_type());
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) >= 1 && weight.size(1) >= 1 &&
                        weight.size(1) <= (1 << 20), who,
                    ": weight must be [vocab, dim] with dim up to 2^20, got ", weight.sizes());
  TORCH_CHECK_VALUE(code(weight.scalar_type()) >= 0, who, ": unsupported dtype ", weight.scalar_type());
  // the kernels multiply by it in fp32
  TORCH_CHECK_VALUE(scale == 0. || (std::abs(scale) >= 0x1p-126 && std::abs(scale) <= 0x1.fffffep127), who,
                    ": scale must be 0 or within fp32, got ", scale);
  EmbeddingCall c;
  c.scale = scale;
  if (padding_idx.has_value()) {
    c.padding = *padding_idx < 0 ? *padding_idx + weight.size(0) : *padding_idx;
    TORCH_CHECK_VALUE(c.padding >= 0 && c.padding < weight.size(0), who, ": padding_idx ", *padding_idx,
                      " is not within the vocabulary of ", weight.size(0));
  }
  TORCH_CHECK(weight.is_cuda() && tokens.device() == weight.device(), who,
              ": tensors must live on one GPU (HIP kernel only)");
  const Tensor t = dense(tokens.to(at::kLong));
  if (at::GradMode::is_enabled() && weight.requires_grad()) return Embedding::apply(weight, t, c);
  return lookup(weight, t, c);
}

}  // namespace
