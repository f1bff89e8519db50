// Autograd operators on the C ABI of libdmuon_amd.so: argument checks, allocation, and the forward
// and backward calls, as one Python extension module.
//
// The operators run many times a second on small tensors, where a Python autograd function costs
// several times the GPU's work: its backward pass takes the interpreter's lock in another thread.
// Here neither direction needs the interpreter.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <optional>

#include "../../include/dmuon_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

int code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return DMUON_DTYPE_F32;
    case at::kBFloat16: return DMUON_DTYPE_BF16;
    case at::kHalf: return DMUON_DTYPE_F16;
    default: return -1;
  }
}

void call(int rc) { TORCH_CHECK(rc == 0, "dmuon_amd: ", dmuon_last_error()); }

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

bool live(const OptTensor& t) { return t.has_value() && t->defined(); }
// NULL stands for an operand that is not there: a subclass that wraps other tensors (a distributed
// one) must not pass for that.
void* ptr(const Tensor& t) {
  if (!t.defined()) return nullptr;
  void* p = t.data_ptr();
  TORCH_CHECK(p || t.numel() == 0, "dmuon_amd: a tensor without memory of its own (a wrapper subclass) "
              "cannot be an operand");
  return p;
}
void* ptr(const OptTensor& t) { return live(t) ? ptr(*t) : nullptr; }

// Torch may put a view's negation off; the kernels read what lies in memory.
Tensor dense(const Tensor& t) { return t.resolve_neg().contiguous(); }

// The same matrix with its last dimension contiguous and rows that do not overlap.
Tensor dense_rows(const Tensor& t) {
  if (t.is_neg()) return dense(t);
  if ((t.stride(1) == 1 || t.size(1) == 1) && (t.stride(0) >= t.size(1) || t.size(0) <= 1)) return t;
  return t.contiguous();
}
int64_t pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// A two-dimensional tensor takes no view: it would be a node of the gradient's graph.
Tensor rows_of(const Tensor& t) {
  return dense_rows(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}));
}

Tensor workspace(int64_t bytes, const Tensor& like) {
  // from the caching allocator: reused in this stream's order, nothing is kept
  return at::empty({bytes}, like.options().dtype(at::kByte));
}

void once(const char* who) {
  TORCH_CHECK(!at::GradMode::is_enabled(), who,
              ": the gradient has no gradient of its own (create_graph=True)");
}

// The kernels write into memory that torch has only seen allocated. A recorder of its operators would
// keep the allocation alone and replay it, and a tangent (forward-mode gradient) would be lost where no
// operand asks for the other kind: both are refused.
void untraced(const char* who) {
  const bool graph = c10::impl::TorchDispatchModeTLS::get_mode(
      c10::impl::TorchDispatchModeKey::PROXY).has_value();
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !graph, who,
              ": cannot be recorded by a tracer (torch.jit.trace, make_fx)");
}
void no_tangent(const char* who, const Tensor& t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), who, ": has no forward-mode gradient (dual tensors)");
}

// ---- losses over a vocabulary -------------------------------------------------------------------

// What a call is measured against, and what its backward pass needs besides hidden and weight.
struct Loss : torch::CustomClassHolder {
  const char* who = "";
  Tensor targets, ids, logits, lse;
  int64_t ignore_index = -100, k_list = 1, chunk = 0;
  double z_loss = 0., temperature = 1.;
  int reduction = DMUON_LOSS_MEAN;
  bool want_hidden = false, want_weight = false;
  at::ScalarType held = at::kFloat;       // the type the gradients are formed in
  Tensor d_hidden, d_weight;              // until the first backward pass takes them

  void against(const Tensor& t, const Tensor& i, const Tensor& l, const Tensor& e) {
    targets = t;
    ids = i;
    logits = l;
    lse = e;
  }

  // The loss of each token or reduced; the gradients into d_hidden and d_weight.
  Tensor launch(const Tensor& hidden, const Tensor& weight, bool grads, const Tensor& row_grad) {
    const c10::DeviceGuard guard(hidden.device());
    const int64_t n = hidden.size(0), dim = hidden.size(1), vocab = weight.size(0);
    const auto f32 = hidden.options().dtype(at::kFloat);
    Tensor loss = reduction == DMUON_LOSS_ROWS ? at::empty({n}, f32) : at::empty({}, f32);
    if (grads && want_hidden) d_hidden = at::empty({n, dim}, hidden.options().dtype(held));
    if (grads && want_weight) d_weight = at::empty({vocab, dim}, hidden.options().dtype(held));
    dmuon_head_loss_args a{};
    a.hidden = ptr(hidden);
    a.weight = ptr(weight);
    a.targets = static_cast<const int64_t*>(ptr(targets));
    a.teacher_ids = static_cast<const int64_t*>(ptr(ids));
    a.teacher_logits = static_cast<const float*>(ptr(logits));
    a.teacher_lse = static_cast<const float*>(ptr(lse));
    a.row_grad = static_cast<const float*>(ptr(row_grad));
    (reduction == DMUON_LOSS_ROWS ? a.loss : a.reduced) = loss.data_ptr<float>();
    a.d_hidden = grads && want_hidden ? d_hidden.data_ptr() : nullptr;
    a.d_weight = grads && want_weight ? d_weight.data_ptr() : nullptr;
    a.ld_hidden = pitch(hidden);
    a.ld_weight = pitch(weight);
    a.tokens = n;
    a.vocab = vocab;
    a.dim = dim;
    a.k_list = k_list;
    a.chunk_tokens = chunk;
    a.ignore_index = ignore_index;
    a.z_loss = (float)z_loss;
    a.temperature = (float)temperature;
    a.dtype = code(hidden.scalar_type());
    a.grad_dtype = code(held);
    a.reduction = reduction;
    int64_t need = 0;
    call(dmuon_head_loss_workspace_size(&a, &need));
    const Tensor ws = workspace(need, hidden);
    call(dmuon_head_loss(&a, ws.data_ptr(), need, stream_of(hidden)));
    return loss;
  }

  // d_hidden and d_weight times `factor` in the operands' type, in place where they have it: bf16
  // gradients, rounded when they were formed, round a second time for a factor that is no power of two
  // (2^-8 again; holding them in fp32 would take twice their memory from one pass to the other).
  void scale(const Tensor& factor, at::ScalarType dtype) {
    const c10::DeviceGuard guard(factor.device());
    Tensor* g[2] = {&d_hidden, &d_weight};
    Tensor out[2];
    for (int i = 0; i < 2; ++i)
      if (g[i]->defined())
        out[i] = held == dtype ? *g[i] : at::empty(g[i]->sizes(), g[i]->options().dtype(dtype));
    const Tensor f = dense(factor.to(at::kFloat));
    call(dmuon_scale_by(ptr(d_hidden), ptr(out[0]), d_hidden.defined() ? d_hidden.numel() : 0,
                        ptr(d_weight), ptr(out[1]), d_weight.defined() ? d_weight.numel() : 0,
                        code(held), code(dtype), static_cast<const float*>(ptr(f)), stream_of(f)));
    d_hidden = out[0];
    d_weight = out[1];
  }
};
using LossPtr = c10::intrusive_ptr<Loss>;

struct HeadLoss : torch::autograd::Function<HeadLoss> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight,
                        const LossPtr& s) {
    const Tensor loss = s->launch(hidden, weight, s->reduction != DMUON_LOSS_ROWS, Tensor());
    ctx->saved_data["call"] = c10::IValue::make_capsule(s);
    // the targets too: a pass that forms the logits anew must not see others than the loss did
    ctx->save_for_backward({hidden, weight, s->targets, s->ids, s->logits, s->lse});
    s->against({}, {}, {}, {});
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const LossPtr s =
        c10::static_intrusive_pointer_cast<Loss>(ctx->saved_data["call"].toCapsule());
    once(s->who);
    const auto saved = ctx->get_saved_variables();
    s->against(saved[2], saved[3], saved[4], saved[5]);
    if (s->reduction == DMUON_LOSS_ROWS) {
      s->launch(saved[0], saved[1], true, dense(grads[0].to(at::kFloat)));
    } else {
      // a second pass over a kept graph forms them anew
      if (!s->d_hidden.defined() && !s->d_weight.defined()) s->launch(saved[0], saved[1], true, Tensor());
      s->scale(grads[0], saved[0].scalar_type());
    }
    s->against({}, {}, {}, {});
    Tensor dh = std::move(s->d_hidden), dw = std::move(s->d_weight);
    s->d_hidden = Tensor();
    s->d_weight = Tensor();
    return {dh, dw, Tensor()};
  }
};

void check_head(const char* who, const Tensor& hidden, const Tensor& weight) {
  untraced(who);
  no_tangent(who, hidden);
  no_tangent(who, weight);
  TORCH_CHECK_VALUE(hidden.dim() >= 1 && weight.dim() == 2 && hidden.size(-1) == weight.size(1), who,
                    ": hidden [..., dim] and weight [vocab, dim] do not fit: ", hidden.sizes(), ", ",
                    weight.sizes());
  TORCH_CHECK_VALUE(weight.size(0) >= 1 && weight.size(1) >= 1, who, ": weight has no values: ",
                    weight.sizes());
  TORCH_CHECK_VALUE((hidden.scalar_type() == at::kBFloat16 || hidden.scalar_type() == at::kHalf) &&
                        weight.scalar_type() == hidden.scalar_type(),
                    who, ": hidden and weight must both be bfloat16 or float16, got ",
                    hidden.scalar_type(), " and ", weight.scalar_type());
  TORCH_CHECK(hidden.is_cuda() && weight.device() == hidden.device(), who,
              ": tensors must live on one GPU (HIP kernel only)");
}

// An operand of the tokens: [*hidden's leading shape], or [*leading, k].
Tensor of_tokens(const char* who, const char* name, const Tensor& t, const Tensor& hidden, int64_t k,
                 bool integers) {
  const bool fits = integers ? at::isIntegralType(t.scalar_type(), false)
                             : at::isFloatingType(t.scalar_type());
  TORCH_CHECK_VALUE(fits, who, ": ", name, integers ? " must be integers" : " must be floating-point",
                    ", got ", t.scalar_type());
  auto shape = hidden.sizes().slice(0, hidden.dim() - 1).vec();
  if (k > 0) shape.push_back(k);
  TORCH_CHECK_VALUE(t.sizes() == at::IntArrayRef(shape), who, ": ", name, " must have the shape ",
                    at::IntArrayRef(shape), ", got ", t.sizes());
  TORCH_CHECK(t.device() == hidden.device(), who, ": ", name, " must live on ", hidden.device());
  return dense(t.detach().to(integers ? at::kLong : at::kFloat));
}

Tensor run_loss(const LossPtr& s, const Tensor& hidden, const Tensor& weight) {
  const bool grad = at::GradMode::is_enabled();
  s->want_hidden = grad && hidden.requires_grad();
  s->want_weight = grad && weight.requires_grad();
  // fp16: the mean's gradients may only fit the type once a loss scale has multiplied them
  s->held = hidden.scalar_type() == at::kHalf && s->reduction != DMUON_LOSS_ROWS
                ? at::kFloat : hidden.scalar_type();
  const Tensor rows = rows_of(hidden), w = dense_rows(weight);
  const Tensor out = s->want_hidden || s->want_weight ? HeadLoss::apply(rows, w, s)
                                                      : s->launch(rows, w, false, Tensor());
  if (s->reduction != DMUON_LOSS_ROWS || hidden.dim() == 2) return out;
  return out.view(hidden.sizes().slice(0, hidden.dim() - 1));
}

Tensor linear_cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& target,
                            int64_t ignore_index, double z_loss, int64_t reduction, int64_t chunk) {
  const char* who = "linear_cross_entropy";
  check_head(who, hidden, weight);
  auto s = c10::make_intrusive<Loss>();
  s->who = who;
  s->targets = of_tokens(who, "target", target, hidden, 0, true);
  s->ignore_index = ignore_index;
  s->z_loss = z_loss;
  s->reduction = (int)reduction;
  s->chunk = chunk;
  return run_loss(s, hidden, weight);
}

Tensor linear_distillation(const Tensor& hidden, const Tensor& weight, const Tensor& ids,
                           const Tensor& logits, const OptTensor& lse, double temperature,
                           int64_t reduction, int64_t chunk) {
  const char* who = "linear_distillation";
  check_head(who, hidden, weight);
  TORCH_CHECK_VALUE(ids.dim() == hidden.dim() && ids.size(-1) >= 1 && ids.size(-1) <= 4096, who,
                    ": teacher_ids must be [..., k] with 1 <= k <= 4096, got ", ids.sizes());
  auto s = c10::make_intrusive<Loss>();
  s->who = who;
  s->k_list = ids.size(-1);
  s->ids = of_tokens(who, "teacher_ids", ids, hidden, s->k_list, true);
  s->logits = of_tokens(who, "teacher_logits", logits, hidden, s->k_list, false);
  if (live(lse)) s->lse = of_tokens(who, "teacher_lse", *lse, hidden, 0, false);
  s->temperature = temperature;
  s->reduction = (int)reduction;
  s->chunk = chunk;
  return run_loss(s, hidden, weight);
}

// ---- norms around a block -----------------------------------------------------------------------

dmuon_residual_norm_args describe(const Tensor& x, const OptTensor& y, const Tensor& pre,
                                  const OptTensor& post, const OptTensor& gate, double scale,
                                  double eps) {
  dmuon_residual_norm_args a{};
  a.x = ptr(x);
  a.rows = x.size(0);
  a.dim = x.size(1);
  a.ld_x = pitch(x);
  a.dtype = code(x.scalar_type());
  a.y = ptr(y);
  if (live(y)) a.ld_y = pitch(*y);
  a.w_pre = ptr(pre);
  a.pre_dtype = code(pre.scalar_type());
  a.w_post = ptr(post);
  if (live(post)) a.post_dtype = code(post->scalar_type());
  a.gate = ptr(gate);
  if (live(gate)) {
    a.gate_dtype = code(gate->scalar_type());
    a.gates = gate->size(0);
  }
  a.scale = (float)scale;
  a.eps = (float)eps;
  return a;
}

// (x_new, h), or h alone where x_new is x; stats for the backward pass.
variable_list norm_forward(const Tensor& x, const OptTensor& y, const Tensor& pre,
                           const OptTensor& post, const OptTensor& gate, double scale, double eps,
                           Tensor* stats) {
  const c10::DeviceGuard guard(x.device());
  auto a = describe(x, y, pre, post, gate, scale, eps);
  Tensor h = at::empty(x.sizes(), x.options()), x_new;
  if (live(y) || scale != 1.) x_new = at::empty(x.sizes(), x.options());
  if (stats) {
    *stats = at::empty({x.size(0), 2}, x.options().dtype(at::kFloat));
    a.stats = stats->data_ptr<float>();
  }
  a.h = h.data_ptr();
  a.x_new = ptr(x_new);
  call(dmuon_residual_norm(&a, stream_of(x)));
  if (x_new.defined()) return {x_new, h};
  return {h};
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& y,
                               const Tensor& pre, const OptTensor& post, const OptTensor& gate,
                               double scale, double eps) {
    Tensor stats;
    variable_list out = norm_forward(x, y, pre, post, gate, scale, eps, &stats);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->save_for_backward({x, y.value_or(Tensor()), pre, post.value_or(Tensor()),
                            gate.value_or(Tensor()), stats});
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("residual_norm");
    const auto s = ctx->get_saved_variables();
    const Tensor& x = s[0];
    const c10::DeviceGuard guard(x.device());
    auto a = describe(x, s[1], s[2], s[3], s[4], ctx->saved_data["scale"].toDouble(),
                      ctx->saved_data["eps"].toDouble());
    a.stats = static_cast<float*>(s[5].data_ptr());
    Tensor dx_new = grads.size() == 2 ? grads[0] : Tensor(), dh = grads.back();
    if (dx_new.defined()) {
      dx_new = dense_rows(dx_new);
      a.dx_new = ptr(dx_new);
      a.ld_dx_new = pitch(dx_new);
    }
    if (dh.defined()) {
      dh = dense_rows(dh);
      a.dh = ptr(dh);
      a.ld_dh = pitch(dh);
    }
    variable_list out(7);
    void** place[5] = {&a.dx, &a.dy, &a.d_pre, &a.d_post, &a.d_gate};
    // the operands that are there count as the graph's inputs, in their order
    for (int i = 0, input = 0; i < 5; ++i) {
      if (!s[i].defined()) continue;
      if (!ctx->needs_input_grad(input++)) continue;
      out[i] = at::empty(s[i].sizes(), s[i].options());
      *place[i] = out[i].data_ptr();
    }
    int64_t need = 0;
    call(dmuon_residual_norm_grad_workspace_size(&a, &need));
    const Tensor ws = workspace(need, x);
    call(dmuon_residual_norm_grad(&a, ws.data_ptr(), need, stream_of(x)));
    return out;
  }
};

// The gate as [g, dim], row i for the i-th of g equal runs of x's rows.
Tensor gate_rows(const char* who, const Tensor& gate, const Tensor& x) {
  const int64_t dim = x.size(-1);
  bool fits = gate.dim() >= 1 && gate.size(-1) == dim;
  if (fits && x.dim() == 2 && gate.dim() == 2) {
    fits = gate.size(0) >= 1 && x.size(0) % gate.size(0) == 0;
  } else if (fits && gate.dim() > 1) {
    // leading dimensions of x, then ones: what broadcasting spreads over consecutive rows
    fits = gate.dim() == x.dim();
    int64_t same = 0;
    while (fits && same < gate.dim() - 1 && gate.size(same) == x.size(same)) ++same;
    for (; fits && same < gate.dim() - 1; ++same) fits = gate.size(same) == 1;
  }
  TORCH_CHECK_VALUE(fits, who, ": a gate of ", gate.sizes(),
                    " has no row for each of equal runs of the rows of x ", x.sizes());
  // no row at all: one that no row of x uses, behind the gate's own
  if (gate.numel() == 0) return at::cat({gate.reshape({0, dim}), gate.new_zeros({1, dim})});
  return dense(gate.dim() == 2 ? gate : gate.reshape({-1, dim}));
}

std::tuple<Tensor, Tensor> residual_norm(const Tensor& x, const OptTensor& y, const Tensor& pre,
                                         const OptTensor& post, const OptTensor& gate, double scale,
                                         double eps, int64_t most) {
  const char* who = "residual_norm";
  untraced(who);
  no_tangent(who, x);
  no_tangent(who, pre);
  for (const OptTensor* t : {&y, &post, &gate})
    if (live(*t)) no_tangent(who, **t);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= most, who,
                    ": x must be [..., dim] with 1 <= dim <= ", most, ", got ", x.sizes());
  TORCH_CHECK_VALUE(code(x.scalar_type()) >= 0, who, ": unsupported dtype ", x.scalar_type());
  const int64_t dim = x.size(-1);
  TORCH_CHECK_VALUE(!live(y) || (y->sizes() == x.sizes() && y->scalar_type() == x.scalar_type()),
                    who, ": y must match x (", x.sizes(), ", ", x.scalar_type(), ")");
  TORCH_CHECK_VALUE(live(y) || (!live(post) && !live(gate)), who,
                    ": post_weight and gate need the block's output y");
  auto weight = [&](const char* name, const Tensor& t) {
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == dim, who, ": ", name, " must be [", dim,
                      "], got ", t.sizes());
  };
  weight("pre_weight", pre);
  if (live(post)) weight("post_weight", *post);
  OptTensor g;
  if (live(gate)) g = gate_rows(who, *gate, x);
  auto type = [&](const char* name, const Tensor& t) {
    TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, who, ": ",
                      name, " must be ", x.scalar_type(), " or Float, got ", t.scalar_type());
  };
  type("pre_weight", pre);
  if (live(post)) type("post_weight", *post);
  if (live(g)) type("gate", *g);
  auto here = [&](const OptTensor& t) { return !live(t) || t->device() == x.device(); };
  TORCH_CHECK(x.is_cuda() && here(y) && pre.device() == x.device() && here(post) && here(g), who,
              ": tensors must live on one GPU (HIP kernel only)");
  const Tensor rows = rows_of(x), w = dense(pre);
  OptTensor yr, p;
  if (live(y)) yr = rows_of(*y);
  if (live(post)) p = dense(*post);
  bool grad = x.requires_grad() || w.requires_grad();
  for (const OptTensor* t : {&yr, &p, &g}) grad = grad || (live(*t) && (*t)->requires_grad());
  const variable_list out = at::GradMode::is_enabled() && grad
                                ? ResidualNorm::apply(rows, yr, w, p, g, scale, eps)
                                : norm_forward(rows, yr, w, p, g, scale, eps, nullptr);
  Tensor x_new = out.size() == 2 ? out[0] : x, h = out.back();
  if (x.dim() == 2) return {x_new, h};
  return {x_new.view(x.sizes()), h.view(x.sizes())};
}

}  // namespace

PYBIND11_MODULE(_dmuon_torch, m) {
  m.attr("abi_version") = DMUON_ABI_VERSION;
  m.attr("torch_version") = DMUON_TORCH;
  const auto free = py::call_guard<py::gil_scoped_release>();
  m.def("linear_cross_entropy", &linear_cross_entropy, free);
  m.def("linear_distillation", &linear_distillation, free);
  m.def("residual_norm", &residual_norm, free);
}
