"""The operators around the optimizer step as cases that can be timed and checked one by one: the
loss over the vocabulary with its gradients (``linear_cross_entropy``, ``linear_distillation``) and
the norms around a block (``residual_norm``).

A case names the operator (``kind``), its sizes and its options. ``mode`` is what the caller does:
``train`` asks for the gradients too, ``score`` for the values alone. With ``own`` false ``run``
computes the same in elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # one token's likelihood under the benchmark model's head (128256 x 4096)
        dict(name="ce_one_token", kind="ce", mode="score", tokens=1, vocab=128256, dim=4096,
             dtype="bf16", ignored=0.0, z_loss=0.0),
        # a unit-test sized model: odd vocabulary, rows that are no multiple of a vector
        dict(name="ce_small_odd", kind="ce", mode="train", tokens=77, vocab=1003, dim=300,
             dtype="fp16", ignored=0.1, z_loss=0.0),
        # a mid-sized model's micro-batch, one position short of a tile
        dict(name="ce_mid", kind="ce", mode="train", tokens=2047, vocab=32001, dim=2048,
             dtype="bf16", ignored=0.0, z_loss=0.0),
        # validation: every token's loss, no gradient
        dict(name="ce_validation", kind="ce", mode="score", tokens=4096, vocab=128256, dim=4096,
             dtype="bf16", ignored=0.25, z_loss=0.0),
        # the head of one training step of the benchmark model, prompt positions ignored
        dict(name="ce_training", kind="ce", mode="train", tokens=8192, vocab=128256, dim=4096,
             dtype="bf16", ignored=0.1, z_loss=1e-4),
        # a small student, a handful of teacher logits
        dict(name="kd_small", kind="kd", mode="train", tokens=64, vocab=8192, dim=512, k=8,
             dtype="bf16", temperature=1.0, full=False),
        # a ragged student with a softened teacher, fp16
        dict(name="kd_ragged", kind="kd", mode="train", tokens=1023, vocab=50001, dim=1528, k=33,
             dtype="fp16", temperature=2.0, full=False),
        # the benchmark model as the student, the teacher's true probabilities of its top 64
        dict(name="kd_training", kind="kd", mode="train", tokens=4096, vocab=128256, dim=4096, k=64,
             dtype="bf16", temperature=1.0, full=True),
        # one token between two blocks
        dict(name="norm_one_token", kind="norm", mode="score", tokens=1, dim=4096, dtype="bf16",
             weights="fp32", post=True, gates=1, scale=1.0),
        # odd rows in fp32 with a gate per sequence
        dict(name="norm_odd", kind="norm", mode="train", tokens=777, dim=1001, dtype="fp32",
             weights="fp32", post=True, gates=3, scale=0.7),
        # generation or validation: wide rows, no gate
        dict(name="norm_forward", kind="norm", mode="score", tokens=8192, dim=8192, dtype="bf16",
             weights="bf16", post=True, gates=0, scale=1.0),
        # between two blocks of the benchmark model in a training step
        dict(name="norm_training", kind="norm", mode="train", tokens=16384, dim=4096, dtype="bf16",
             weights="fp32", post=True, gates=1, scale=1.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("ce", "ce", "kd", "norm", "norm"))
    mode = rng.choice(("train", "train", "score"))
    if kind == "norm":
        gates = rng.choice((0, 1, 1, 2, 4))
        tokens = max(gates, 1) * _log_int(rng, 1, 16384 // max(gates, 1))
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        return dict(kind=kind, mode=mode, tokens=tokens, dim=_log_int(rng, 64, 8192 if
                    dtype != "fp32" else 4096), dtype=dtype, weights=rng.choice(("fp32", dtype)),
                    post=rng.random() < 0.7, gates=gates, scale=rng.choice((1.0, 0.5)))
    dim = _log_int(rng, 64, 4096)
    if rng.random() < 0.7:                 # most models' widths are whole vectors
        dim = -(-dim // 8) * 8
    case = dict(kind=kind, mode=mode, tokens=_log_int(rng, 1, 8192),
                vocab=_log_int(rng, 1000, 128256), dim=dim, dtype=rng.choice(("bf16", "bf16", "fp16")))
    if kind == "ce":
        case.update(ignored=rng.choice((0.0, 0.1, 0.5)), z_loss=rng.choice((0.0, 0.0, 1e-4)))
    else:
        case.update(k=_log_int(rng, 1, 128), temperature=rng.choice((1.0, 1.0, 2.0)),
                    full=rng.random() < 0.5)
    return case


# ---- inputs -----------------------------------------------------------------------------------

def _randn(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n, d, dt = case["tokens"], case["dim"], DTYPES[case["dtype"]]
    train = case["mode"] == "train"
    state = dict(case=case)
    if case["kind"] == "norm":
        wt = DTYPES[case["weights"]]
        g = case["gates"]
        state["x"] = (2.0 * _randn(gen, n, d)).to(dt)
        state["y"] = (0.5 * _randn(gen, n, d)).to(dt)
        state["pre"] = (1 + 0.1 * _randn(gen, d)).to(wt)
        state["post"] = (1 + 0.1 * _randn(gen, d)).to(wt) if case["post"] else None
        state["gate"] = (0.5 + 0.1 * _randn(gen, g, d)).to(wt) if g else None
        if train:
            state["dx_new"] = (1e-2 * _randn(gen, n, d)).to(dt)
            state["dh"] = (1e-2 * _randn(gen, n, d)).to(dt)
            for k in ("x", "y", "pre", "post", "gate"):
                if state[k] is not None:
                    state[k].requires_grad_(True)
        return state
    v = case["vocab"]
    w = _randn(gen, v, d).mul_(0.02)
    target = torch.randint(0, v, (n,), device=DEV, generator=gen)
    # normed hidden states that lean towards their next token: losses between 0 and log(vocab)
    lean = w[target] * (10.0 / (0.02 * 0.02 * d))
    h = _randn(gen, n, d) + lean * torch.rand(n, 1, device=DEV, generator=gen)
    state["hidden"], state["weight"] = h.to(dt), w.to(dt)
    if case["kind"] == "ce":
        drop = torch.rand(n, device=DEV, generator=gen) < case["ignored"]
        drop[0] = False
        state["target"] = torch.where(drop, -100, target)
    else:
        k, t = min(case["k"], v), case["temperature"]
        step = torch.randint(1, v // k + 1, (n, 1), device=DEV, generator=gen)
        ids = (target[:, None] + step * torch.arange(k, device=DEV)) % v
        fall = torch.rand(n, k, device=DEV, generator=gen).cumsum(1)
        logits = 18.0 - fall
        # shorter lists, and now and then no teacher at all
        keep = torch.randint(1, 2 * k + 1, (n, 1), device=DEV, generator=gen)
        keep[torch.rand(n, 1, device=DEV, generator=gen) < 0.05] = 0
        keep[0] = k
        state["ids"] = torch.where(torch.arange(k, device=DEV) < keep, ids, -1)
        state["logits"] = logits
        lse = torch.logsumexp(logits / t, 1)
        state["teacher_lse"] = lse + 0.3 * torch.rand(n, device=DEV, generator=gen) \
            if case["full"] else None
    if train:
        state["hidden"].requires_grad_(True)
        state["weight"].requires_grad_(True)
    return state


# ---- one pass ---------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["kind"]](state, case)


def _own_loss(state, case, call):
    if case["mode"] == "score":
        with torch.no_grad():
            return {"loss": call("none")}
    loss = call("mean")
    dh, dw = torch.autograd.grad(loss, (state["hidden"], state["weight"]))
    return {"loss": loss.detach(), "d_hidden": dh, "d_weight": dw}


def _own_ce(state, case):
    import dmuon_amd as dmuon
    return _own_loss(state, case, lambda reduction: dmuon.linear_cross_entropy(
        state["hidden"], state["weight"], state["target"], z_loss=case["z_loss"],
        reduction=reduction))


def _own_kd(state, case):
    import dmuon_amd as dmuon
    return _own_loss(state, case, lambda reduction: dmuon.linear_distillation(
        state["hidden"], state["weight"], state["ids"], state["logits"],
        teacher_lse=state["teacher_lse"], temperature=case["temperature"], reduction=reduction))


def _own_norm(state, case):
    import dmuon_amd as dmuon

    def call():
        return dmuon.residual_norm(state["x"], state["y"], state["pre"], post_weight=state["post"],
                                   gate=state["gate"], residual_scale=case["scale"], eps=EPS)
    if case["mode"] == "score":
        with torch.no_grad():
            x_new, h = call()
        return {"x": x_new, "h": h}
    x_new, h = call()
    names = [k for k in ("x", "y", "pre", "post", "gate") if state[k] is not None]
    grads = torch.autograd.grad((x_new, h), [state[k] for k in names],
                                (state["dx_new"], state["dh"]))
    return {"x": x_new.detach(), "h": h.detach(), **{"d_" + k: g for k, g in zip(names, grads)}}


def _plain_products(state, case, p, sub, sub_ids, coef):
    """Gradients of a loss whose logit gradient is coef (p - sub at sub_ids)."""
    p.mul_(coef[:, None])
    p.scatter_add_(1, sub_ids, -(coef[:, None] * sub))
    h, w = state["hidden"].detach(), state["weight"].detach()
    return {"d_hidden": (p @ w.float()).to(h.dtype), "d_weight": (p.t() @ h.float()).to(w.dtype)}


@torch.no_grad()
def _plain_ce(state, case):
    h, w, target = state["hidden"], state["weight"], state["target"]
    z = h.float() @ w.float().t()
    top = z.amax(1, keepdim=True)
    at = target.clamp(min=0)[:, None]
    z_at = z.gather(1, at)
    z.sub_(top).exp_()
    total = z.sum(1, keepdim=True)
    lse = total.log() + top
    counted = target != -100
    loss = torch.where(counted, (lse - z_at + case["z_loss"] * lse * lse)[:, 0], 0.0)
    if case["mode"] == "score":
        return {"loss": loss}
    count = counted.sum().clamp(min=1)
    p = z.div_(total).mul_(1 + 2 * case["z_loss"] * lse)
    return {"loss": loss.sum() / count,
            **_plain_products(state, case, p, torch.ones_like(z_at), at, counted / count)}


@torch.no_grad()
def _plain_kd(state, case):
    h, w, ids, t = state["hidden"], state["weight"], state["ids"], case["temperature"]
    live = ids >= 0
    counted = live.any(1)
    soft = torch.where(live, state["logits"] / t, float("-inf"))
    if state["teacher_lse"] is None:
        high = torch.where(counted[:, None], soft.amax(1, keepdim=True), 0.0)
        q = (soft - high).exp()
        q = q / q.sum(1, keepdim=True).clamp(min=1e-30)
    else:
        q = (soft - state["teacher_lse"][:, None]).exp()
    z = (h.float() @ w.float().t()).div_(t)
    top = z.amax(1, keepdim=True)
    at = ids.clamp(min=0)
    z_at = z.gather(1, at)
    z.sub_(top).exp_()
    total = z.sum(1, keepdim=True)
    lse = total.log() + top
    terms = torch.where(q > 0, q * (q.log() - (z_at - lse)), 0.0)
    loss = t * t * terms.sum(1)
    if case["mode"] == "score":
        return {"loss": loss}
    count = counted.sum().clamp(min=1)
    p = z.div_(total).mul_(q.sum(1, keepdim=True))
    return {"loss": loss.sum() / count,
            **_plain_products(state, case, p, q, at, t * counted / count)}


@torch.no_grad()
def _plain_norm(state, case):
    x, y, a, n, d = state["x"], state["y"], case["scale"], case["tokens"], case["dim"]
    groups = max(case["gates"], 1)
    post = state["post"].float() if case["post"] else None
    gate = state["gate"].float().repeat_interleave(n // groups, 0) if case["gates"] else None
    xf, yf, pre = x.float(), y.float(), state["pre"].float()
    r = (yf.square().mean(1, keepdim=True) + EPS).rsqrt()
    u = yf * r * post if case["post"] else yf
    x_new = a * xf + (gate * u if case["gates"] else u)
    s = (x_new.square().mean(1, keepdim=True) + EPS).rsqrt()
    x_hat = x_new * s
    out = {"x": x_new.to(x.dtype), "h": (x_hat * pre).to(x.dtype)}
    if case["mode"] == "score":
        return out
    e, dh = state["dx_new"].float(), state["dh"].float()
    g = dh * pre
    dx_new = e + s * (g - x_hat * (g * x_hat).mean(1, keepdim=True))
    du = dx_new * gate if case["gates"] else dx_new
    out["d_x"] = (a * dx_new).to(x.dtype)
    out["d_pre"] = (dh * x_hat).sum(0).to(state["pre"].dtype)
    if case["gates"]:
        out["d_gate"] = (dx_new * u).view(groups, -1, d).sum(1).to(state["gate"].dtype)
    if case["post"]:
        y_hat = yf * r
        out["d_post"] = (du * y_hat).sum(0).to(state["post"].dtype)
        g = du * post
        out["d_y"] = (r * (g - y_hat * (g * y_hat).mean(1, keepdim=True))).to(y.dtype)
    else:
        out["d_y"] = du.to(y.dtype)
    return out


_plain = {"ce": _plain_ce, "kd": _plain_kd, "norm": _plain_norm}
_own = {"ce": _own_ce, "kd": _own_kd, "norm": _own_norm}


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    n, d = case["tokens"], case["dim"]
    size = 4 if case["dtype"] == "fp32" else 2
    train = case["mode"] == "train"
    if case["kind"] == "norm":
        params = d * (1 + case["post"] + case["gates"]) * (4 if case["weights"] == "fp32" else 2)
        passes = 10 if train else 4            # x, y, x', h; then x, y, dx', dh, dx, dy
        return {"bytes": float(passes * n * d * size + (3 if train else 1) * params),
                "flops": float((40 if train else 12) * n * d)}
    v = case["vocab"]
    lists = 8 * n if case["kind"] == "ce" else 12 * n * min(case["k"], v)
    return {"bytes": float((2 if train else 1) * (n * d + v * d) * size + lists + 4 * n),
            "flops": float((6 if train else 2) * n * v * d)}


# ---- the definitions in 64 bits -----------------------------------------------------------------

def _double(t):
    return None if t is None else t.detach().double().requires_grad_(True)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "norm":
        v = {k: _double(state[k]) for k in ("x", "y", "pre", "post", "gate")}
        u = v["y"]
        if v["post"] is not None:
            u = u / (u.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * v["post"]
        if v["gate"] is not None:
            u = (u.view(case["gates"], -1, case["dim"]) * v["gate"][:, None]).view_as(u)
        x_new = case["scale"] * v["x"] + u
        h = x_new / (x_new.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * v["pre"]
        out = {"x": x_new.detach(), "h": h.detach()}
        if case["mode"] == "train":
            names = [k for k in v if v[k] is not None]
            grads = torch.autograd.grad((x_new, h), [v[k] for k in names],
                                        (state["dx_new"].double(), state["dh"].double()))
            out.update({"d_" + k: g for k, g in zip(names, grads)})
        return out
    h, w = _double(state["hidden"]), _double(state["weight"])
    z = h @ w.t()
    if case["kind"] == "ce":
        target = state["target"]
        counted = target != -100
        logp = torch.log_softmax(z, 1)
        loss = -logp.gather(1, target.clamp(min=0)[:, None])[:, 0]
        if case["z_loss"]:
            loss = loss + case["z_loss"] * torch.logsumexp(z, 1) ** 2
        loss = loss.masked_fill(~counted, 0.0)
    else:
        t, ids = case["temperature"], state["ids"]
        logp = torch.log_softmax(z / t, 1).gather(1, ids.clamp(min=0))
        teacher = state["logits"].double() / t
        counted = (ids >= 0).any(1)
        if state["teacher_lse"] is None:
            teacher = torch.where(ids >= 0, teacher, -1e300)
            logq = torch.log_softmax(teacher, 1)
        else:
            logq = teacher - state["teacher_lse"].double()[:, None]
        each = logq.exp() * (logq - logp)
        loss = t * t * each.masked_fill(ids < 0, 0.0).sum(1)
    if case["mode"] == "score":
        return {"loss": loss.detach()}
    loss = loss.sum() / counted.sum().clamp(min=1)
    dh, dw = torch.autograd.grad(loss, (h, w))
    return {"loss": loss.detach(), "d_hidden": dh, "d_weight": dw}
