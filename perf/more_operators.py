"""The operators of a block's attention and of the model's first layer as cases that can be timed and
checked one by one: ``attention``, the norms and rotation of its heads (``rotary_heads``) and the
token lookup (``embedding``), each with its gradient.

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
        # one sequence's next token under the benchmark model's heads, a short cache
        dict(name="attn_one_token", kind="attn", layout="cache", mode="score", dtype="bf16", batch=1,
             sq=1, sk=1024, heads=32, kv_heads=8, dim=128, causal=True, window=0),
        # the next token of a batch of sequences in a cache that holds 8192 positions of each
        dict(name="attn_decode", kind="attn", layout="cache", mode="score", dtype="bf16", batch=48,
             sq=1, sk=8192, heads=32, kv_heads=8, dim=128, causal=True, window=0),
        # a piece of a long prompt over what the cache holds already
        dict(name="attn_prompt", kind="attn", layout="cache", mode="score", dtype="bf16", batch=1,
             sq=2047, sk=32768, heads=32, kv_heads=8, dim=128, causal=True, window=0),
        # a unit-test sized encoder with odd lengths
        dict(name="attn_small_odd", kind="attn", layout="dense", mode="train", dtype="fp16", batch=2,
             sq=197, sk=197, heads=6, kv_heads=2, dim=72, causal=False, window=0),
        # documents of all lengths packed into one micro-batch
        dict(name="attn_packed", kind="attn", layout="packed", mode="train", dtype="bf16", batch=23,
             sq=16384, sk=16384, heads=32, kv_heads=8, dim=128, causal=True, window=0),
        # a smaller model with local attention, one position short of a tile
        dict(name="attn_window", kind="attn", layout="dense", mode="train", dtype="fp16", batch=1,
             sq=8191, sk=8191, heads=16, kv_heads=16, dim=64, causal=True, window=1024),
        # the attention of one training step of the benchmark model
        dict(name="attn_training", kind="attn", layout="dense", mode="train", dtype="bf16", batch=2,
             sq=8192, sk=8192, heads=32, kv_heads=8, dim=128, causal=True, window=0),
        # one token far into a text
        dict(name="heads_one_token", kind="heads", mode="score", dtype="bf16", tokens=1, heads=32,
             kv_heads=8, dim=128, rotary=128, norm=True, interleaved=False, far=100000),
        # half of each head rotated, pairs side by side, positions of no special kind
        dict(name="heads_odd", kind="heads", mode="train", dtype="fp32", tokens=1777, heads=5,
             kv_heads=1, dim=72, rotary=36, norm=True, interleaved=True, far=1000000),
        # the heads of one training step of the benchmark model
        dict(name="heads_training", kind="heads", mode="train", dtype="bf16", tokens=16384, heads=32,
             kv_heads=8, dim=128, rotary=128, norm=True, interleaved=False, far=0),
        # a small model's lookup, rows that are no multiple of a vector, padded
        dict(name="embed_odd", kind="embed", mode="train", dtype="fp16", tokens=1023, vocab=5003,
             dim=300, scale=17.5, padding=True),
        # the first layer of one training step of the benchmark model
        dict(name="embed_training", kind="embed", mode="train", dtype="bf16", tokens=16384,
             vocab=128256, dim=4096, scale=1.0, padding=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn", "heads", "embed"))
    mode = rng.choice(("train", "train", "score"))
    if kind == "embed":
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        dim = _log_int(rng, 64, 4096 if dtype != "fp32" else 2048)
        if rng.random() < 0.7:                 # most models' widths are whole vectors
            dim = -(-dim // 8) * 8
        return dict(kind=kind, mode=mode, dtype=dtype, tokens=_log_int(rng, 1, 16384),
                    vocab=_log_int(rng, 1000, 128256), dim=dim,
                    scale=rng.choice((1.0, 1.0, 32.0)), padding=rng.random() < 0.3)
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4))
    dim = rng.choice((64, 128, 128, 8 * rng.randint(4, 16)))
    if kind == "heads":
        return dict(kind=kind, mode=mode, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")),
                    tokens=_log_int(rng, 1, 16384), heads=heads, kv_heads=kv_heads, dim=dim,
                    rotary=rng.choice((dim, dim, dim // 2)), norm=rng.random() < 0.7,
                    interleaved=rng.random() < 0.3, far=rng.choice((0, 0, 1000000)))
    case = dict(kind=kind, mode=mode, dtype=rng.choice(("bf16", "bf16", "fp16")), heads=heads,
                kv_heads=kv_heads, dim=dim)
    layout = rng.choice(("dense", "packed", "cache"))
    if layout == "cache":                      # tokens after what a cache holds
        sq = rng.choice((1, 1, _log_int(rng, 2, 1024)))
        case.update(mode="score", batch=_log_int(rng, 1, 48 if sq == 1 else 4), sq=sq,
                    sk=_log_int(rng, max(sq, 64), 8192 if sq == 1 else 16384), causal=True)
    elif layout == "packed":
        n = _log_int(rng, 64, 16384)
        case.update(batch=rng.randint(4, 24), sq=n, sk=n, causal=rng.random() < 0.8)
    else:
        n = _log_int(rng, 16, 8192)
        other = n if rng.random() < 0.7 else _log_int(rng, 16, 8192)
        causal = n <= other and rng.random() < 0.8
        case.update(batch=rng.randint(1, 2) if causal else 1, sq=n, sk=other, causal=causal)
    case.update(layout=layout,
                window=_log_int(rng, 16, 4096) if case["causal"] and rng.random() < 0.25 else 0)
    return case


# ---- inputs -----------------------------------------------------------------------------------

def _randn(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _inv_freq(rotary):
    at = torch.arange(0, rotary, 2, device=DEV, dtype=torch.float64)
    return (500000.0 ** (-at / rotary)).float()


def _prepare_heads(case, gen, state):
    n, h, hk, d, dt = (case["tokens"], case["heads"], case["kv_heads"], case["dim"],
                       DTYPES[case["dtype"]])
    # queries and keys as they lie in the result of one product for q, k and v
    qkv = _randn(gen, n, (h + 2 * hk) * d).to(dt)
    state["q"] = qkv[:, :h * d].view(n, h, d).detach()
    state["k"] = qkv[:, h * d:(h + hk) * d].view(n, hk, d).detach()
    state["positions"] = torch.arange(n, device=DEV) + case["far"]
    state["inv_freq"] = _inv_freq(case["rotary"])
    for name in ("q_weight", "k_weight"):
        state[name] = 1 + 0.1 * _randn(gen, d) if case["norm"] else None
    if case["mode"] == "train":
        state["dq"] = (1e-2 * _randn(gen, n, h, d)).to(dt)
        state["dk"] = (1e-2 * _randn(gen, n, hk, d)).to(dt)
        for name in ("q", "k", "q_weight", "k_weight"):
            if state[name] is not None:
                state[name].requires_grad_(True)


def _prepare_embed(case, gen, state):
    n, v, dt = case["tokens"], case["vocab"], DTYPES[case["dtype"]]
    # a text's tokens: a few classes often, most hardly ever
    rank = torch.exp(torch.rand(n, device=DEV, generator=gen) * math.log(v)).long() - 1
    tokens = (rank.clamp(max=v - 1) * 7919 + 5) % v
    if case["padding"]:
        tokens[torch.rand(n, device=DEV, generator=gen) < 0.2] = 0
    state["tokens"] = tokens
    state["weight"] = _randn(gen, v, case["dim"]).mul_(0.02).to(dt)
    if case["mode"] == "train":
        state["dy"] = (1e-2 * _randn(gen, n, case["dim"])).to(dt)
        state["weight"].requires_grad_(True)


def _prepare_attn(case, gen, state):
    h, hk, d, dt, b = (case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]],
                       case["batch"])
    sq, sk = case["sq"], case["sk"]
    lead = () if case["layout"] == "packed" else (b,)
    # normed and rotated queries and keys
    state["q"] = (1.5 * _randn(gen, *lead, sq, h, d)).to(dt)
    state["k"] = _randn(gen, *lead, sk, hk, d).to(dt)
    state["v"] = _randn(gen, *lead, sk, hk, d).to(dt)
    state["kv_lengths"] = state["starts"] = None
    if case["layout"] == "cache":
        low = max(sq, sk // 4)
        lengths = torch.randint(low, sk + 1, (b,), device=DEV, generator=gen)
        lengths[0] = sk
        state["kv_lengths"] = lengths
    elif case["layout"] == "packed":
        cuts = torch.randint(0, sq + 1, (b - 1,), device=DEV, generator=gen).sort().values
        ends = torch.tensor([sq], device=DEV)
        state["starts"] = torch.cat([torch.zeros_like(ends), cuts, ends])
        # the loader that packed them has the lengths on the host too
        state["bounds"] = state["starts"].tolist()
    if case["mode"] == "train":
        state["dout"] = (1e-2 * _randn(gen, *lead, sq, h, d)).to(dt)
        for name in ("q", "k", "v"):
            state[name].requires_grad_(True)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    state = dict(case=case)
    {"attn": _prepare_attn, "heads": _prepare_heads, "embed": _prepare_embed}[case["kind"]](
        case, gen, state)
    return state


# ---- one pass ---------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["kind"]](state, case)


def _own_attn(state, case):
    import dmuon_amd as dmuon

    def call():
        return dmuon.attention(state["q"], state["k"], state["v"], causal=case["causal"],
                               window=case["window"] or None, kv_lengths=state["kv_lengths"],
                               q_starts=state["starts"], kv_starts=state["starts"])
    if case["mode"] == "score":
        with torch.no_grad():
            return {"out": call()}
    out = call()
    dq, dk, dv = torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


def _own_heads(state, case):
    import dmuon_amd as dmuon

    def call():
        return dmuon.rotary_heads(state["q"], state["k"], state["positions"], state["inv_freq"],
                                  q_weight=state["q_weight"], k_weight=state["k_weight"], eps=EPS,
                                  interleaved=case["interleaved"])
    if case["mode"] == "score":
        with torch.no_grad():
            q, k = call()
        return {"q": q, "k": k}
    q, k = call()
    names = [n for n in ("q", "k", "q_weight", "k_weight") if state[n] is not None]
    grads = torch.autograd.grad((q, k), [state[n] for n in names], (state["dq"], state["dk"]))
    return {"q": q.detach(), "k": k.detach(), **{"d_" + n: g for n, g in zip(names, grads)}}


def _own_embed(state, case):
    import dmuon_amd as dmuon

    def call():
        return dmuon.embedding(state["tokens"], state["weight"], scale=case["scale"],
                               padding_idx=0 if case["padding"] else None)
    if case["mode"] == "score":
        with torch.no_grad():
            return {"y": call()}
    y = call()
    (dw,) = torch.autograd.grad(y, (state["weight"],), state["dy"])
    return {"y": y.detach(), "d_weight": dw}


def _fold(x, kv_heads):
    """[b, s, h, d] -> [b, kv_heads, s * h / kv_heads, d] in 32 bits, a key head's queries together."""
    b, s, h, d = x.shape
    x = x.float().view(b, s, kv_heads, h // kv_heads, d).permute(0, 2, 1, 3, 4)
    return x.reshape(b, kv_heads, s * (h // kv_heads), d)


def _unfold(x, heads, dtype):
    b, kv_heads, rows, d = x.shape
    g = heads // kv_heads
    x = x.view(b, kv_heads, rows // g, g, d).permute(0, 2, 1, 3, 4)
    return x.reshape(b, rows // g, heads, d).to(dtype)


def _plain_dense(case, q, k, v, lengths, dout):
    """Attention of a batch of rectangles; key lengths [b] or None."""
    (b, sq, h, d), sk, hk, dt = q.shape, k.shape[1], case["kv_heads"], q.dtype
    group = h // hk
    qf, kf, vf = _fold(q, hk), _fold(k, hk), _fold(v, hk)
    last = torch.full((b, 1, 1), sk, device=DEV) if lengths is None else lengths.view(b, 1, 1)
    j = torch.arange(sk, device=DEV)
    seen = (j < last).expand(b, sq, sk)
    if case["causal"]:
        at = torch.arange(sq, device=DEV).view(1, sq, 1) + last - sq
        seen = seen & (j <= at)
        if case["window"]:
            seen = seen & (j > at - case["window"])
    hidden = ~seen.repeat_interleave(group, 1)[:, None]
    scale = d ** -0.5
    p = (qf @ kf.transpose(2, 3).contiguous()).mul_(scale).masked_fill_(hidden, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top.isinf(), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total > 0, total, 1.0))
    out = [_unfold(p @ vf, h, dt)]
    if dout is not None:
        do = _fold(dout, hk)
        dv = p.transpose(2, 3) @ do
        dp = do @ vf.transpose(2, 3).contiguous()
        dp.sub_((p * dp).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out += [_unfold(dp @ kf, h, dt), _unfold(dp.transpose(2, 3) @ qf, hk, dt),
                _unfold(dv, hk, dt)]
    return out


@torch.no_grad()
def _plain_attn(state, case):
    q, k, v, dout = state["q"], state["k"], state["v"], state.get("dout")
    parts = []
    if case["layout"] == "packed":
        for lo, hi in zip(state["bounds"], state["bounds"][1:]):
            if hi > lo:
                cut = [t if t is None else t[None, lo:hi] for t in (q, k, v, dout)]
                parts.append([t[0] for t in _plain_dense(case, *cut[:3], None, cut[3])])
    else:
        # as many sequences at a time as keep the scores within 8 GiB
        step = max(1, 2 ** 31 // (case["heads"] * case["sq"] * case["sk"]))
        for at in range(0, case["batch"], step):
            cut = [t if t is None else t[at:at + step]
                   for t in (q, k, v, state["kv_lengths"], dout)]
            parts.append(_plain_dense(case, *cut))
    outs = [torch.cat(x) if len(x) > 1 else x[0] for x in zip(*parts)]
    return dict(zip(("out", "dq", "dk", "dv"), outs))


def _turn(x, cos, sin, rotary, interleaved):
    """The first ``rotary`` values of each head rotated; ``sin`` negated turns back."""
    r, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
    else:
        a, b = r[..., :rotary // 2], r[..., rotary // 2:]
    pair = (a * cos - b * sin, b * cos + a * sin)
    r = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat((r, rest), -1)


@torch.no_grad()
def _plain_heads(state, case):
    # angles of far positions in 64 bits
    angle = state["positions"].double()[:, None, None] * state["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    out = {}
    for name in ("q", "k"):
        x, w = state[name].float(), state[name + "_weight"]
        z = x
        if w is not None:
            r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
            x_hat = x * r
            z = x_hat * w
        out[name] = _turn(z, cos, sin, case["rotary"], case["interleaved"]).to(state[name].dtype)
        if case["mode"] == "train":
            g = _turn(state["d" + name].float(), cos, -sin, case["rotary"], case["interleaved"])
            if w is not None:
                out["d_" + name + "_weight"] = (g * x_hat).sum((0, 1))
                g = g * w
                g = r * (g - x_hat * (g * x_hat).mean(-1, keepdim=True))
            out["d_" + name] = g.to(state[name].dtype)
    return out


@torch.no_grad()
def _plain_embed(state, case):
    tokens, w, s = state["tokens"], state["weight"], case["scale"]
    out = {"y": (w[tokens].float() * s).to(w.dtype)}
    if case["mode"] == "train":
        dy = state["dy"].float() * s
        if case["padding"]:
            dy = dy * (tokens != 0)[:, None]
        dw = torch.zeros(w.shape, device=DEV)
        out["d_weight"] = dw.index_add_(0, tokens, dy).to(w.dtype)
    return out


_plain = {"attn": _plain_attn, "heads": _plain_heads, "embed": _plain_embed}
_own = {"attn": _own_attn, "heads": _own_heads, "embed": _own_embed}


# ---- what a pass cannot do without --------------------------------------------------------------

def _pairs(case):
    """Query and key positions that see each other, of all sequences; key positions held. A cache's
    and a packing's lengths, which the seed gives, stand at their expected sizes."""
    b, sq, sk, w = case["batch"], case["sq"], case["sk"], case["window"]
    if case["layout"] == "packed":
        # b pieces of a broken stick: E[length^2] = 2 n^2 / (b (b + 1))
        square = 2.0 * sq * sq / (b + 1)
        if not case["causal"]:
            return square, sk
        return min(0.5 * (square + sq), float(w) * sq if w else math.inf), sk
    held = float(sk)
    if case["layout"] == "cache" and b > 1:
        held = (sk + (b - 1) * 0.5 * (max(sq, sk // 4) + sk)) / b
    if not case["causal"]:
        return float(b) * sq * held, b * held
    pairs = 0.0
    for i in range(sq):
        seen = held - sq + i + 1
        pairs += max(0.0, min(seen, w) if w else seen)
    if w:
        held = min(held, float(w + sq - 1))
    return b * pairs, b * held


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    train = case["mode"] == "train"
    if case["kind"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        return {"bytes": float(size * d * (3 * n + v if train else 2 * n) + 8 * n),
                "flops": float((2 if train else 1) * n * d)}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "heads":
        values = case["tokens"] * (h + hk) * d
        return {"bytes": float((4 if train else 2) * values * size + 8 * case["tokens"]),
                "flops": float((24 if train else 8) * values)}
    pairs, held = _pairs(case)
    rows = case["sq"] * (1 if case["layout"] == "packed" else case["batch"])
    # q, k, v -> out; with do -> dq, dk, dv
    values = rows * h * d * (4 if train else 2) + held * hk * d * (4 if train else 2)
    return {"bytes": float(values * size), "flops": float((14 if train else 4) * pairs * h * d)}


# ---- the definitions in 64 bits -----------------------------------------------------------------

def _double(t):
    return None if t is None else t.detach().double().requires_grad_(True)


def _exact_sequence(case, q, k, v, dout):
    """One sequence, [s, h, d] each, query head by query head."""
    sq, sk, group = q.shape[0], k.shape[0], case["heads"] // case["kv_heads"]
    behind = (torch.arange(sq, device=DEV) + (sk - sq))[:, None] - torch.arange(sk, device=DEV)
    visible = torch.ones_like(behind, dtype=torch.bool)
    if case["causal"]:
        visible = behind >= 0
        if case["window"]:
            visible &= behind < case["window"]
    some = visible.any(1, keepdim=True)
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    grads = None
    if dout is not None:
        grads = [torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in (q, k, v)]
    for head in range(case["heads"]):
        at = head // group
        leaf = [_double(q[:, head]), _double(k[:, at]), _double(v[:, at])]
        with torch.set_grad_enabled(dout is not None):
            logits = leaf[0] @ leaf[1].t() / math.sqrt(case["dim"])
            # a row that sees nothing is 0
            probs = torch.softmax(torch.where(visible | ~some, logits, -1e300), -1)
            o = torch.where(some, probs @ leaf[2], 0.0)
            del logits, probs
        out[:, head] = o.detach()
        if dout is not None:
            for total, where, g in zip(grads, (head, at, at), torch.autograd.grad(
                    o, leaf, dout[:, head].double())):
                total[:, where] += g
    return [out] + (grads or [])


def _exact_attn(case, state):
    q, k, v, dout = state["q"], state["k"], state["v"], state.get("dout")
    total = [torch.zeros(t.shape, dtype=torch.float64, device=DEV)
             for t in ((q, q, k, v) if dout is not None else (q,))]
    sequences = []
    if case["layout"] == "packed":
        sequences = [(slice(lo, hi), slice(lo, hi))
                     for lo, hi in zip(state["bounds"], state["bounds"][1:]) if hi > lo]
    elif case["layout"] == "cache":
        sequences = [(b, (b, slice(0, n))) for b, n in enumerate(state["kv_lengths"].tolist())]
    else:
        sequences = [(b, b) for b in range(case["batch"])]
    for mine, theirs in sequences:
        parts = _exact_sequence(case, q[mine], k[theirs], v[theirs],
                                None if dout is None else dout[mine])
        for t, where, part in zip(total, (mine, mine, theirs, theirs), parts):
            t[where] = part
    return dict(zip(("out", "dq", "dk", "dv"), total))


def _exact_heads(case, state):
    angle = state["positions"].double()[:, None] * state["inv_freq"].double()
    unit = torch.polar(torch.ones_like(angle), angle)[:, None]
    out, r = {}, case["rotary"]
    for name in ("q", "k"):
        x, w = _double(state[name]), _double(state[name + "_weight"])
        z = x
        if w is not None:
            z = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w
        turned = z[..., :r]
        if case["interleaved"]:
            turned = torch.view_as_real(torch.complex(turned[..., 0::2], turned[..., 1::2])
                                        * unit).flatten(-2)
        else:
            turned = torch.complex(turned[..., :r // 2], turned[..., r // 2:]) * unit
            turned = torch.cat((turned.real, turned.imag), -1)
        y = torch.cat((turned, z[..., r:]), -1)
        out[name] = y.detach()
        if case["mode"] == "train":
            leaves = [x] if w is None else [x, w]
            grads = torch.autograd.grad(y, leaves, state["d" + name].double())
            out["d_" + name] = grads[0]
            if w is not None:
                out["d_" + name + "_weight"] = grads[1]
    return out


def _exact_embed(case, state):
    tokens, w = state["tokens"], state["weight"].detach().double()
    out = {"y": case["scale"] * w.index_select(0, tokens)}
    if case["mode"] == "train":
        kept = tokens if not case["padding"] else tokens[tokens != 0]
        dy = state["dy"] if not case["padding"] else state["dy"][tokens != 0]
        out["d_weight"] = torch.zeros_like(w).index_add_(0, kept, case["scale"] * dy.double())
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"attn": _exact_attn, "heads": _exact_heads, "embed": _exact_embed}[case["kind"]](
        case, state)
