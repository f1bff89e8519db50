"""The operators of a block in a row, as a model calls them: token lookup, a product for queries, keys and
values, the heads' norms and rotation, attention, a product, the norms around it and the loss.

Every operator is checked by itself against its definition, and gives the same bits for the same call; so
the chain's gradients must be, bit for bit, those of the single calls, each fed with what the one behind it
gave. And the chain's loss must follow its gradient, as differences of a definition in 64 bits show.
"""
import pytest
import torch

import dmuon_amd as dmuon

HEADS, KV_HEADS, DIM, WIDTH, VOCAB = 4, 2, 32, 128, 211


def _model(dev, dt=torch.bfloat16, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*s, scale=1.0):
        return (scale * torch.randn(*s, device=dev, generator=gen)).to(dt)
    w = {"embed": randn(VOCAB, WIDTH), "qkv": randn((HEADS + 2 * KV_HEADS) * DIM, WIDTH, scale=WIDTH ** -0.5),
         "out": randn(WIDTH, HEADS * DIM, scale=WIDTH ** -0.5), "head": randn(VOCAB, WIDTH, scale=WIDTH ** -0.5)}
    for k, n in (("pre0", WIDTH), ("pre1", WIDTH), ("q_norm", DIM), ("k_norm", DIM)):
        w[k] = 1 + 0.1 * torch.randn(n, device=dev, generator=gen)
    return w


def _data(dev, seed=1):
    gen = torch.Generator(device=dev).manual_seed(seed)
    tokens = torch.randint(0, VOCAB, (2, 150), device=dev, generator=gen)
    target = torch.randint(0, VOCAB, (2, 150), device=dev, generator=gen)
    return tokens, target, torch.arange(150, device=dev), \
        (10000.0 ** (-torch.arange(0, 1, 2 / DIM))).to(dev)


def _chain(w, tokens, target, positions, inv_freq, keep=None):
    """The loss; ``keep`` takes every operator's operands and results."""
    def seen(name, ins, outs):
        if keep is not None:
            for t in outs:
                t.retain_grad()
            keep.append((name, ins, outs))
        return outs
    (e,) = seen("embedding", (tokens, w["embed"]), (dmuon.embedding(tokens, w["embed"], scale=2.0),))
    x, h = dmuon.residual_norm(e, None, w["pre0"])
    heads = (h @ w["qkv"].t()).unflatten(-1, (-1, DIM))
    q, k, v = heads.split([HEADS, KV_HEADS, KV_HEADS], -2)
    qr, kr = seen("rotary", (q, k), dmuon.rotary_heads(q, k, positions, inv_freq, q_weight=w["q_norm"],
                                                       k_weight=w["k_norm"]))
    (o,) = seen("attention", (qr, kr, v), (dmuon.attention(qr, kr, v),))
    x, h = dmuon.residual_norm(x, o.flatten(-2) @ w["out"].t(), w["pre1"])
    return dmuon.linear_cross_entropy(h, w["head"], target)


@pytest.mark.gpu
def test_the_chains_gradients_are_the_operators(gpu):
    w = {k: t.requires_grad_(True) for k, t in _model(gpu).items()}
    data, keep = _data(gpu), []
    _chain(w, *data, keep=keep).backward()
    for name, ins, outs in keep:
        leaves = [t.detach().requires_grad_(t.is_floating_point()) for t in ins]
        if name == "embedding":
            again, extra = (dmuon.embedding(*leaves, scale=2.0),), {}
            extra = {"embed": leaves[1]}
        elif name == "rotary":
            norms = [w[k].detach().requires_grad_(True) for k in ("q_norm", "k_norm")]
            again = dmuon.rotary_heads(*leaves, *data[2:], q_weight=norms[0], k_weight=norms[1])
            extra = dict(zip(("q_norm", "k_norm"), norms))
        else:
            again, extra = (dmuon.attention(*leaves),), {}
        assert all(torch.equal(a, b) for a, b in zip(again, outs))
        torch.autograd.backward(again, [t.grad for t in outs])
        for k, leaf in extra.items():
            assert torch.equal(w[k].grad, leaf.grad), (name, k)
        if name == "attention":
            # its gradients are what the rotation was given
            assert torch.equal(keep[1][2][0].grad, leaves[0].grad)
            assert torch.equal(keep[1][2][1].grad, leaves[1].grad)


def _exact_loss(w, tokens, target, positions, inv_freq):
    def norm(x, weight):
        return x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight
    e = 2 * w["embed"][tokens]
    heads = (norm(e, w["pre0"]) @ w["qkv"].t()).unflatten(-1, (-1, DIM))
    q, k, v = heads.split([HEADS, KV_HEADS, KV_HEADS], -2)
    angle = positions.double()[:, None, None] * inv_freq.double()

    def turn(x):
        z = torch.complex(x[..., :DIM // 2], x[..., DIM // 2:]) * torch.polar(torch.ones_like(angle), angle)
        return torch.cat((z.real, z.imag), -1)
    q, k = turn(norm(q, w["q_norm"])), turn(norm(k, w["k_norm"]))
    k, v = (t.repeat_interleave(HEADS // KV_HEADS, 2).transpose(1, 2) for t in (k, v))
    s = q.transpose(1, 2) @ k.transpose(2, 3) / DIM ** 0.5
    s = s.masked_fill(torch.ones_like(s[0, 0]).triu(1).bool(), float("-inf"))
    o = (s.softmax(-1) @ v).transpose(1, 2).flatten(-2)
    logits = norm(e + o @ w["out"].t(), w["pre1"]) @ w["head"].t()
    return torch.nn.functional.cross_entropy(logits.flatten(0, 1), target.flatten())


@pytest.mark.gpu
def test_the_chains_loss_follows_its_gradient(gpu):
    """Some ten roundings of 2^-8 on the way back, of independent signs over hundreds of values: the slope
    along the whole gradient is off by far less than 10 * 2^-8."""
    w = {k: t.requires_grad_(True) for k, t in _model(gpu, seed=2).items()}
    data = _data(gpu, 3)
    _chain(w, *data).backward()
    size = sum(float(t.grad.double().pow(2).sum()) for t in w.values()) ** 0.5
    step = {k: t.grad.double() / size for k, t in w.items()}

    def value(eps):
        with torch.no_grad():
            return float(_exact_loss({k: t.detach().double() + eps * step[k] for k, t in w.items()}, *data))
    slope = (value(1e-4) - value(-1e-4)) / 2e-4
    assert abs(slope - size) <= 10 * 2.0 ** -8 * size


@pytest.mark.gpu
def test_the_chain_in_a_graph(gpu):
    """Forward and backward captured together, replayed with other tokens and weights between eager steps."""
    w = {k: t.requires_grad_(True) for k, t in _model(gpu, seed=4).items()}
    data = _data(gpu, 5)

    def step():
        loss = _chain(w, *data)
        return [loss.detach()] + list(torch.autograd.grad(loss, list(w.values())))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        data[0].copy_(_data(gpu, 10 + seed)[0])
        data[1].copy_(_data(gpu, 10 + seed)[1])
        with torch.no_grad():
            for k, t in _model(gpu, seed=20 + seed).items():
                w[k].copy_(t)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))
