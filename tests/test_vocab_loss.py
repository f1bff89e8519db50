"""``linear_cross_entropy`` and ``linear_distillation`` against their definitions in 64 bits.

Bounds. Products accumulate in fp32: a logit of ``dim`` products is off by at most
``dim * 2^-24 * sum|h w|`` in the worst order; the kernels' blocked order and random signs leave a
fraction of its square root, and the tests allow ``2^-24 * (8 + sqrt(dim)) * sum|h w|``
(``z_err``). A loss is off by two logits plus a few ulp of its own size and of the row's largest
logit. A gradient ``dZ`` between the products is rounded to the operands' type (relative ``u`` =
2^-8 for bf16, 2^-11 for fp16, absolute 2^-34 of the largest row weight for fp16, which is stored
shifted by 2^10) after a relative error of 2^-11 at most in the probabilities; the result is
rounded once more. So an element of ``dH = dZ W`` is off by at most
``(u + 2^-11 + 3 z_err) (|dZ| |W|) + u |dH|`` and accordingly for ``dW``.
"""
import math

import pytest
import torch

import dmuon_amd as dmuon

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}          # half the smallest fp16 step


def _inputs(dev, n, v, d, dt, seed=0, lean=8.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    w = torch.randn(v, d, device=dev, generator=gen) / math.sqrt(d)
    t = torch.randint(0, v, (n,), device=dev, generator=gen)
    h = torch.randn(n, d, device=dev, generator=gen)
    h = h + lean * torch.rand(n, 1, device=dev, generator=gen) * w[t] if n else h
    return h.to(dt), w.to(dt), t, gen


class _Exact:
    """Row losses, logit gradients and their bounds from dense target probabilities q [n, v]."""

    def __init__(self, h, w, q, counted, temperature=1.0, z_loss=0.0, entropy=None):
        self.h, self.w, self.dt = h.double(), w.double(), h.dtype
        d = h.shape[1]
        z = self.h @ self.w.t() / temperature
        scale = self.h.abs() @ self.w.abs().t() / temperature
        self.z_err = 2.0 ** -24 * (8 + math.sqrt(d)) * (scale.amax() if scale.numel() else 0.0)
        lse = torch.logsumexp(z, 1)
        mass = q.sum(1)
        ent = torch.where(q > 0, q * q.log(), 0.0).sum(1) if entropy is None else entropy
        self.loss = temperature ** 2 * (ent + mass * lse - torch.where(q > 0, q * z, 0.0).sum(1))
        self.loss = self.loss + z_loss * lse ** 2
        self.loss = torch.where(counted, self.loss, 0.0)
        top = z.abs().amax() if z.numel() else 0.0
        self.loss_tol = temperature ** 2 * (1 + 2 * z_loss * top) * (
            2 * self.z_err + 2.0 ** -20 * (1 + top))
        p = (z - lse[:, None]).exp()
        self.dz = temperature * ((mass + 2 * z_loss * lse)[:, None] * p - q)
        self.dz = torch.where(counted[:, None], self.dz, 0.0)
        self.p = temperature * p
        self.counted = counted

    def grads(self, row):
        """((d_hidden, bound), (d_weight, bound)) for the row gradients ``row``."""
        row = torch.where(self.counted, row.double(), 0.0)
        dz = row[:, None] * self.dz
        u, rel = U[self.dt], 2.0 ** -11 + 3 * self.z_err
        # probabilities are off relatively, their difference from a target absolutely
        slack = u * dz.abs() + rel * row.abs()[:, None] * torch.maximum(self.p, self.dz.abs())
        if self.dt == torch.float16 and row.numel():
            slack = slack + 2.0 ** -34 * row.abs().amax()
        out = []
        for g, b in ((dz @ self.w, slack @ self.w.abs()), (dz.t() @ self.h, slack.t() @ self.h.abs())):
            out.append((g, b + u * g.abs() + TINY[self.dt] + 1e-30))
        return out


def _ce(h, w, t, ignore=-100, z_loss=0.0):
    counted = t != ignore
    q = torch.zeros(h.shape[0], w.shape[0], dtype=torch.float64, device=h.device)
    if h.shape[0]:
        q.scatter_(1, t.clamp(min=0)[:, None], counted.double()[:, None])
    return _Exact(h, w, q, counted, z_loss=z_loss)


def _kd(h, w, ids, logits, lse=None, temperature=1.0):
    live = ids >= 0
    soft = torch.where(live, logits.double() / temperature, float("-inf"))
    if lse is None:
        probs = torch.softmax(soft, 1).nan_to_num(0.0)
    else:
        probs = (soft - lse.double()[:, None]).exp()
    q = torch.zeros(h.shape[0], w.shape[0], dtype=torch.float64, device=h.device)
    q.scatter_add_(1, ids.clamp(min=0), torch.where(live, probs, 0.0))
    entropy = torch.where(probs > 0, probs * probs.log(), 0.0).sum(1)
    return _Exact(h, w, q, live.any(1), temperature, entropy=entropy)


def _within(got, want, bound):
    assert bool(((got.double() - want).abs() <= bound).all()), \
        float(((got.double() - want).abs() / bound).max())


def _check(exact, call, h, w, reduction):
    """Loss and gradients of ``call(hidden, weight, reduction)`` against ``exact``."""
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = call(h, w, reduction)
    assert loss.dtype == torch.float32
    count = max(int(exact.counted.sum()), 1)
    n = exact.loss.shape[0]
    if reduction == "none":
        _within(loss, exact.loss, exact.loss_tol)
        row = torch.linspace(-1.0, 2.0, n, device=h.device) if n else loss.detach()
        loss.backward(row)
    else:
        div = count if reduction == "mean" else 1
        _within(loss, exact.loss.sum() / div, exact.loss_tol * n / div + 1e-30)
        loss.backward()
        row = torch.full((n,), 1.0 / div, device=h.device)
    (dh, bh), (dw, bw) = exact.grads(row)
    assert h.grad.dtype == h.dtype and w.grad.dtype == w.dtype
    _within(h.grad, dh, bh)
    _within(w.grad, dw, bw)


SIZES = [  # tokens, vocabulary, dim: single ones, tile edges on both sides, odd pitches
    (1, 1, 1), (1, 1000, 64), (2, 63, 8), (3, 65, 100), (63, 257, 72), (64, 256, 64),
    (65, 1003, 300), (255, 511, 129), (256, 512, 256), (257, 2049, 320), (513, 700, 1001),
    (5, 5000, 2048), (1100, 129, 96),
    # both sides of the sizes at which a call takes other kernels: rows of one tile and few rows,
    # tokens of a short weight gradient, split sums
    (16, 3000, 520), (17, 3000, 520), (192, 1500, 264), (193, 1500, 264), (512, 1000, 72),
    (520, 1000, 72), (30, 20000, 256), (300, 12000, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,v,d", SIZES)
def test_cross_entropy_sizes(gpu, n, v, d, dt):
    h, w, t, gen = _inputs(gpu, n, v, d, dt)
    t = torch.where(torch.rand(n, device=gpu, generator=gen) < 0.2, -100, t)
    _check(_ce(h, w, t), lambda a, b, r: dmuon.linear_cross_entropy(a, b, t, reduction=r), h, w,
           "mean")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("z_loss,ignore", [(0.0, -100), (1e-2, 7)])
def test_cross_entropy_options(gpu, reduction, z_loss, ignore, dt):
    h, w, t, _ = _inputs(gpu, 300, 777, 136, dt, seed=3)
    t[::5] = ignore
    _check(_ce(h, w, t, ignore, z_loss),
           lambda a, b, r: dmuon.linear_cross_entropy(a, b, t, ignore_index=ignore, z_loss=z_loss,
                                                      reduction=r), h, w, reduction)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,v,d", SIZES)
@pytest.mark.parametrize("k,temperature,full", [(1, 1.0, False), (5, 2.0, True), (70, 0.7, False)])
def test_distillation(gpu, n, v, d, k, temperature, full, dt):
    h, w, t, gen = _inputs(gpu, n, v, d, dt, seed=1)
    k = min(k, v)
    ids = torch.rand(n, v, device=gpu, generator=gen).argsort(1)[:, :k]
    logits = 4 * torch.randn(n, k, device=gpu, generator=gen)
    ids = torch.where(torch.rand(n, k, device=gpu, generator=gen) < 0.2, -1, ids)
    ids[n // 2] = -1                                       # a token without a teacher
    logits[n // 3, 0] = float("-inf")                      # a class of no weight
    lse = torch.logsumexp(logits / temperature, 1) + 0.1 if full else None
    if full:
        lse = torch.where(lse.isfinite(), lse, 0.0)
    _check(_kd(h, w, ids, logits, lse, temperature),
           lambda a, b, r: dmuon.linear_distillation(a, b, ids, logits, teacher_lse=lse,
                                                     temperature=temperature, reduction=r),
           h, w, "mean")


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_distillation_reductions_and_repeated_classes(gpu, reduction):
    h, w, t, gen = _inputs(gpu, 90, 400, 64, torch.bfloat16, seed=2)
    ids = torch.randint(0, 40, (90, 33), device=gpu, generator=gen)     # classes occur twice
    logits = torch.randn(90, 33, device=gpu, generator=gen)
    _check(_kd(h, w, ids, logits), lambda a, b, r: dmuon.linear_distillation(
        a, b, ids, logits, reduction=r), h, w, reduction)


@pytest.mark.gpu
def test_a_teacher_of_lowest_values(gpu):
    """A list masked with the type's lowest value is uniform over what is left; one masked with
    -inf throughout has no weight, loss 0 and no gradient."""
    h, w, t, _ = _inputs(gpu, 4, 300, 64, torch.bfloat16)
    ids = torch.arange(8, device=gpu).expand(4, 8).contiguous()
    logits = torch.zeros(4, 8, device=gpu)
    logits[0, 1:] = torch.finfo(torch.float32).min
    logits[1] = torch.finfo(torch.float32).min
    logits[2] = float("-inf")
    exact = _kd(h, w, ids, torch.where(logits < -1e30, logits.clamp(min=-1e30), logits))
    a = h.clone().requires_grad_(True)
    loss = dmuon.linear_distillation(a, w, ids, logits, reduction="none")
    live = [0, 1, 3]
    _within(loss[live], exact.loss[live], exact.loss_tol)
    assert float(loss[2].detach()) == 0.0
    loss.sum().backward()
    assert not bool(a.grad[2].any()) and bool(a.grad[live].isfinite().all())


@pytest.mark.gpu
def test_no_counted_token_gives_zeros(gpu):
    h, w, t, _ = _inputs(gpu, 40, 130, 64, torch.bfloat16)
    for call in (lambda a, b: dmuon.linear_cross_entropy(a, b, torch.full_like(t, -100)),
                 lambda a, b: dmuon.linear_distillation(a, b, torch.full((40, 3), -1, device=gpu),
                                                        torch.zeros(40, 3, device=gpu))):
        a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = call(a, b)
        loss.backward()
        assert float(loss.detach()) == 0.0 and not bool(a.grad.any()) and not bool(b.grad.any())


@pytest.mark.gpu
def test_no_token_at_all(gpu):
    h, w, t, _ = _inputs(gpu, 0, 130, 64, torch.float16)
    a, b = h.requires_grad_(True), w.requires_grad_(True)
    loss = dmuon.linear_cross_entropy(a, b, t)
    loss.backward()
    assert float(loss.detach()) == 0.0 and a.grad.shape == (0, 64) and not bool(b.grad.any())
    rows = dmuon.linear_cross_entropy(a, b, t, reduction="none")
    b.grad = None
    rows.sum().backward()
    assert rows.shape == (0,) and not bool(b.grad.any())


@pytest.mark.gpu
def test_values_that_are_no_numbers(gpu):
    """A target outside the vocabulary, an infinity or a NaN in a token's state: its loss is not a
    number, the other tokens' losses stand. An ignored token's NaN state stays out of the weight's
    gradient only if its state is finite, so its loss alone is looked at."""
    h, w, t, _ = _inputs(gpu, 70, 500, 64, torch.bfloat16)
    want = _ce(h, w, t)
    bad_t = t.clone()
    bad_t[3], bad_t[4] = 500, -7
    loss = dmuon.linear_cross_entropy(h, w, bad_t, reduction="none")
    assert bool(loss[[3, 4]].isnan().all())
    keep = [i for i in range(70) if i not in (3, 4)]
    _within(loss[keep], want.loss[keep], want.loss_tol)
    ids = t[:, None].clone()
    ids[5] = 500
    loss = dmuon.linear_distillation(h, w, ids, torch.zeros(70, 1, device=gpu), reduction="none")
    assert bool(loss[5].isnan()) and bool(loss[[4, 6]].isfinite().all())
    bad_h = h.clone()
    bad_h[8, 0], bad_h[9, 0] = float("nan"), float("inf")
    loss = dmuon.linear_cross_entropy(bad_h, w, t, reduction="none")
    assert not bool(loss[[8, 9]].isfinite().any())
    keep = [i for i in range(70) if i not in (8, 9)]
    _within(loss[keep], want.loss[keep], want.loss_tol)


@pytest.mark.gpu
def test_confident_rows_keep_their_small_gradients(gpu):
    """Where the student is sure, softmax - 1 at the target cancels: 1 - p must come out right."""
    d, v, n = 64, 257, 32
    w = torch.zeros(v, d, device=gpu)
    w[:d] = torch.eye(d, device=gpu)
    t = torch.arange(n, device=gpu)
    h = 14.0 * torch.eye(d, device=gpu)[:n]
    for dt in U:
        _check(_ce(h.to(dt), w.to(dt), t),
               lambda a, b, r: dmuon.linear_cross_entropy(a, b, t, reduction=r), h.to(dt), w.to(dt),
               "sum")
        a = h.to(dt).requires_grad_(True)
        dmuon.linear_cross_entropy(a, w.to(dt), t, reduction="sum").backward()
        z = (h @ w.t()).double()
        p = torch.softmax(z, 1)
        at = a.grad[t, t].double()
        want = p[t, t] - 1
        assert bool(((at - want).abs() <= 4 * U[dt] * want.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("chunk", [1, 100, 256, 300, 1000])
def test_chunks_give_the_same_losses(gpu, chunk, dt):
    h, w, t, _ = _inputs(gpu, 700, 600, 128, dt, seed=5)
    whole = dmuon.linear_cross_entropy(h, w, t, reduction="none")
    part = dmuon.linear_cross_entropy(h, w, t, reduction="none", chunk_tokens=chunk)
    assert torch.equal(whole, part)
    if chunk > 1:
        _check(_ce(h, w, t), lambda a, b, r: dmuon.linear_cross_entropy(
            a, b, t, reduction=r, chunk_tokens=chunk), h, w, "mean")


@pytest.mark.gpu
def test_strides_leading_shapes_and_index_types(gpu):
    h, w, t, gen = _inputs(gpu, 60, 321, 72, torch.bfloat16, seed=6)
    want = dmuon.linear_cross_entropy(h, w, t, reduction="none")
    wide = torch.full((60, 75), float("nan"), dtype=h.dtype, device=gpu)
    wide[:, 2:74] = h                                     # rows of an odd pitch and base
    tall = torch.full((330, 81), float("nan"), dtype=w.dtype, device=gpu)
    tall[5:326, 1:73] = w
    hv, wv = wide[:, 2:74], tall[5:326, 1:73]
    assert torch.equal(dmuon.linear_cross_entropy(hv, wv, t, reduction="none"), want)
    got = dmuon.linear_cross_entropy(hv.unflatten(0, (3, 20)), wv, t.view(3, 20).int(),
                                     reduction="none")
    assert got.shape == (3, 20) and torch.equal(got.flatten(), want)
    # columns apart, rows repeated
    hc = h.t().contiguous().t()
    assert torch.equal(dmuon.linear_cross_entropy(hc, w, t, reduction="none"), want)
    one = dmuon.linear_cross_entropy(h[:1].expand(60, 72), w, t[:1].expand(60), reduction="none")
    assert torch.equal(one, want[:1].expand(60))
    # the gradients of strided operands
    a, b = wide.requires_grad_(True), tall.requires_grad_(True)
    dmuon.linear_cross_entropy(a[:, 2:74], b[5:326, 1:73], t).backward()
    (dh, bh), (dw, bw) = _ce(h, w, t).grads(torch.full((60,), 1 / 60, device=gpu))
    _within(a.grad[:, 2:74], dh, bh)
    _within(b.grad[5:326, 1:73], dw, bw)
    assert float(a.grad[:, :2].abs().sum()) == 0 and float(b.grad[:5].abs().sum()) == 0


@pytest.mark.gpu
def test_only_the_gradients_that_are_asked_for(gpu):
    h, w, t, _ = _inputs(gpu, 50, 300, 64, torch.bfloat16)
    both = [x.clone().requires_grad_(True) for x in (h, w)]
    dmuon.linear_cross_entropy(*both, t).backward()
    a = h.clone().requires_grad_(True)
    dmuon.linear_cross_entropy(a, w, t).backward()
    b = w.clone().requires_grad_(True)
    dmuon.linear_cross_entropy(h, b, t).backward()
    assert torch.equal(a.grad, both[0].grad) and torch.equal(b.grad, both[1].grad)
    assert not dmuon.linear_cross_entropy(h, w, t).requires_grad
    with torch.no_grad():
        assert not dmuon.linear_cross_entropy(*both, t).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_incoming_gradients_and_retained_graphs(gpu, dt):
    h, w, t, _ = _inputs(gpu, 80, 300, 64, dt, seed=8)
    a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = dmuon.linear_cross_entropy(a, b, t)
    one = torch.autograd.grad(loss, (a, b), retain_graph=True)
    again = torch.autograd.grad(loss, (a, b), retain_graph=True)       # formed anew
    assert all(torch.equal(x, y) for x, y in zip(one, again))
    # a power of two: the same bits, shifted (nothing here is subnormal in bf16)
    four = torch.autograd.grad(4.0 * loss, (a, b))
    if dt == torch.bfloat16:
        assert all(torch.equal(4 * x, y) for x, y in zip(one, four))
    # a loss scale: gradients that fp16 alone would lose
    loss = dmuon.linear_cross_entropy(a, b, t)
    big = torch.autograd.grad(loss * 1024.0, (a, b))
    for got, (want, bound) in zip(big, _ce(h, w, t).grads(torch.full((80,), 1024 / 80, device=gpu))):
        _within(got, want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["target", "ids", "logits", "lse", "hidden", "weight"])
def test_operands_that_change_before_the_gradient(gpu, what):
    """A gradient that forms the logits anew refuses operands that were written to meanwhile."""
    h, w, t, gen = _inputs(gpu, 20, 300, 64, torch.bfloat16, seed=10)
    a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    ids = t[:, None].clone()
    logits, lse = torch.randn(20, 1, device=gpu, generator=gen), torch.full((20,), 3.0, device=gpu)
    if what == "target":
        loss = dmuon.linear_cross_entropy(a, b, t, reduction="none")
    else:
        loss = dmuon.linear_distillation(a, b, ids, logits, teacher_lse=lse, reduction="none")
    with torch.no_grad():
        dict(target=t, ids=ids, logits=logits, lse=lse, hidden=a, weight=b)[what].zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


@pytest.mark.gpu
def test_gradient_against_differences(gpu):
    """Directional derivative of the mean loss by central differences of the exact losses."""
    h, w, t, gen = _inputs(gpu, 33, 190, 48, torch.bfloat16, seed=9)
    a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dmuon.linear_cross_entropy(a, b, t, z_loss=1e-3).backward()
    dh = torch.randn(h.shape, device=gpu, generator=gen, dtype=torch.float64)
    dw = torch.randn(w.shape, device=gpu, generator=gen, dtype=torch.float64) / 7

    def mean(eps):
        z = (h.double() + eps * dh) @ (w.double() + eps * dw).t()
        lse = torch.logsumexp(z, 1)
        return (lse - z.gather(1, t[:, None])[:, 0] + 1e-3 * lse ** 2).mean()
    slope = float(mean(1e-5) - mean(-1e-5)) / 2e-5
    got = float((a.grad.double() * dh).sum() + (b.grad.double() * dw).sum())
    (_, bh), (_, bw) = _ce(h, w, t, z_loss=1e-3).grads(torch.full((33,), 1 / 33, device=gpu))
    assert abs(got - slope) <= float((bh * dh.abs()).sum() + (bw * dw.abs()).sum()) + 1e-6
    assert abs(got - slope) <= 0.02 * abs(slope)


@pytest.mark.gpu
def test_another_stream_and_a_captured_graph(gpu):
    h, w, t, gen = _inputs(gpu, 200, 1000, 128, torch.bfloat16, seed=4)
    ids = torch.randint(0, 1000, (200, 6), device=gpu, generator=gen)
    logits = torch.randn(200, 6, device=gpu, generator=gen)
    a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)

    def step():
        loss = dmuon.linear_cross_entropy(a, b, t) + dmuon.linear_distillation(a, b, ids, logits)
        return (loss.detach(), *torch.autograd.grad(loss, (a, b)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        new, _, _, _ = _inputs(gpu, 200, 1000, 128, torch.bfloat16, seed=20 + seed)
        with torch.no_grad():
            a.copy_(new)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, held))


@pytest.mark.gpu
def test_the_workspace_does_not_grow_with_the_tokens(gpu):
    """The logits of 40000 tokens over 50000 classes would be 8 GB in fp32; what the call holds
    beside its results stays within its chunk workspace and the weight gradient's fp32 sums."""
    n, v, d = 40000, 50000, 64
    h, w, t, _ = _inputs(gpu, n, v, d, torch.bfloat16)
    a, b = h.requires_grad_(True), w.requires_grad_(True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    dmuon.linear_cross_entropy(a, b, t).backward()
    assert torch.cuda.max_memory_allocated() - before < 4.5e9


@pytest.mark.gpu
def test_weights_past_32_bit_offsets(gpu):
    """A weight of more than 2^31 values: losses and gradients at its end and beginning."""
    n, v, d = 8, (1 << 20) + 37, 2056
    gen = torch.Generator(device=gpu).manual_seed(0)
    w = torch.empty(v, d, dtype=torch.bfloat16, device=gpu).normal_(0, 0.02, generator=gen)
    assert w.numel() > 1 << 31
    h = torch.randn(n, d, device=gpu, generator=gen).bfloat16()
    t = torch.tensor([0, 1, 70000, v // 2, v - 70000, v - 3, v - 2, v - 1], device=gpu)
    a, b = h.requires_grad_(True), w.requires_grad_(True)
    loss = dmuon.linear_cross_entropy(a, b, t)
    loss.backward()
    hd, wd = h.detach(), w.detach()
    z = torch.cat([hd.double() @ part.double().t() for part in wd.split(1 << 17)], 1)
    lse = torch.logsumexp(z, 1)
    want = float((lse - z.gather(1, t[:, None])[:, 0]).mean())
    assert abs(float(loss.detach()) - want) <= 2.0 ** -20 * (1 + abs(want)) * 4
    dz = (z - lse[:, None]).exp()
    dz[torch.arange(n, device=gpu), t] -= 1
    dz /= n
    for rows in (slice(0, 300), slice(v // 2 - 100, v // 2 + 100), slice(v - 300, v)):
        want = dz[:, rows].t() @ hd.double()
        slack = (U[hd.dtype] + 2.0 ** -11 + 1e-4) * (dz[:, rows].abs().t() @ hd.double().abs())
        _within(b.grad[rows], want, slack + U[hd.dtype] * want.abs() + 1e-30)
    want = sum(dz[:, i:i + (1 << 17)] @ part.double()
               for i, part in zip(range(0, v, 1 << 17), wd.split(1 << 17)))
    size = sum(dz[:, i:i + (1 << 17)].abs() @ part.double().abs()
               for i, part in zip(range(0, v, 1 << 17), wd.split(1 << 17)))
    _within(a.grad, want, (U[hd.dtype] + 2.0 ** -11 + 1e-4) * size + U[hd.dtype] * want.abs())


def _refuse(match, call, kind=ValueError):
    with pytest.raises(kind, match=match):
        call()


def test_refusals_without_gpu():
    h, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(10, 8, dtype=torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int64)
    ce, kd = dmuon.linear_cross_entropy, dmuon.linear_distillation
    _refuse("reduction", lambda: ce(h, w, t, reduction="batchmean"))
    _refuse("do not fit", lambda: ce(h[:, :7], w, t))
    _refuse("do not fit", lambda: ce(h, w[0], t))
    _refuse("no values", lambda: ce(h, w[:0], t))
    _refuse("bfloat16 or float16", lambda: ce(h.float(), w.float(), t))
    _refuse("bfloat16 or float16", lambda: ce(h, w.half(), t))
    _refuse("GPU", lambda: ce(h, w, t), RuntimeError)
    _refuse("GPU", lambda: kd(h, w, t[:, None], torch.zeros(4, 1)), RuntimeError)


@pytest.mark.gpu
def test_refusals(gpu):
    h, w, t, _ = _inputs(gpu, 4, 10, 8, torch.bfloat16)
    ce, kd = dmuon.linear_cross_entropy, dmuon.linear_distillation
    ids, logits = t[:, None], torch.zeros(4, 1, device=gpu)
    _refuse("integers", lambda: ce(h, w, t.float()))
    _refuse("shape", lambda: ce(h, w, t[:3]))
    _refuse("chunk_tokens", lambda: ce(h, w, t, chunk_tokens=0))
    _refuse("live on", lambda: ce(h, w, t.cpu()), RuntimeError)
    _refuse("temperature", lambda: kd(h, w, ids, logits, temperature=0.0))
    _refuse("temperature", lambda: kd(h, w, ids, logits, temperature=float("nan")))
    _refuse("teacher_ids", lambda: kd(h, w, ids[:, :0], logits[:, :0]))
    _refuse("teacher_ids", lambda: kd(h, w, t, logits))
    _refuse("teacher_logits", lambda: kd(h, w, ids, logits[:3]))
    _refuse("teacher_lse", lambda: kd(h, w, ids, logits, teacher_lse=logits))


def test_c_entry_refusals_without_gpu():
    import ctypes

    from dmuon_amd import _C
    lib, need = _C.lib(), ctypes.c_int64()
    good = dict(dtype=1, grad_dtype=1, reduction=1, tokens=4, vocab=100, dim=64, ld_hidden=64,
                ld_weight=64, hidden=4096, weight=4096, targets=4096, loss=4096, reduced=4096,
                d_hidden=4096, d_weight=4096, temperature=1.0)

    def size(**kw):
        return lib.dmuon_head_loss_workspace_size(ctypes.byref(_C.HeadLossArgs(**{**good, **kw})),
                                                  ctypes.byref(need))

    def says(rc, text):
        assert rc != 0 and text in lib.dmuon_last_error().decode()

    assert size() == 0 and need.value >= 4 * 128 * 2      # two bytes a logit, rows of whole 64
    says(size(dtype=0), "16-bit")
    says(size(grad_dtype=2), "gradients")
    says(size(tokens=-1), "tokens")
    says(size(vocab=0), "vocab")
    says(size(dim=0), "dim")
    says(size(ld_weight=63), "pitches")
    says(size(chunk_tokens=-1), "chunk_tokens")
    says(size(reduction=3), "reduction")
    says(size(targets=None), "either")
    says(size(teacher_ids=4096), "either")
    says(size(targets=None, teacher_ids=4096, k_list=0), "k_list")
    says(size(targets=None, teacher_ids=4096, k_list=1), "teacher_logits")
    says(size(targets=None, teacher_ids=4096, k_list=1, teacher_logits=4096, temperature=0.0),
         "temperature")
    says(size(targets=None, teacher_ids=4096, k_list=1, teacher_logits=4096, z_loss=1.0), "z_loss")

    def run(ws=4096, nbytes=1 << 40, **kw):
        return lib.dmuon_head_loss(ctypes.byref(_C.HeadLossArgs(**{**good, **kw})), ws, nbytes, None)

    says(run(nbytes=16), "workspace")
    says(run(ws=4100), "aligned")
    says(run(weight=None), "NULL")
    says(run(reduced=None), "reduced")
    says(run(reduction=0), "row_grad")
    says(lib.dmuon_head_loss_workspace_size(None, ctypes.byref(need)), "NULL")
    says(run(reduction=0, d_hidden=None, d_weight=None, loss=None), "loss")
    says(lib.dmuon_scale_by(4096, 4096, 4, None, None, 0, 7, 1, 4096, None), "dtype")
    says(lib.dmuon_scale_by(4096, 4096, 4, None, None, 0, 1, 2, 4096, None), "in place")
    says(lib.dmuon_scale_by(None, None, 4, None, None, 0, 1, 1, 4096, None), "NULL")
    says(lib.dmuon_scale_by(4096, 4096, 4, None, 4096, 2, 1, 1, 4096, None), "NULL")
    assert lib.dmuon_scale_by(None, None, 0, None, None, 0, 1, 1, None, None) == 0


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_tangents_and_tracers_are_refused(dev):
    """A tangent would be lost and a recorded call would return memory that nothing has written."""
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    h = torch.zeros(4, 8, dtype=torch.bfloat16, device=dev)
    w = torch.zeros(10, 8, dtype=torch.bfloat16, device=dev)
    t = torch.zeros(4, dtype=torch.int64, device=dev)
    ids, logits = t[:, None], torch.zeros(4, 1, device=dev)
    calls = (lambda a, b: dmuon.linear_cross_entropy(a, b, t),
             lambda a, b: dmuon.linear_distillation(a, b, ids, logits))
    for call in calls:
        with forward_ad.dual_level():
            _refuse("forward-mode", lambda: call(forward_ad.make_dual(h, h), w), RuntimeError)
            _refuse("forward-mode", lambda: call(h, forward_ad.make_dual(w, w)), RuntimeError)
        _refuse("tracer", lambda: torch.jit.trace(call, (h, w), check_trace=False), RuntimeError)
        _refuse("tracer", lambda: make_fx(call)(h, w), RuntimeError)


@pytest.mark.gpu
@pytest.mark.parametrize("n,chunks", [(200, (1, 100)), (1100, (256, 512, 1024))])
@pytest.mark.parametrize("v", [1003, 5000, 32001])
def test_chunks_do_not_change_a_losss_bits(gpu, n, chunks, v):
    """Statistics of many classes join in one order whatever the chunk: calls on both sides of 128
    and 1024 tokens, in chunks on the other side and with a shorter last one."""
    h, w, t, gen = _inputs(gpu, n, v, 64, torch.bfloat16, seed=11)
    ids = torch.randint(0, v, (n, 70), device=gpu, generator=gen)
    logits = torch.randn(n, 70, device=gpu, generator=gen)
    for call in (lambda c: dmuon.linear_cross_entropy(h, w, t, reduction="none", chunk_tokens=c),
                 lambda c: dmuon.linear_distillation(h, w, ids, logits, reduction="none",
                                                     chunk_tokens=c)):
        whole = call(None)
        for chunk in chunks:
            assert torch.equal(call(chunk), whole)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,chunk", [(150, None), (700, 256)])
@pytest.mark.parametrize("what", ["z_loss", "negative z_loss", "teacher_lse"])
def test_large_factors_of_the_probabilities(gpu, what, n, chunk, dt):
    """A probability's factor in the gradient is c = mass + 2 z_loss lse, which a z_loss, or a teacher's
    log-sum-exp under its own logits, makes large: 16-bit gradients stay finite and right.

    Bounds, beside those above: c p is off relatively (c itself by z_err / lse at most, lse > 1); what
    the type holds of the smallest values goes with the largest c, 2^-34 of it in fp16 and 2^-39 of
    exponentials in bf16; the loss has c's size."""
    v, d = 300, 64
    h, w, t, gen = _inputs(gpu, n, v, d, dt, seed=12, lean=30.0)
    t[::7] = -100
    z = h.double() @ w.double().t()
    top = z.abs().amax()
    if what == "teacher_lse":
        ids = torch.rand(n, v, device=gpu, generator=gen).argsort(1)[:, :6]
        logits = torch.randn(n, 6, device=gpu, generator=gen)
        lse = -3.0 * torch.rand(n, device=gpu, generator=gen)
        lse[: n // 2] += 3.0                                       # the largest in a later chunk
        exact = _kd(h, w, ids, logits, lse)
        c = (logits.double() - lse.double()[:, None]).exp().sum(1)
        exact.loss_tol = 8 * (1 + c.amax()) * exact.loss_tol
        def call(a, b, r):
            return dmuon.linear_distillation(a, b, ids, logits, teacher_lse=lse, reduction=r,
                                             chunk_tokens=chunk)
    else:
        zl = 4.0 if what == "z_loss" else -4.0
        exact = _ce(h, w, t, z_loss=zl)
        c = 1 + 2 * abs(zl) * torch.logsumexp(z, 1)
        exact.loss_tol = (1 + 2 * abs(zl) * top) * (2 * exact.z_err + 2.0 ** -20 * (1 + top))
        def call(a, b, r):
            return dmuon.linear_cross_entropy(a, b, t, z_loss=zl, reduction=r, chunk_tokens=chunk)
    assert float(c.amax()) > 64
    exact.p = exact.p * c[:, None]
    least = float(c.amax()) * (2.0 ** -34 if dt == torch.float16 else 2.0 ** -39)
    plain = exact.grads
    exact.grads = lambda row: [(g, b + least * row.abs().amax() * other.abs().sum(0))
                               for (g, b), other in zip(plain(row), (exact.w, exact.h))]
    for reduction in ("mean", "none"):
        _check(exact, call, h, w, reduction)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_a_row_gradient_that_is_no_number_stays_in_its_row(gpu, dt):
    h, w, t, _ = _inputs(gpu, 40, 300, 64, dt, seed=13)
    t[9] = -100
    row = torch.linspace(-1.0, 2.0, 40, device=gpu)
    exact = _ce(h, w, t)
    want, bound = exact.grads(row)[0]
    for bad in (float("inf"), float("-inf"), float("nan")):
        for others in (row, torch.zeros_like(row)):
            a = h.clone().requires_grad_(True)
            g = others.clone()
            g[5] = bad
            g[9] = bad                                       # of an ignored token: no share
            dmuon.linear_cross_entropy(a, w, t, reduction="none").backward(g)
            keep = [i for i in range(40) if i != 5]
            assert not bool(a.grad[5].isfinite().all())
            if others is row:
                _within(a.grad[keep], want[keep], bound[keep])
            else:
                assert not bool(a.grad[keep].any())


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [0.25, 0.5, 1.0, 2.0])
def test_lists_of_extreme_logits_at_any_temperature(gpu, temperature):
    """Lists throughout of the type's lowest value, or with its highest, have finite logits: their
    probabilities are those of the differences."""
    h, w, t, _ = _inputs(gpu, 3, 300, 64, torch.bfloat16)
    big = torch.finfo(torch.float32).max
    ids = torch.arange(8, device=gpu).expand(3, 8).contiguous()
    logits = torch.zeros(3, 8, device=gpu)
    logits[0] = -big
    logits[1, 3] = big
    logits[2] = big
    even = torch.zeros(3, 8, device=gpu)
    even[1] = float("-inf")
    even[1, 3] = 0.0
    exact = _kd(h, w, ids, even, temperature=temperature)
    _check(exact, lambda a, b, r: dmuon.linear_distillation(a, b, ids, logits, reduction=r,
                                                            temperature=temperature), h, w, "none")


def test_temperatures_past_fp32_are_refused():
    import ctypes

    from dmuon_amd import _C
    h, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(10, 8, dtype=torch.bfloat16)
    ids, logits = torch.zeros(4, 1, dtype=torch.int64), torch.zeros(4, 1)
    for t in (1e-300, 1e-45, 1e-40, 1e39, float("inf"), -1.0):
        _refuse("temperature", lambda: dmuon.linear_distillation(h, w, ids, logits, temperature=t))
    lib, need = _C.lib(), ctypes.c_int64()
    for t in (1e-40, float("inf"), float("nan")):
        a = _C.HeadLossArgs(dtype=1, grad_dtype=1, reduction=1, tokens=4, vocab=100, dim=64,
                            ld_hidden=64, ld_weight=64, teacher_ids=4096, teacher_logits=4096,
                            k_list=1, temperature=t)
        assert lib.dmuon_head_loss_workspace_size(ctypes.byref(a), ctypes.byref(need)) != 0
        assert "temperature" in lib.dmuon_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,chunk", [(700, 256), (300, 100), (20, 7)])
def test_unreduced_losses_in_chunks(gpu, n, chunk, dt):
    h, w, t, gen = _inputs(gpu, n, 600, 72, dt, seed=14)
    t[::6] = -100
    _check(_ce(h, w, t), lambda a, b, r: dmuon.linear_cross_entropy(
        a, b, t, reduction=r, chunk_tokens=chunk), h, w, "none")
    ids = torch.rand(n, 600, device=gpu, generator=gen).argsort(1)[:, :9]
    logits = torch.randn(n, 9, device=gpu, generator=gen)
    _check(_kd(h, w, ids, logits, temperature=1.5), lambda a, b, r: dmuon.linear_distillation(
        a, b, ids, logits, temperature=1.5, reduction=r, chunk_tokens=chunk), h, w, "none")


@pytest.mark.gpu
def test_the_default_chunks(gpu):
    """More tokens than a default chunk holds: the memory stays the chunk's, and loss and gradients
    are those of 64 bits."""
    n, v, d = 90000, 50000, 64
    h, w, t, _ = _inputs(gpu, n, v, d, torch.bfloat16)
    t[::9] = -100
    a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    loss = dmuon.linear_cross_entropy(a, b, t)
    loss.backward()
    assert torch.cuda.max_memory_allocated() - before < 4.5e9      # two bytes a logit would be 9e9
    count = int((t != -100).sum())
    cols = torch.tensor([0, 1, 63, 64, 255, 256, 25000, v - 2, v - 1], device=gpu)
    total, dw, bw = 0.0, 0.0, 0.0
    for i in range(0, n, 3000):
        exact = _ce(h[i:i + 3000], w, t[i:i + 3000])
        total += float(exact.loss.sum())
        row = torch.full((exact.loss.shape[0],), 1.0 / count, device=gpu)
        dz = exact.dz[:, cols] / count
        slack = U[h.dtype] * dz.abs() + (2.0 ** -11 + 3 * exact.z_err) / count * torch.maximum(
            exact.p[:, cols], exact.dz[:, cols].abs())
        dw = dw + dz.t() @ exact.h
        bw = bw + slack.t() @ exact.h.abs()
        if i in (0, 30000, 60000, 87000):                          # chunks begin and end here
            (dh, bh), _ = exact.grads(row)
            _within(a.grad[i:i + 3000], dh, bh)
    assert abs(float(loss.detach()) - total / count) <= exact.loss_tol
    _within(b.grad[cols], dw, bw + U[h.dtype] * dw.abs() + 1e-30)


class _Wrapped(torch.Tensor):
    """A tensor that holds another and has no memory itself, as distributed tensors do."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype,
                                                   device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        out = func(*(t.inner if isinstance(t, _Wrapped) else t for t in args), **(kwargs or {}))
        return _Wrapped(out) if isinstance(out, torch.Tensor) else out


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["hidden", "weight", "target", "ids", "logits", "lse"])
def test_tensors_without_memory_are_refused(gpu, which):
    """An optional operand must not count as absent."""
    h, w, t, _ = _inputs(gpu, 4, 10, 8, torch.bfloat16)
    v = dict(hidden=h, weight=w, target=t, ids=t[:, None], logits=torch.zeros(4, 1, device=gpu),
             lse=torch.ones(4, device=gpu))
    v[which] = _Wrapped(v[which])
    with pytest.raises(RuntimeError, match="memory"):
        if which == "target":
            dmuon.linear_cross_entropy(v["hidden"], v["weight"], v["target"])
        else:
            dmuon.linear_distillation(v["hidden"], v["weight"], v["ids"], v["logits"],
                                      teacher_lse=v["lse"])


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["hidden", "weight", "target", "ids", "logits", "lse"])
def test_lazily_negated_operands(gpu, which):
    """A view whose negation torch has put off (as of a conjugate's imaginary part)."""
    h, w, t, gen = _inputs(gpu, 6, 50, 40, torch.bfloat16, seed=15)
    v = dict(hidden=h, weight=w, target=t, ids=t[:, None], lse=torch.ones(6, device=gpu),
             logits=torch.randn(6, 1, device=gpu, generator=gen))

    def call(v):
        if which == "target":
            return dmuon.linear_cross_entropy(v["hidden"], v["weight"], v["target"], reduction="none")
        return dmuon.linear_distillation(v["hidden"], v["weight"], v["ids"], v["logits"],
                                         teacher_lse=v["lse"], reduction="none")

    put_off = {**v, which: torch._neg_view((-v[which]).contiguous())}
    assert put_off[which].is_neg()
    assert torch.equal(call(put_off), call(v))
    for reduction in ("none", "sum"):
        grads = []
        for f in (torch._neg_view, torch.neg):
            a = h.clone().requires_grad_(True)
            loss = dmuon.linear_cross_entropy(a, w, t, reduction=reduction)
            grads += torch.autograd.grad(loss, a, f(torch.ones_like(loss)))
        assert torch.equal(*grads)


@pytest.mark.parametrize("n,v,d,k", [(8192, 128256, 4096, 0), (20000, 128256, 4096, 0),
                                     (20000, 128256, 4100, 0), (65536, 128256, 4096, 4096),
                                     (90000, 50000, 64, 0)])
def test_the_workspace_is_what_is_documented(n, v, d, k):
    """A chunk's logits, gradient and statistics within 4 GiB, and the terms beside them: the weight
    gradient's fp32 sums over several chunks, padded copies, a few bytes a token and list entry."""
    import ctypes

    from dmuon_amd import _C
    need = ctypes.c_int64()
    what = dict(teacher_ids=4096, teacher_logits=4096, k_list=k) if k else dict(targets=4096)
    a = _C.HeadLossArgs(dtype=1, grad_dtype=1, reduction=1, tokens=n, vocab=v, dim=d, ld_hidden=d,
                        ld_weight=d, hidden=4096, weight=4096, reduced=4096, d_hidden=4096,
                        d_weight=4096, temperature=1.0, **what)
    assert _C.lib().dmuon_head_loss_workspace_size(ctypes.byref(a), ctypes.byref(need)) == 0
    row = -(-v // 64) * (64 * 2 + 8)
    most = (4 << 30) // row
    chunks = -(-n // most)
    chunk = min(n, -(-(-(-n // chunks)) // 256) * 256) if chunks > 1 else n
    assert chunk * row <= 4 << 30
    pad = -(-d // 64) * 64
    total = chunk * row + n * (20 + 12 * max(k, 1)) + (4 * v * d if chunks > 1 else 0) + \
        (2 * (v + chunk) * pad if d % 8 else 0)
    assert total <= need.value <= total + 16 * 256
