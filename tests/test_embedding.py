"""``embedding`` against its definition in 64 bits.

The lookup is one fp32 product, rounded once (twice in all: ``2^-24 + u`` relative). A class's gradient
is an fp32 sum of ``n`` rows in runs of 8 to 32 and then of the runs' sums: off by at most
``2^-24 (32 + n / 8 + 2)`` times the sum of magnitudes, and by the result's rounding.
"""
import pytest
import torch

import dmuon_amd as dmuon

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _within(name, got, want, dt, mag):
    assert got.dtype == dt, name
    err = (got.double() - want).abs()
    bound = U[dt] * (want.abs() + mag) + mag + TINY[dt]
    assert bool((err <= bound).all()), (name, float((err / bound).max()))


def _check(tokens, weight, dy, scale=1.0, padding_idx=None):
    leaf = weight.detach().requires_grad_(True)
    y = dmuon.embedding(tokens, leaf, scale=scale, padding_idx=padding_idx)
    (dw,) = torch.autograd.grad(y, leaf, dy)
    v, d = weight.shape
    t = tokens.reshape(-1).long()
    want = scale * weight.double()[t].view(*tokens.shape, d)
    _within("y", y.detach(), want, weight.dtype, 2.0 ** -24 * want.abs())
    g = scale * dy.reshape(-1, d).double()
    kept = torch.ones_like(t, dtype=torch.bool)
    if padding_idx is not None:
        kept = t != padding_idx % v
    total = torch.zeros(v, d, dtype=torch.float64, device=weight.device).index_add_(0, t[kept], g[kept])
    size = torch.zeros_like(total).index_add_(0, t[kept], g[kept].abs())
    n = torch.bincount(t[kept], minlength=v)[:, None].double()
    assert dw.shape == weight.shape
    _within("d_weight", dw, total, weight.dtype, 2.0 ** -24 * (34 + n / 8) * size)
    return y.detach(), dw


def _make(dev, n, v, d, dt, seed=0, hot=0.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    tokens = torch.randint(0, v, (n,), device=dev, generator=gen)
    tokens[torch.rand(n, device=dev, generator=gen) < hot] = v // 2
    weight = torch.randn(v, d, device=dev, generator=gen).to(dt)
    return tokens, weight, torch.randn(n, d, device=dev, generator=gen).to(dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("hot", [0.0, 0.5])
@pytest.mark.parametrize("n,v,d", [
    (1, 1, 1), (1, 3, 1), (2, 9, 1), (1, 1003, 4096), (31, 7, 3), (32, 2, 8), (33, 50, 300), (64, 512, 64), (1000, 511, 130),
    (1025, 300000, 12), (5000, 128256, 40), (3000, 3, 520), (70000, 1000, 24), (200, 9, 4100)])
def test_sizes_and_types(gpu, n, v, d, dt, hot):
    _check(*_make(gpu, n, v, d, dt, hot=hot), scale=1.0 if hot else 5.5)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 32, 64, 65, 4000])
def test_one_class_only(gpu, n):
    tokens, weight, dy = _make(gpu, n, 100, 72, torch.bfloat16, 1, hot=1.1)
    _check(tokens, weight, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(), (3, 0), (2, 3, 5)])
def test_shapes_of_tokens(gpu, shape):
    gen = torch.Generator(device=gpu).manual_seed(2)
    for kind in (torch.int64, torch.int32, torch.uint8):
        tokens = torch.randint(0, 20, shape, device=gpu, generator=gen).to(kind)
        weight = torch.randn(20, 16, device=gpu, generator=gen)
        _check(tokens, weight, torch.randn(*shape, 16, device=gpu, generator=gen))


@pytest.mark.gpu
@pytest.mark.parametrize("padding_idx", [0, 7, -1])
def test_padding_has_no_gradient(gpu, padding_idx):
    tokens, weight, dy = _make(gpu, 500, 30, 64, torch.float16, 3)
    y, dw = _check(tokens, weight, dy, padding_idx=padding_idx)
    assert not bool(dw[padding_idx].any())
    # whatever its rows' gradients hold
    dy[tokens == padding_idx % 30] = float("nan")
    leaf = weight.clone().requires_grad_(True)
    (again,) = torch.autograd.grad(dmuon.embedding(tokens, leaf, padding_idx=padding_idx), leaf, dy)
    assert torch.equal(again, dw)


@pytest.mark.gpu
def test_tokens_outside_the_vocabulary(gpu):
    tokens, weight, dy = _make(gpu, 300, 40, 64, torch.bfloat16, 4)
    good_y, good = _check(tokens, weight, dy)
    bad = tokens.repeat_interleave(2)
    bad[1::2] = torch.tensor([-1, 40, -100, 2 ** 40, -2 ** 63, 2 ** 32], device=gpu).repeat(50)
    leaf = weight.clone().requires_grad_(True)
    y = dmuon.embedding(bad, leaf)
    (dw,) = torch.autograd.grad(y, leaf, dy.repeat_interleave(2, 0))
    assert torch.equal(y[0::2].detach(), good_y) and bool(torch.isnan(y[1::2]).all())
    assert torch.equal(dw, good)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["pitch", "columns_first", "odd", "negated"])
def test_strides_and_alignment(gpu, kind):
    tokens, weight, dy = _make(gpu, 400, 60, 72, torch.float16, 5)
    want = _check(tokens, weight, dy)

    def lay(t):
        if kind == "pitch":
            wide = torch.zeros(t.shape[0], 100, device=gpu, dtype=t.dtype)
            wide[:, :72] = t
            return wide[:, :72]
        if kind == "columns_first":
            return t.t().contiguous().t()
        if kind == "odd":
            wide = torch.zeros(t.shape[0], 75, device=gpu, dtype=t.dtype)
            wide[:, 1:73] = t
            return wide[:, 1:73]
        return torch._neg_view(-t)
    got = _check(tokens.repeat_interleave(3)[::3], lay(weight), lay(dy))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    expanded = dy[:1].expand(400, 72)
    _check(tokens, weight, expanded)


@pytest.mark.gpu
def test_rows_past_32_bits(gpu):
    """A weight and a gradient of more than 2^32 bytes."""
    v, d = 70001, 32768
    weight = torch.empty(v, d, device=gpu, dtype=torch.bfloat16)
    tokens = torch.tensor([v - 1, 3, v - 1, 69000], device=gpu)
    weight[tokens] = torch.randn(4, d, device=gpu).bfloat16()
    leaf = weight.requires_grad_(True)
    y = dmuon.embedding(tokens, leaf)
    dy = torch.randn(4, d, device=gpu).bfloat16()
    assert torch.equal(y.detach(), weight.detach()[tokens])
    (dw,) = torch.autograd.grad(y, leaf, dy)
    assert torch.equal(dw[v - 1], (dy[0].float() + dy[2].float()).bfloat16())
    assert torch.equal(dw[3], dy[1]) and torch.equal(dw[69000], dy[3])
    dw[tokens] = 0
    assert not bool(dw.any())


@pytest.mark.gpu
def test_same_bits_every_time_on_any_stream_and_in_a_graph(gpu):
    tokens, weight, dy = _make(gpu, 6000, 700, 72, torch.bfloat16, 6, hot=0.3)
    leaf = weight.clone().requires_grad_(True)

    def step():
        y = dmuon.embedding(tokens, leaf, scale=3.0, padding_idx=5)
        return (y.detach(), *torch.autograd.grad(y, leaf, dy))
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        new = _make(gpu, 6000, 700, 72, torch.bfloat16, 20 + seed, hot=0.1 * seed)
        tokens.copy_(new[0])
        dy.copy_(new[2])
        with torch.no_grad():
            leaf.copy_(new[1])
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))


@pytest.mark.gpu
def test_gradient_against_differences(gpu):
    """The loss is linear in the weight: any step shows the slope."""
    tokens, weight, dy = _make(gpu, 200, 30, 64, torch.float32, 7)
    leaf = weight.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(dmuon.embedding(tokens, leaf, scale=0.5), leaf, dy)
    step = dw.double() / dw.double().norm()

    def value(e):
        return float((0.5 * (weight.double() + e * step)[tokens] * dy.double()).sum())
    slope, along = (value(1.0) - value(-1.0)) / 2, float((dw.double() * step).sum())
    assert abs(along - slope) <= 2.0 ** -18 * along


@pytest.mark.gpu
def test_tokens_written_to_in_between_and_second_gradients_are_refused(gpu):
    tokens, weight, dy = _make(gpu, 20, 30, 64, torch.float32, 8)
    leaf = weight.clone().requires_grad_(True)
    y = dmuon.embedding(tokens, leaf)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        torch.autograd.grad(y, leaf, dy, create_graph=True)
    y = dmuon.embedding(tokens, leaf)
    tokens.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward(dy)


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
@pytest.mark.parametrize("which", [0, 1])
def test_tensors_without_memory_are_refused(gpu, which):
    ops = list(_make(gpu, 20, 30, 64, torch.float32)[:2])
    ops[which] = _Wrapped(ops[which])
    with pytest.raises(RuntimeError, match="memory"):
        dmuon.embedding(*ops)


def _refuse(match, *args, kind=ValueError, **kw):
    with pytest.raises(kind, match=match):
        dmuon.embedding(*args, **kw)


def test_refusals_without_gpu():
    t, w = torch.zeros(3, dtype=torch.long), torch.zeros(5, 8)
    _refuse("tokens must be integers", t.float(), w)
    _refuse("tokens must be integers", t.bool(), w)
    _refuse("weight must be", t, w[0])
    _refuse("weight must be", t, w[:0])
    _refuse("weight must be", t, w[:, :0])
    _refuse("dtype", t, w.double())
    for bad in (5, -6):
        _refuse("padding_idx", t, w, padding_idx=bad)
    _refuse("GPU", t, w, kind=RuntimeError)


def test_c_entry_refusals_without_gpu():
    import ctypes

    from dmuon_amd import _C
    lib, need = _C.lib(), ctypes.c_int64()
    good = dict(tokens=4096, weight=4096, out=4096, dy=4096, d_weight=4096, tokens_n=100, vocab=50, dim=64,
                ld_weight=64, ld_dy=64, padding_idx=-1, scale=1.0, dtype=1)

    def says(rc, text):
        assert rc != 0 and text in lib.dmuon_last_error().decode()

    def args(**kw):
        return ctypes.byref(_C.EmbeddingArgs(**{**good, **kw}))

    size = lambda a: lib.dmuon_embedding_grad_workspace_size(a, ctypes.byref(need))
    grad = lambda a: lib.dmuon_embedding_grad(a, 4096, 1 << 40, None)
    forward = lambda a: lib.dmuon_embedding(a, None)
    assert size(args()) == 0 and need.value >= 100 * 8
    for fn in (forward, size, grad):
        says(fn(args(dtype=4)), "dtype")
        says(fn(args(tokens_n=-1)), "tokens")
        says(fn(args(vocab=0)), "vocab")
        says(fn(args(dim=0)), "dim")
        says(fn(args(tokens=None)), "tokens is NULL")
    says(forward(args(ld_weight=63)), "pitch")
    says(forward(args(out=None)), "NULL")
    says(grad(args(ld_dy=63)), "pitch")
    says(grad(args(d_weight=None)), "NULL")
    says(lib.dmuon_embedding_grad(args(), 4096, 16, None), "workspace")
    says(lib.dmuon_embedding_grad(args(), 4097, 1 << 40, None), "aligned")


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_tangents_and_tracers_are_refused(dev):
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    t, w = torch.zeros(3, dtype=torch.long, device=dev), torch.ones(5, 8, device=dev)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            dmuon.embedding(t, forward_ad.make_dual(w, w))
    with pytest.raises(RuntimeError, match="tracer"):
        torch.jit.trace(lambda x: dmuon.embedding(t, x), (w,), check_trace=False)
    with pytest.raises(RuntimeError, match="tracer"):
        make_fx(lambda x: dmuon.embedding(t, x))(w)


def test_scales_that_leave_fp32_are_refused():
    """The kernels multiply in fp32: a scale that it holds as infinity or not in full would give other rows."""
    t, w = torch.zeros(3, dtype=torch.long), torch.ones(5, 8)
    for bad in (1e39, -1e39, 1e-39, float("inf"), float("nan")):
        _refuse("scale must", t, w, scale=bad)
    for good in (0.0, -2.0, 1e38, 2.0 ** -126):
        _refuse("GPU", t, w, scale=good, kind=RuntimeError)
