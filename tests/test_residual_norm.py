"""``residual_norm`` against its definition in 64 bits.

Bounds. A row's mean square is an fp32 sum of ``dim`` positive terms (relative error at most
``2^-24 (dim / 64 + 16)`` in the kernels' order), its root halves that; the element operations add a
few more roundings of 2^-24. Every result is rounded once to its type (``u``). The gradients' row
sums have terms of both signs: their error is bounded by the same relative error times the sum of
magnitudes. Column sums over ``rows`` rows add ``2^-24 * rows / 8`` relative to the sum of
magnitudes (registers, then partial rows).
"""
import pytest
import torch

import dmuon_amd as dmuon

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}


def _inputs(dev, shape, dt, wt, post, gate_shape, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, device=dev, generator=gen)
    d = shape[-1]
    v = {"x": (2 * randn(*shape)).to(dt), "y": randn(*shape).to(dt),
         "pre": (1 + 0.2 * randn(d)).to(wt),
         "post": (1 + 0.2 * randn(d)).to(wt) if post else None,
         "gate": randn(*gate_shape).to(wt) if gate_shape is not None else None}
    return v, (randn(*shape).to(dt), randn(*shape).to(dt))


def _call(v, scale, eps=1e-6):
    return dmuon.residual_norm(v["x"], v["y"], v["pre"], post_weight=v["post"], gate=v["gate"],
                               residual_scale=scale, eps=eps)


def _spread(gate, x):
    if gate.dim() == 2 and x.dim() == 2:
        return gate.repeat_interleave(x.shape[0] // gate.shape[0], 0)
    return gate


def _exact(v, scale, eps=1e-6):
    """(x_new, h) in 64 bits, with the gradient's graph, and the leaves."""
    leaf = {k: None if t is None else t.detach().double().requires_grad_(True) for k, t in v.items()}
    x_new = scale * leaf["x"]
    if leaf["y"] is not None:
        u = leaf["y"]
        if leaf["post"] is not None:
            u = u / (u.pow(2).mean(-1, keepdim=True) + eps).sqrt() * leaf["post"]
        if leaf["gate"] is not None:
            u = u * _spread(leaf["gate"], u)
        x_new = x_new + u
    h = x_new / (x_new.pow(2).mean(-1, keepdim=True) + eps).sqrt() * leaf["pre"]
    return x_new, h, leaf


def _within(name, got, want, dt, mag):
    """|got - want| against the rounding of the result and fp32 errors relative to ``mag``."""
    assert got.dtype == dt, name
    err = (got.double() - want).abs()
    bound = U[dt] * want.abs() + mag + TINY[dt]
    assert bool((err <= bound).all()), (name, float((err / bound).max()))


def _check(v, outs, scale, eps=1e-6):
    d = v["x"].shape[-1]
    rows = v["x"].numel() // d
    leaves = {k: None if t is None else t.detach().requires_grad_(True) for k, t in v.items()}
    x_new, h = _call(leaves, scale, eps)
    ex, eh, el = _exact(v, scale, eps)
    ex.retain_grad()
    rel = 2.0 ** -24 * (d / 64 + 24)
    # the terms of a sum bound its error
    parts = scale * el["x"].detach().abs() + (ex.detach() - scale * el["x"].detach()).abs()
    s = 1 / (ex.detach().pow(2).mean(-1, keepdim=True) + eps).sqrt()
    grow = parts.amax(-1, keepdim=True) * s            # how far x_new's error shows in its norm
    _within("x_new", x_new.detach(), ex.detach(), v["x"].dtype, rel * parts)
    _within("h", h.detach(), eh.detach(), v["x"].dtype,
            rel * (parts * s * el["pre"].detach().abs() + grow * eh.detach().abs()))
    names = [k for k in v if v[k] is not None]
    got = torch.autograd.grad((x_new, h), [leaves[k] for k in names], outs)
    want = torch.autograd.grad((ex, eh), [el[k] for k in names], [o.double() for o in outs])
    # magnitudes: every gradient as a sum of its terms, the row sums by Cauchy-Schwarz
    e, g = outs[0].double().abs(), outs[1].double().abs() * el["pre"].detach().abs()
    norm = lambda t: t.pow(2).mean(-1, keepdim=True).sqrt()
    d_mag = e + s * (1 + grow) * (g + (ex.detach().abs() * s + grow) * norm(g))
    mags = {"x": abs(scale) * d_mag}
    mags["pre"] = outs[1].double().abs() * (ex.detach().abs() * s + grow)
    gate = 1.0 if v["gate"] is None else _spread(el["gate"].detach(), ex).abs()
    if v["y"] is not None:
        y = el["y"].detach()
        if v["post"] is None:
            mags["y"] = gate * d_mag
            u = y.abs()
        else:
            r = 1 / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt()
            c = gate * el["post"].detach().abs()
            mags["y"] = r * (c * d_mag + y.abs() * r * norm(c * d_mag))
            mags["post"] = gate * d_mag * y.abs() * r
            u = y.abs() * r * el["post"].detach().abs()
        if v["gate"] is not None:
            mags["gate"] = d_mag * u
    for k, a, b in zip(names, got, want):
        mag = mags[k]
        if k in ("pre", "post"):
            mag = mag.reshape(-1, d).sum(0) * (1 + rows / 8 / (d / 64 + 24))
        elif k == "gate":
            per = rows // max(1, v["gate"].numel() // d)
            mag = mag.reshape(-1, per, d).sum(1).reshape(v["gate"].shape)
            mag = mag * (1 + per / 8 / (d / 64 + 24))
        _within("d_" + k, a, b, v[k].dtype, 4 * rel * mag)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,wt", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                   (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                   (torch.float16, torch.float16)])
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 4096), (3, 7), (5, 64), (64, 513), (777, 1001),
                                    (33, 512), (130, 2048), (1500, 300), (2100, 72), (9, 8192),
                                    (4, 8200), (3, 12345), (2, 16384)])
def test_sizes_and_types(gpu, rows, d, dt, wt):
    v, outs = _inputs(gpu, (rows, d), dt, wt, True, (d,))
    _check(v, outs, 0.75)


@pytest.mark.gpu
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("shape,gate", [
    ((6, 50, 96), None), ((6, 50, 96), (96,)), ((6, 50, 96), (6, 1, 96)), ((6, 50, 96), (1, 1, 96)),
    ((6, 50, 96), (6, 50, 96)), ((300, 96), (4, 96)), ((300, 96), (300, 96)), ((2600, 40), (1300, 40)),
    ((2600, 40), (2600, 40)), ((2, 1100, 40), (2, 1, 40)), ((1, 1, 40), (1, 1, 40))])
def test_gates(gpu, shape, gate, post):
    v, outs = _inputs(gpu, shape, torch.float32, torch.float32, post, gate, seed=1)
    _check(v, outs, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_first_norm_without_a_block(gpu, scale):
    v, outs = _inputs(gpu, (70, 200), torch.float32, torch.float32, False, None, seed=2)
    v["y"] = None
    _check(v, outs, scale)
    if scale == 1.0:
        assert _call(v, scale)[0].data_ptr() == v["x"].data_ptr()


@pytest.mark.gpu
def test_one_gradient_may_be_missing(gpu):
    """Only the stream or only the block's input is used further on."""
    v, outs = _inputs(gpu, (90, 260), torch.float32, torch.float32, True, (260,), seed=3)
    for which in (0, 1):
        leaves = {k: t.detach().requires_grad_(True) for k, t in v.items()}
        got = torch.autograd.grad(_call(leaves, 0.5)[which], list(leaves.values()), outs[which],
                                  allow_unused=True)
        *both, el = _exact(v, 0.5)
        want = torch.autograd.grad(both[which], list(el.values()), outs[which].double(),
                                   allow_unused=True)
        for a, b in zip(got, want):
            b = torch.zeros_like(a, dtype=torch.float64) if b is None else b
            # 90 rows of values around 1: sums within 2^-24 * 90 of their magnitude, at most ~90
            assert float((a.double() - b).abs().max()) <= 2.0 ** -24 * 90 * 90


@pytest.mark.gpu
def test_wanted_gradients_only(gpu):
    v, outs = _inputs(gpu, (40, 100), torch.bfloat16, torch.float32, True, (100,), seed=4)
    every = {k: t.clone().requires_grad_(True) for k, t in v.items()}
    want = dict(zip(v, torch.autograd.grad(_call(every, 1.0), list(every.values()), outs)))
    for k in v:
        some = {j: t.clone().requires_grad_(j == k) for j, t in v.items()}
        got, = torch.autograd.grad(_call(some, 1.0), some[k], outs)
        assert torch.equal(got, want[k])
    with torch.no_grad():
        x_new, h = _call(every, 1.0)
    assert not x_new.requires_grad and not h.requires_grad


@pytest.mark.gpu
def test_zero_rows_large_values_and_no_numbers(gpu):
    v, outs = _inputs(gpu, (8, 128), torch.float32, torch.float32, True, None, seed=5)
    v["x"][0] = 0.0
    v["y"][0] = 0.0                                   # a row of zeros: eps alone under the root
    v["y"][1] = 1e-30                                 # squares that underflow
    v["x"][2] = 1e15
    _check(v, outs, 1.0)
    v["x"][4, 3] = float("nan")
    v["y"][5, 3] = float("inf")
    x_new, h = _call(v, 1.0)
    assert bool(h[4].isnan().all()) and not bool(h[5].isfinite().all())
    assert bool(h[[0, 1, 2, 3, 6, 7]].isfinite().all())


@pytest.mark.gpu
def test_no_rows(gpu):
    v, outs = _inputs(gpu, (0, 96), torch.bfloat16, torch.float32, True, (96,), seed=6)
    # memory that was used before: every result has to be written
    held = [torch.full((96,), 7.0, device=gpu) for _ in range(8)]
    del held
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items()}
    got = torch.autograd.grad(_call(leaves, 1.0), list(leaves.values()), outs)
    for a, t in zip(got, leaves.values()):
        assert a.shape == t.shape and not bool(a.any())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [96, 131])
def test_strides_and_alignment(gpu, d, dt):
    v, outs = _inputs(gpu, (50, d), dt, torch.float32, True, (d,), seed=7)
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items()}
    want = _call(leaves, 0.5)
    want = [*want, *torch.autograd.grad(want, list(leaves.values()), outs)]

    def spread(t, off):
        if t.dim() == 1:
            wide = torch.full((d + 9,), float("nan"), dtype=t.dtype, device=gpu)
            wide[off:off + d] = t
            return wide[off:off + d]
        wide = torch.full((50, d + 9), float("nan"), dtype=t.dtype, device=gpu)
        wide[:, off:off + d] = t
        return wide[:, off:off + d]

    for off in (1, 3):
        views = {k: spread(t, off).detach().requires_grad_(True) for k, t in v.items()}
        got = _call(views, 0.5)
        got = [*got, *torch.autograd.grad(got, list(views.values()),
                                          [spread(o, off) for o in outs])]
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    # columns apart, and one row for all
    apart = {**v, "x": v["x"].t().contiguous().t()}
    assert torch.equal(_call(apart, 0.5)[1], want[1])
    one = _call({**v, "x": v["x"][:1].expand(50, d), "y": v["y"][:1].expand(50, d)}, 0.5)[1]
    assert torch.equal(one, want[1][:1].expand(50, d))


@pytest.mark.gpu
def test_gradient_against_differences(gpu):
    v, outs = _inputs(gpu, (12, 60), torch.float32, torch.float32, True, (3, 60), seed=8)
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items()}
    got = torch.autograd.grad(_call(leaves, 0.9), list(leaves.values()), outs)
    gen = torch.Generator(device=gpu).manual_seed(1)
    step = {k: torch.randn(t.shape, device=gpu, generator=gen, dtype=torch.float64)
            for k, t in v.items()}

    def value(eps):
        ex, eh, _ = _exact({k: t.double() + eps * step[k] for k, t in v.items()}, 0.9)
        return float((ex * outs[0].double()).sum() + (eh * outs[1].double()).sum())
    slope = (value(1e-6) - value(-1e-6)) / 2e-6
    along = sum(float((g.double() * step[k]).sum()) for k, g in zip(v, got))
    size = sum(float((g.double() * step[k]).abs().sum()) for k, g in zip(v, got))
    assert abs(along - slope) <= 2.0 ** -20 * size + 1e-6 * abs(slope)


@pytest.mark.gpu
def test_same_bits_every_time_on_any_stream_and_in_a_graph(gpu):
    v, outs = _inputs(gpu, (3000, 264), torch.bfloat16, torch.float32, True, (264,), seed=9)
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items()}

    def step():
        pair = _call(leaves, 1.0)
        return [t.detach() for t in pair] + list(
            torch.autograd.grad(pair, list(leaves.values()), outs))

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
        new, _ = _inputs(gpu, (3000, 264), torch.bfloat16, torch.float32, True, (264,), 30 + seed)
        with torch.no_grad():
            leaves["x"].copy_(new["x"])
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))


def _refuse(match, *args, kind=ValueError, **kw):
    with pytest.raises(kind, match=match):
        dmuon.residual_norm(*args, **kw)


def test_refusals_without_gpu():
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    _refuse("dim", torch.zeros(2, 0), None, torch.ones(0))
    _refuse("dim", torch.zeros(1, 16385), None, torch.ones(16385))
    _refuse("dtype", x.double(), x.double(), w)
    _refuse("y must match", x, x.half(), w)
    _refuse("y must match", x, x[:1], w)
    _refuse("need the block", x, None, w, post_weight=w)
    _refuse("need the block", x, None, w, gate=w)
    _refuse("pre_weight", x, x, w[:7])
    _refuse("post_weight", x, x, w, post_weight=w[None])
    _refuse("pre_weight must be", x.half(), x.half(), w.bfloat16())
    for shape in ((7,), (3, 8), (1, 3, 8), (2, 2, 8), (4, 1, 8), (1, 1, 1, 8)):
        _refuse("gate", x, x, w, gate=torch.ones(shape))
    _refuse("gate", x[0], x[0], w, gate=torch.ones(2, 8))
    _refuse("GPU", x, x, w, kind=RuntimeError)


def test_c_entry_refusals_without_gpu():
    import ctypes

    from dmuon_amd import _C
    lib, need = _C.lib(), ctypes.c_int64()
    good = dict(x=4096, y=4096, w_pre=4096, w_post=4096, gate=4096, stats=4096, x_new=4096, h=4096,
                dx_new=4096, dh=4096, dx=4096, dy=4096, d_pre=4096, d_post=4096, d_gate=4096,
                rows=6, dim=64, gates=3, ld_x=64, ld_y=64, ld_dx_new=64, ld_dh=64, scale=1.0,
                eps=1e-6, dtype=1, pre_dtype=0, post_dtype=0, gate_dtype=0)

    def says(rc, text):
        assert rc != 0 and text in lib.dmuon_last_error().decode()

    def args(**kw):
        return ctypes.byref(_C.ResidualNormArgs(**{**good, **kw}))

    size = lib.dmuon_residual_norm_grad_workspace_size
    assert size(args(), ctypes.byref(need)) == 0 and need.value >= 2 * 64 * 4
    for fn in (lambda a: lib.dmuon_residual_norm(a, None), lambda a: size(a, ctypes.byref(need))):
        says(fn(args(dtype=5)), "dtype")
        says(fn(args(gate_dtype=9)), "dtype")
        says(fn(args(rows=-1)), "rows")
        says(fn(args(dim=0)), "dim")
        says(fn(args(dim=1 << 20)), "dim")
        says(fn(args(w_pre=None)), "w_pre")
        says(fn(args(y=None)), "need the block")
        says(fn(args(gates=4)), "divide")
        says(fn(args(ld_x=63)), "pitch")
    says(lib.dmuon_residual_norm(args(h=None), None), "h is NULL")
    grad = lib.dmuon_residual_norm_grad
    says(grad(args(), 4096, 16, None), "workspace")
    says(grad(args(), 4097, 1 << 30, None), "aligned")
    says(grad(args(stats=None), 4096, 1 << 30, None), "stats")
    says(grad(args(ld_dh=63), 4096, 1 << 30, None), "pitch")
    says(grad(args(w_post=None), 4096, 1 << 30, None), "not there")


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_tangents_and_tracers_are_refused(dev):
    """A tangent would be lost and a recorded call would return memory that nothing has written."""
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    v = [torch.ones(2, 8, device=dev), torch.ones(2, 8, device=dev), torch.ones(8, device=dev),
         torch.ones(8, device=dev), torch.ones(8, device=dev)]

    def call(x, y, pre, post, gate):
        return dmuon.residual_norm(x, y, pre, post_weight=post, gate=gate)

    for k in range(5):
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(t, t) if i == k else t for i, t in enumerate(v)]
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*dual)
    with pytest.raises(RuntimeError, match="tracer"):
        torch.jit.trace(call, tuple(v), check_trace=False)
    with pytest.raises(RuntimeError, match="tracer"):
        make_fx(call)(*v)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,gate", [((0, 5, 40), (0, 1, 40)), ((0, 5, 40), (0, 5, 40)),
                                        ((3, 0, 40), (3, 1, 40)), ((0, 40), (7, 40))])
def test_no_rows_give_every_gate_a_gradient(gpu, shape, gate):
    v, outs = _inputs(gpu, shape, torch.bfloat16, torch.float32, True, gate, seed=10)
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items()}
    got = torch.autograd.grad(_call(leaves, 1.0), list(leaves.values()), outs)
    for a, t in zip(got, leaves.values()):
        assert a.shape == t.shape and not bool(a.any())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,gate", [((300, 8200), (300, 8200)), ((600, 8200), (300, 8200)),
                                        ((2, 130, 16384), (2, 130, 16384)), ((130, 4096), (130, 4096)),
                                        ((1100, 2056), (550, 2056))])
def test_gates_of_wide_rows(gpu, shape, gate, dt):
    """Several gate groups in a block, one and two chunks of columns a thread."""
    v, outs = _inputs(gpu, shape, dt, torch.float32, True, gate, seed=11)
    _check(v, outs, 0.5)


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
@pytest.mark.parametrize("which", ["x", "y", "pre", "post", "gate"])
def test_tensors_without_memory_are_refused(gpu, which):
    """An optional operand must not count as absent."""
    v, _ = _inputs(gpu, (2, 8), torch.float32, torch.float32, True, (1, 8), seed=12)
    v[which] = _Wrapped(v[which])
    with pytest.raises(RuntimeError, match="memory"):
        _call(v, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["x", "y", "pre", "post", "gate"])
def test_lazily_negated_operands(gpu, which):
    """A view whose negation torch has put off (as of a conjugate's imaginary part)."""
    v, outs = _inputs(gpu, (6, 40), torch.float32, torch.float32, True, (2, 40), seed=13)
    put_off = {**v, which: torch._neg_view(v[which])}
    assert put_off[which].is_neg()
    v[which] = -v[which]
    for a, b in zip(_call(put_off, 0.5), _call(v, 0.5)):
        assert torch.equal(a, b)
    grads = [torch.autograd.grad(_call({**v, "x": x}, 0.5), x, [f(o) for o in outs])[0]
             for f in (torch._neg_view, torch.neg) for x in [v["x"].clone().requires_grad_(True)]]
    assert torch.equal(*grads)
