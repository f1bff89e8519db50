"""``rotary_heads`` against its definition in 64 bits.

Bounds. A head's mean square is an fp32 sum of ``dim`` positive terms (relative error at most
``2^-24 (dim / 16 + 12)`` in the kernels' order), its root halves that; a rotation adds the errors of its
cosine and sine (an angle reduced in 64 bits and rounded to fp32 within an eighth of a turn: 2^-27 turns, and
the functions' own 2^-22) and two products. Every result is rounded once to its type (``u``). Relative to the
pair's size ``|z_i| + |z_j|`` that is ``2^-24 (dim / 16 + 24)``. The gradients' row sums have terms of both
signs, bounded by the same error times the sum of magnitudes; a weight's gradient sums over all heads and
tokens, ``2^-24`` times a few hundred additions in one lane, relative to the sum of magnitudes.
"""
import pytest
import torch

import dmuon_amd as dmuon

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
EPS = 1e-6


def _make(dev, lead, h, hk, d, r, dt, wt, norm=(True, True), seed=0, far=0, freq=torch.float32):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, device=dev, generator=gen)
    v = {"q": (2 * randn(*lead, h, d)).to(dt), "k": randn(*lead, hk, d).to(dt),
         "q_weight": (1 + 0.2 * randn(d)).to(wt) if norm[0] else None,
         "k_weight": (1 + 0.2 * randn(d)).to(wt) if norm[1] else None}
    n = lead[-1] if lead else 1
    positions = torch.arange(n, device=dev) * 3 + far if lead else torch.tensor(far, device=dev)
    at = torch.arange(r // 2, device=dev, dtype=torch.float64)
    inv_freq = (10000.0 ** (-2 * at / r)).to(freq)
    return v, positions, inv_freq, (randn(*lead, h, d).to(dt), randn(*lead, hk, d).to(dt))


def _call(v, positions, inv_freq, interleaved=False):
    return dmuon.rotary_heads(v["q"], v["k"], positions, inv_freq, q_weight=v["q_weight"],
                              k_weight=v["k_weight"], eps=EPS, interleaved=interleaved)


def _partner(z, r, interleaved):
    """The other value of each value's pair; those behind ``r`` have none."""
    t, rest = z[..., :r], torch.zeros_like(z[..., r:])
    if interleaved:
        t = t.unflatten(-1, (-1, 2)).flip(-1).flatten(-2)
    else:
        t = t.roll(r // 2, -1)
    return torch.cat((t, rest), -1)


def _exact(x, w, positions, inv_freq, interleaved):
    r = 2 * inv_freq.numel()
    z = x if w is None else x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w
    angle = (positions.double()[..., None] * inv_freq.double())[..., None, :]
    both = (lambda t: t.repeat_interleave(2, -1)) if interleaved else (lambda t: torch.cat((t, t), -1))
    cos, sin = both(angle.cos()), both(angle.sin())
    sign = torch.ones(r, device=x.device, dtype=torch.float64)
    if interleaved:
        sign[0::2] = -1
    else:
        sign[:r // 2] = -1
    y = z[..., :r] * cos + _partner(z, r, interleaved)[..., :r] * sin * sign
    return torch.cat((y, z[..., r:]), -1), z


def _within(name, got, want, dt, mag):
    assert got.dtype == dt, name
    err = (got.double() - want).abs()
    bound = U[dt] * (want.abs() + mag) + mag + TINY[dt]
    assert bool((err <= bound).all()), (name, float((err / bound).max()))


def _check(v, positions, inv_freq, outs, interleaved=False):
    leaves = {k: None if t is None else t.detach().requires_grad_(True) for k, t in v.items()}
    got = _call(leaves, positions, inv_freq, interleaved)
    names = [k for k in v if v[k] is not None]
    grads = dict(zip(names, torch.autograd.grad(got, [leaves[k] for k in names], outs)))
    d, r = v["q"].shape[-1], 2 * inv_freq.numel()
    rel = 2.0 ** -24 * (d / 16 + 24)
    for i, name in enumerate(("q", "k")):
        x = v[name].double().requires_grad_(True)
        w = v[name + "_weight"]
        wd = None if w is None else w.double().requires_grad_(True)
        y, z = _exact(x, wd, positions, inv_freq, interleaved)
        z = z.detach()
        _within(name, got[i].detach(), y.detach(), v[name].dtype,
                rel * (z.abs() + _partner(z, r, interleaved).abs()))
        dy = outs[i].double()
        want = torch.autograd.grad(y, [x] if w is None else [x, wd], dy)
        g = dy.abs() + _partner(dy, r, interleaved).abs()
        if w is None:
            _within("d_" + name, grads[name], want[0], v[name].dtype, rel * g)
            continue
        s = 1 / (x.detach().pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        hat = x.detach().abs() * s
        gw = g * wd.detach().abs()
        _within("d_" + name, grads[name], want[0], v[name].dtype,
                2 * rel * s * (gw + hat * (gw * hat).mean(-1, keepdim=True)))
        rows = x.numel() // d
        total = (g * hat).reshape(-1, d).sum(0)
        _within("d_%s_weight" % name, grads[name + "_weight"], want[1], w.dtype,
                (rel + 2.0 ** -24 * (32 + rows / 16)) * total)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt,wt", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                   (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
@pytest.mark.parametrize("lead,h,hk,d,r", [
    ((1,), 1, 1, 2, 2), ((1,), 32, 8, 128, 128), ((), 3, 2, 64, 32), ((7,), 5, 1, 72, 36), ((3, 50), 4, 2, 128, 64),
    ((2, 3, 33), 1, 1, 96, 96), ((130,), 3, 3, 20, 6), ((65,), 2, 1, 130, 130), ((40,), 2, 2, 256, 128),
    ((19,), 1, 2, 512, 512), ((21,), 1, 1, 510, 10), ((900,), 6, 2, 64, 64), ((5,), 40, 8, 80, 80),
    ((11,), 2, 1, 40, 16), ((2,), 71, 1, 64, 64)])
def test_sizes_and_types(gpu, lead, h, hk, d, r, dt, wt, interleaved):
    _check(*_make(gpu, lead, h, hk, d, r, dt, wt), interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("d,r", [(64, 64), (20, 10)])
def test_without_norms(gpu, norm, d, r):
    _check(*_make(gpu, (2, 45), 4, 1, d, r, torch.float32, torch.float32, norm, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("freq", [torch.float32, torch.float64])
@pytest.mark.parametrize("far", [10 ** 6, -10 ** 7, 2 ** 40])
def test_far_positions(gpu, far, freq):
    """Frequencies of powers of two make 2^40's products exact; its 2^-53 2^28 / (2 pi) turns of error in
    the reduction are far under the bound."""
    v, p, f, outs = _make(gpu, (77,), 2, 1, 64, 64, torch.float32, torch.float32, seed=2, far=far, freq=freq)
    if abs(far) > 2 ** 30:
        f = (2.0 ** -torch.arange(12, 44, device=gpu)).to(freq)
    _check(v, p, f, outs)


@pytest.mark.gpu
def test_positions_of_each_row_or_of_all(gpu):
    v, p, f, outs = _make(gpu, (3, 20), 4, 2, 64, 64, torch.bfloat16, torch.float32, seed=3)
    one = _call(v, p, f)
    for q in (p.expand(3, 20), p[None], p.int(), p[None].expand(3, 20).contiguous()):
        assert all(torch.equal(a, b) for a, b in zip(one, _call(v, q, f)))
    each = torch.randint(0, 1000, (3, 20), device=gpu)
    _check(v, each, f, outs)
    same = _call(v, torch.tensor(5, device=gpu), f)
    again = _call(v, torch.full((3, 20), 5, device=gpu), f)
    assert all(torch.equal(a, b) for a, b in zip(same, again))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fused", "heads_first", "odd", "negated", "strided_values"])
def test_strides_and_alignment(gpu, kind):
    v, p, f, outs = _make(gpu, (2, 30), 4, 2, 64, 64, torch.bfloat16, torch.float32, seed=4)
    w = dict(v)
    if kind == "fused":
        both = torch.cat((v["q"].flatten(2), v["k"].flatten(2), v["k"].flatten(2)), -1)
        w["q"], w["k"] = both[..., :256].unflatten(-1, (4, 64)), both[..., 256:384].unflatten(-1, (2, 64))
    elif kind == "heads_first":
        w["q"], w["k"] = (v[k].transpose(1, 2).contiguous().transpose(1, 2) for k in ("q", "k"))
    elif kind == "odd":
        def odd(t):
            wide = torch.zeros(*t.shape[:-1], 67, device=gpu, dtype=t.dtype)
            wide[..., 1:65] = t
            return wide[..., 1:65]
        w["q"], w["k"] = odd(v["q"]), odd(v["k"])
    elif kind == "negated":
        w["q"], w["k"] = torch._neg_view(-v["q"]), torch._neg_view(-v["k"])
        w["q_weight"] = torch._neg_view(-v["q_weight"])
    else:
        w["q"] = v["q"].repeat_interleave(2, -1)[..., ::2]
    douts = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in outs]

    def run(x, o):
        leaves = {k: t.detach().requires_grad_(True) for k, t in x.items()}
        y = _call(leaves, p, f)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, list(leaves.values()), o))
    assert all(torch.equal(a, b) for a, b in zip(run(v, outs), run(w, douts)))


@pytest.mark.gpu
def test_as_many_heads_as_there_may_be(gpu):
    _check(*_make(gpu, (1,), 65536, 40000, 8, 8, torch.float32, torch.float32, seed=11))


@pytest.mark.gpu
def test_one_gradient_may_be_missing(gpu):
    v, p, f, outs = _make(gpu, (50,), 3, 2, 64, 64, torch.float32, torch.float32, seed=5)
    for i, (name, other) in enumerate((("q", "k"), ("k", "q"))):
        leaves = {k: t.clone().requires_grad_(True) for k, t in v.items()}
        _call(leaves, p, f)[i].backward(outs[i])
        full = {k: t.clone().requires_grad_(True) for k, t in v.items()}
        zero = [o if j == i else torch.zeros_like(o) for j, o in enumerate(outs)]
        torch.autograd.backward(_call(full, p, f), zero)
        for k in v:
            assert torch.equal(leaves[k].grad, full[k].grad)
        assert not bool(leaves[other].grad.any())


@pytest.mark.gpu
def test_wanted_gradients_only(gpu):
    v, p, f, outs = _make(gpu, (50,), 3, 2, 64, 64, torch.bfloat16, torch.float32, seed=6)
    full = {k: t.clone().requires_grad_(True) for k, t in v.items()}
    torch.autograd.backward(_call(full, p, f), outs)
    for want in v:
        leaves = {k: t.clone().requires_grad_(k == want) for k, t in v.items()}
        y = _call(leaves, p, f)
        live = [(a, o) for a, o in zip(y, outs) if a.requires_grad]
        torch.autograd.backward([a for a, _ in live], [o for _, o in live])
        assert all((leaves[k].grad is None) == (k != want) for k in v)
        assert torch.equal(leaves[want].grad, full[want].grad)


@pytest.mark.gpu
def test_no_tokens_zero_rows_and_no_numbers(gpu):
    v, p, f, outs = _make(gpu, (0, 4), 3, 2, 64, 64, torch.bfloat16, torch.float32)
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items()}
    y = _call(leaves, p, f)
    got = torch.autograd.grad(y, list(leaves.values()), outs)
    for a, t in zip(got, leaves.values()):
        assert a.shape == t.shape and not bool(a.any())
    v, p, f, outs = _make(gpu, (6,), 3, 2, 64, 64, torch.bfloat16, torch.float32, seed=7)
    v["q"][2] = 0
    _check(v, p, f, outs)
    clean = _call(v, p, f)[0]
    v["q"][3, 1] = float("nan")
    got = _call(v, p, f)[0]
    hit = torch.isnan(got).flatten(2).all(-1)
    assert hit[3, 1] and int(hit.sum()) == 1
    assert torch.equal(got[~hit], clean[~hit])


@pytest.mark.gpu
def test_same_bits_every_time_on_any_stream_and_in_a_graph(gpu):
    v, p, f, outs = _make(gpu, (4, 500), 6, 2, 64, 64, torch.bfloat16, torch.float32, seed=8)
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items()}

    def step():
        y = _call(leaves, p, f)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, list(leaves.values()), outs))
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
        new = _make(gpu, (4, 500), 6, 2, 64, 64, torch.bfloat16, torch.float32, seed=30 + seed)[0]
        with torch.no_grad():
            for k in leaves:
                leaves[k].copy_(new[k])
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))


@pytest.mark.gpu
def test_gradient_against_differences(gpu):
    v, p, f, outs = _make(gpu, (33,), 2, 1, 64, 48, torch.float32, torch.float32, seed=9)
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items()}
    got = torch.autograd.grad(_call(leaves, p, f), list(leaves.values()), outs)
    step = {k: g.double() / g.double().norm() for k, g in zip(v, got)}

    def value(e):
        x = {k: t.double() + e * step[k] for k, t in v.items()}
        return sum(float((_exact(x[n], x[n + "_weight"], p, f, False)[0] * o.double()).sum())
                   for n, o in zip(("q", "k"), outs))
    slope = (value(1e-5) - value(-1e-5)) / 2e-5
    along = sum(float((g.double() * step[k]).sum()) for k, g in zip(v, got))
    size = sum(float((g.double() * step[k]).abs().sum()) for k, g in zip(v, got))
    assert abs(along - slope) <= 2.0 ** -18 * size + 1e-6 * abs(slope)


@pytest.mark.gpu
def test_no_second_gradient(gpu):
    v, p, f, outs = _make(gpu, (5,), 2, 1, 64, 48, torch.float32, torch.float32)
    v["q"].requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        torch.autograd.grad(_call(v, p, f)[0], v["q"], outs[0], create_graph=True)


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
@pytest.mark.parametrize("which", ["q", "k", "q_weight", "k_weight", "positions", "inv_freq"])
def test_tensors_without_memory_are_refused(gpu, which):
    v, p, f, _ = _make(gpu, (5,), 2, 1, 64, 48, torch.float32, torch.float32)
    v.update(positions=p, inv_freq=f)
    v[which] = _Wrapped(v[which])
    with pytest.raises(RuntimeError, match="memory"):
        _call(v, v["positions"], v["inv_freq"])


@pytest.mark.gpu
def test_operands_written_to_in_between_are_refused(gpu):
    v, p, f, outs = _make(gpu, (5,), 2, 1, 64, 48, torch.float32, torch.float32)
    for which in ("q", "q_weight", "positions"):
        leaves = {k: t.clone().requires_grad_(True) for k, t in v.items()}
        held = {k: t * 1 for k, t in leaves.items()}
        spots = p.clone()
        y = _call(held, spots, f)
        with torch.no_grad():
            (spots if which == "positions" else held[which]).mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.backward(y, outs)


def _refuse(match, *args, kind=ValueError, **kw):
    with pytest.raises(kind, match=match):
        dmuon.rotary_heads(*args, **kw)


def test_refusals_without_gpu():
    q, k, p, f, w = torch.zeros(2, 5, 4, 64), torch.zeros(2, 5, 2, 64), torch.arange(5), torch.ones(16), torch.ones(64)
    _refuse("do not fit", q, k[:1], p, f)
    _refuse("do not fit", q, k[..., :32], p, f)
    _refuse("do not fit", q[0, 0, 0], k[0, 0, 0], p, f)
    _refuse("dim must", q[..., :63], k[..., :63], p, f)
    _refuse("dim must", torch.zeros(1, 1, 514), torch.zeros(1, 1, 514), p[:1], f)
    _refuse("one dtype", q, k.half(), p, f)
    _refuse("one dtype", q.double(), k.double(), p, f)
    _refuse("positions must be integers", q, k, p.float(), f)
    for bad in (torch.arange(2), torch.zeros(2, 1).long(), torch.zeros(5, 2).long(), torch.arange(10),
                torch.zeros(3, 2, 5).long()):
        _refuse("do not fit the leading shape", q, k, bad, f)
    _refuse("inv_freq", q, k, p, f.half())
    _refuse("inv_freq", q, k, p, torch.ones(33))
    _refuse("inv_freq", q, k, p, f[:0])
    _refuse("inv_freq has no gradient", q, k, p, f.clone().requires_grad_(True))
    _refuse("q_weight must be", q, k, p, f, q_weight=w[:63])
    _refuse("k_weight must be", q.half(), k.half(), p, f, k_weight=w.bfloat16())
    _refuse("GPU", q, k, p, f, kind=RuntimeError)


def test_c_entry_refusals_without_gpu():
    import ctypes

    from dmuon_amd import _C
    lib, need = _C.lib(), ctypes.c_int64()
    good = dict(q=4096, k=4096, positions=4096, inv_freq=4096, q_weight=4096, k_weight=4096, q_out=4096,
                k_out=4096, dq_out=4096, dk_out=4096, dq=4096, dk=4096, d_q_weight=4096, d_k_weight=4096,
                tokens=30, period=10, heads=4, kv_heads=2, dim=64, rotary_dim=32, q_token=256, q_head=64,
                k_token=128, k_head=64, dq_out_token=256, dq_out_head=64, dk_out_token=128, dk_out_head=64,
                eps=1e-6, dtype=1)

    def says(rc, text):
        assert rc != 0 and text in lib.dmuon_last_error().decode()

    def args(**kw):
        return ctypes.byref(_C.RotaryHeadsArgs(**{**good, **kw}))

    size = lambda a: lib.dmuon_rotary_heads_grad_workspace_size(a, ctypes.byref(need))
    grad = lambda a: lib.dmuon_rotary_heads_grad(a, 4096, 1 << 40, None)
    assert size(args()) == 0 and need.value >= 2 * 64 * 4
    for fn in (lambda a: lib.dmuon_rotary_heads(a, None), size, grad):
        says(fn(args(dtype=3)), "dtype")
        says(fn(args(k_weight_dtype=7)), "dtype")
        says(fn(args(tokens=-1)), "tokens")
        says(fn(args(heads=0)), "heads")
        says(fn(args(dim=63)), "dim")
        says(fn(args(dim=514)), "dim")
        says(fn(args(rotary_dim=66)), "rotary_dim")
        says(fn(args(rotary_dim=0)), "rotary_dim")
        says(fn(args(period=7)), "positions")
        says(fn(args(inv_freq=None)), "NULL")
        says(fn(args(q=None)), "NULL")
    says(lib.dmuon_rotary_heads(args(k_out=None), None), "NULL")
    says(lib.dmuon_rotary_heads_grad(args(), 4096, 16, None), "workspace")
    says(lib.dmuon_rotary_heads_grad(args(), 4097, 1 << 40, None), "aligned")
    says(grad(args(q_weight=None)), "not there")


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_tangents_and_tracers_are_refused(dev):
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    v = [torch.ones(3, 2, 8, device=dev), torch.ones(3, 1, 8, device=dev), torch.ones(8, device=dev),
         torch.ones(8, device=dev)]
    p, f = torch.arange(3, device=dev), torch.ones(4, device=dev)

    def call(q, k, a, b):
        return dmuon.rotary_heads(q, k, p, f, q_weight=a, k_weight=b)
    for k in range(4):
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(t, t) if i == k else t for i, t in enumerate(v)]
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*dual)
    with pytest.raises(RuntimeError, match="tracer"):
        torch.jit.trace(call, tuple(v), check_trace=False)
    with pytest.raises(RuntimeError, match="tracer"):
        make_fx(call)(*v)


def _turns(positions, inv_freq):
    """cos and sin of the exact products, in 64 bits: whole numbers reduced by 2 pi to 300 bits (Machin)."""
    from fractions import Fraction
    bits = 300

    def arctan_of_inverse(n):
        total, term, k = 0, (1 << bits) // n, 0
        while term:
            total += (-term if k & 1 else term) // (2 * k + 1)
            term //= n * n
            k += 1
        return total
    turn = 8 * (4 * arctan_of_inverse(5) - arctan_of_inverse(239))         # 2 pi, times 2^bits
    angles = []
    for p in positions.tolist():
        for f in inv_freq.double().tolist():
            exact = Fraction(f) * p * (1 << bits)
            rest = (exact.numerator // exact.denominator) % turn
            angles.append((rest - turn if 2 * rest > turn else rest) / (1 << bits))
    angle = torch.tensor(angles, dtype=torch.float64).view(len(positions), -1).to(positions.device)
    return angle.cos(), angle.sin()


@pytest.mark.gpu
@pytest.mark.parametrize("freq", [torch.float32, torch.float64])
@pytest.mark.parametrize("far", [0, 2 ** 28, 2 ** 31, -2 ** 33, 2 ** 40, 2 ** 53 + 1, -2 ** 57 - 3, 2 ** 63 - 500, -2 ** 63])
def test_positions_of_any_size_with_any_frequencies(gpu, far, freq):
    """Angles of whole 64-bit positions and frequencies that are no powers of two, as exact as near ones:
    the bounds of near positions hold."""
    d, n = 64, 40
    gen = torch.Generator(device=gpu).manual_seed(20)
    q, k, dq, dk = (torch.randn(n, h, d, device=gpu, generator=gen) for h in (2, 1, 2, 1))
    positions = torch.arange(n, device=gpu) * 7 + far
    inv_freq = (10000.0 ** (-torch.arange(d // 2, device=gpu, dtype=torch.float64) * 2 / d)).to(freq)
    inv_freq[-3:] = torch.tensor([1.7, 0.0, -0.31], device=gpu)
    cos, sin = (t[:, None] for t in _turns(positions, inv_freq))
    leaves = [t.clone().requires_grad_(True) for t in (q, k)]
    got = dmuon.rotary_heads(*leaves, positions, inv_freq)
    grads = torch.autograd.grad(got, leaves, (dq, dk))
    rel = 2.0 ** -24 * (d / 16 + 24)
    for x, y, sign in ((q, got[0], 1), (k, got[1], 1), (dq, grads[0], -1), (dk, grads[1], -1)):
        a, b = x.double().chunk(2, -1)
        want = torch.cat((a * cos - sign * b * sin, b * cos + sign * a * sin), -1)
        _within(f"{far}", y.detach(), want, torch.float32, rel * (a.abs() + b.abs()).repeat(1, 1, 2))
