"""``attention`` against its definition in 64 bits.

Bounds, with u the rounding of the type (2^-8 bf16, 2^-11 fp16: half a step) and S the scores. A score is
an fp32 sum of ``dim`` exact products and its exponent a few roundings more, so a probability is off by
at most ``E = 2^-24 (dim + 8) scale max|q||k| + 2^-22 (|lse| + 4)`` relatively (``lse`` in powers of
two). A probability rounds once more (u) before it meets v, and the result rounds to the type:

    |out - exact| <= u |out| + (P |v|) (u + 2 E + n 2^-24),   n keys
    |dv - exact| <= u |dv| + (P^T |do|) (u + 2 E + n 2^-24),  n rows

The score's gradient dS = P (dP - delta) takes delta from the rounded out, so its error is
``e = P ((u + 2 E) |dP - delta| + 2^-24 dim |do||v| + |do| . bound(out))`` and dq, dk are off by
``scale e |k|``, ``scale e^T |q|`` plus their own rounding. fp16 holds P (at 1 or more for the largest of a
row, in the gradient times 2^10) and dS (times a power of two that brings 2 max|do| max|v| 2^10 to 2^14
or more) with absolute errors of 2^-25 where they are under the normal range.
"""
import math

import pytest
import torch

import dmuon_amd as dmuon

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
TYPES = [torch.bfloat16, torch.float16]


def _randn(gen, *shape):
    return torch.randn(*shape, device=gen.device, generator=gen)


def _make(dev, q_shape, k_shape, dt, seed=0, spread=1.0, do_scale=1.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    q, k = (spread * _randn(gen, *q_shape)).to(dt), _randn(gen, *k_shape).to(dt)
    v, do = _randn(gen, *k_shape).to(dt), (do_scale * _randn(gen, *q_shape)).to(dt)
    return q, k, v, do


def _one_head(q, k, v, do, scale, causal, window, peak):
    """[sq, d], [sk, d] in 64 bits: (out, dq, dk, dv) and their bounds without the result's rounding;
    ``peak``: 2 max|do| max|v| of the call for fp16, or None."""
    sq, sk, d = q.shape[0], k.shape[0], q.shape[1]
    u = U[torch.bfloat16] if peak is None else U[torch.float16]
    at = torch.arange(sq, device=q.device)[:, None] + sk - sq
    j = torch.arange(sk, device=q.device)[None]
    seen = torch.ones(sq, sk, dtype=torch.bool, device=q.device)
    if causal:
        seen = j <= at
        if window:
            seen &= j > at - window
    some = seen.any(1, keepdim=True)
    s = (q @ k.t()) * scale
    s = torch.where(seen, s, float("-inf"))
    lse = torch.where(some, torch.logsumexp(s, 1, keepdim=True), 0.0)
    p = torch.where(seen, (s - lse).exp(), 0.0)
    out = p @ v
    size = (q.abs() @ k.abs().t()).amax(1, keepdim=True) * scale if sk else torch.zeros_like(lse)
    err = 2.0 ** -24 * (d + 8) * size + 2.0 ** -22 * (lse.abs() / math.log(2) + 4)
    each = u + 2 * err + 2.0 ** -24 * sk
    b_out = (p @ v.abs()) * each
    if peak is not None:
        b_out = b_out + 2.0 ** -25 * torch.where(seen, 1.0, 0.0).to(v) @ v.abs()
    if do is None:
        return (out,), (b_out,)
    dp = do @ v.t()
    delta = (do * out).sum(1, keepdim=True)
    ds = p * (dp - delta)
    each_p = p * (u + 2 * err + 2.0 ** -24 * sq)
    b_ds = p * ((u + 2 * err) * (dp - delta).abs() + 2.0 ** -23 * d * (do.abs() @ v.abs().t()) +
                (do.abs() * (b_out + u * out.abs())).sum(1, keepdim=True)) + 2.0 ** -23 * (sq + sk) * ds.abs()
    if peak is not None:
        each_p = each_p + 2.0 ** -35 * seen
        b_ds = b_ds + 2.0 ** -39 * peak * seen
    return ((out, scale * ds @ k, scale * ds.t() @ q, p.t() @ do),
            (b_out, scale * b_ds @ k.abs(), scale * b_ds.t() @ q.abs(), each_p.t() @ do.abs()))


def _within(name, got, want, bound, dt):
    assert got.dtype == dt, name
    err = (got.double() - want).abs()
    bound = U[dt] * (want.abs() + bound) + bound + TINY[dt]
    # what lies half a step or more past the type's largest value rounds to infinity (fp16: 65520)
    over = torch.finfo(dt).max * (1 + U[dt] / 2) <= want.abs() + bound
    fine = (err <= bound) | (over & torch.isinf(got) & (got.sign() == want.sign()))
    assert bool(fine.all()), (name, float((err / bound)[~fine].max()))


def _check(got, spans, q, k, v, do, causal, window, scale=None):
    """``got``: out or (out, dq, dk, dv). ``spans``: index pairs (queries', keys') of the sequences, whose
    tensors are then [tokens, heads, dim]; what lies in none of them is 0."""
    dt, d = q.dtype, q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    group = q.shape[-2] // k.shape[-2]
    full = len(got) == 4
    where = [q, q, k, v] if full else [q]
    want = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in where]
    bound = [torch.zeros_like(t) for t in want]
    peak = None
    if dt == torch.float16:
        peak = 2 * float(do.double().norm(dim=-1).max() * v.double().norm(dim=-1).nan_to_num(0).max()) \
            if full and do.numel() and v.numel() else 0.0
    for mine, theirs in spans:
        for h in range(q.shape[-2]):
            one = _one_head(q[mine][:, h].double(), k[theirs][:, h // group].double(),
                            v[theirs][:, h // group].double(), do[mine][:, h].double() if full else None,
                            scale, causal, window, peak)
            for i, (value, b) in enumerate(zip(*one)):
                at, hh = (mine, h) if i < 2 else (theirs, h // group)
                if value.numel():
                    want[i][at][:, hh] += value
                    bound[i][at][:, hh] += b
    for name, g, w, b in zip(("out", "dq", "dk", "dv"), got, want, bound):
        _within(name, g.detach(), w, b, dt)


def _grads(q, k, v, do, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = dmuon.attention(*leaves, **kw)
    return (out.detach(), *torch.autograd.grad(out, leaves, do))


SHAPES = [  # batch, tokens, keys, heads, key heads, dim, causal, window
    (1, 1, 1, 1, 1, 8, True, None), (2, 1, 77, 4, 2, 64, True, None), (1, 33, 33, 3, 1, 40, False, None),
    (2, 130, 130, 4, 4, 128, True, None), (1, 65, 257, 6, 2, 72, True, None),
    (1, 257, 65, 2, 1, 128, True, None), (1, 300, 300, 8, 2, 64, True, 37), (1, 64, 1000, 2, 2, 96, False, None),
    (1, 5, 2100, 8, 1, 128, True, None), (3, 70, 70, 2, 1, 16, True, 1), (1, 128, 128, 1, 1, 128, False, None),
    (1, 200, 450, 5, 1, 120, True, 64), (1, 1, 3000, 12, 2, 56, True, 500), (2, 64, 64, 7, 7, 64, True, 1000),
    (1, 500, 1, 3, 3, 32, True, None), (2, 40, 40, 71, 1, 64, True, None), (1, 70, 90, 130, 1, 128, True, 33),
    (1, 150, 150, 96, 1, 24, False, None), (2, 1, 400, 64, 1, 64, True, None), (3, 300, 40, 33, 3, 64, True, None), (1, 129, 640, 4, 2, 128, True, 128), (1, 700, 700, 2, 2, 128, True, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("b,sq,sk,h,hk,d,causal,window", SHAPES)
def test_shapes(gpu, b, sq, sk, h, hk, d, causal, window, dt):
    q, k, v, do = _make(gpu, (b, sq, h, d), (b, sk, hk, d), dt)
    got = _grads(q, k, v, do, causal=causal, window=window)
    _check(got, [(i, i) for i in range(b)], q, k, v, do, causal, window)
    with torch.no_grad():
        assert torch.equal(dmuon.attention(q, k, v, causal=causal, window=window), got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("do_scale", [1e-6, 1.0, 3000.0])
@pytest.mark.parametrize("spread,scale", [(8.0, None), (1.0, 3.0), (0.01, 0.125)])
def test_sizes_of_values(gpu, dt, do_scale, spread, scale):
    """Sharp and flat rows; gradients far under and over 1, as a loss scale makes them."""
    q, k, v, do = _make(gpu, (1, 150, 4, 64), (1, 340, 2, 64), dt, 1, spread, do_scale)
    got = _grads(q, k, v, do, scale=scale)
    _check(got, [(0, 0)], q, k, v, do, True, None, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("sq,causal,window", [(1, True, None), (3, True, 90), (40, True, None), (9, False, None)])
def test_key_lengths(gpu, dt, sq, causal, window):
    """Lengths of nothing, one, some and all; what lies behind them is no number and is not read."""
    b, sk, h, hk, d = 7, 333, 6, 2, 128
    q, k, v, do = _make(gpu, (b, sq, h, d), (b, sk, hk, d), dt, 2)
    lengths = torch.tensor([0, 1, 5, 64, 200, 333, 128], device=gpu)
    behind = torch.arange(sk, device=gpu)[None, :, None, None] >= lengths[:, None, None, None]
    kn, vn = k.masked_fill(behind, float("nan")), v.masked_fill(behind, float("inf"))
    got = _grads(q, kn, vn, do, causal=causal, window=window, kv_lengths=lengths)
    spans = [((i,), (i, slice(0, int(n)))) for i, n in enumerate(lengths)]
    _check(got, spans, q, k.masked_fill(behind, 0), v.masked_fill(behind, 0), do, causal, window)
    # held to the keys that are there; any integer type
    odd = torch.tensor([-3, 1, 5, 64, 200, 999, 128], device=gpu, dtype=torch.int32)
    with torch.no_grad():
        again = dmuon.attention(q, kn, vn, causal=causal, window=window, kv_lengths=odd)
    assert torch.equal(again, got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("causal,window", [(True, None), (True, 70), (False, None)])
@pytest.mark.parametrize("lead,tail", [(0, 0), (5, 9)])
def test_packed(gpu, dt, causal, window, lead, tail):
    lens = [1, 0, 130, 64, 3, 257, 0, 65]
    klens = [1, 4, 130, 60, 200, 257, 0, 64]
    starts = torch.tensor([lead] + lens, device=gpu).cumsum(0)
    kstarts = torch.tensor([lead] + klens, device=gpu).cumsum(0)
    n, m = int(starts[-1]) + tail, int(kstarts[-1]) + tail
    q, k, v, do = _make(gpu, (n, 6, 80), (m, 2, 80), dt, 3)
    for t, s in ((k, kstarts), (v, kstarts)):     # tokens in no sequence: no numbers
        t[:lead] = float("nan")
        t[int(s[-1]):] = float("nan")
    got = _grads(q, k, v, do, causal=causal, window=window, q_starts=starts, kv_starts=kstarts)
    spans = [(slice(int(a), int(b)), slice(int(c), int(e))) for a, b, c, e in
             zip(starts, starts[1:], kstarts, kstarts[1:])]
    _check(got, spans, q, k, v, do, causal, window)


@pytest.mark.gpu
def test_many_sequences(gpu):
    """More than one pass of the tables, most of one token."""
    gen = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 3, (2500,), generator=gen)
    lens[1200] = 300
    starts = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).to(gpu)
    n = int(starts[-1])
    q, k, v, do = _make(gpu, (n, 2, 64), (n, 1, 64), torch.bfloat16, 4)
    got = _grads(q, k, v, do, q_starts=starts, kv_starts=starts)
    for i in (0, 1, 599, 1199, 1200, 1201, 2499):
        span = slice(int(starts[i]), int(starts[i + 1]))
        every = slice(0, span.stop - span.start)
        _check([t[span] for t in got], [(every, every)], q[span], k[span], v[span], do[span], True, None)


@pytest.mark.gpu
def test_starts_that_are_no_starts_stay_within_the_tokens(gpu):
    q, k, v, do = _make(gpu, (50, 2, 64), (70, 2, 64), torch.bfloat16, 5)
    starts = torch.tensor([-7, 20, 10, 1000], device=gpu)
    got = _grads(q, k, v, do, q_starts=starts, kv_starts=torch.tensor([3, -1, 40, 2 ** 40], device=gpu))
    spans = [(slice(0, 20), slice(3, 3)), (slice(20, 20), slice(3, 40)), (slice(20, 50), slice(40, 70))]
    _check(got, spans, q, k, v, do, True, None)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fused", "heads_first", "misaligned", "odd_rows", "expanded", "negated"])
def test_strides_and_alignment(gpu, kind):
    b, s, h, hk, d, dt = 2, 150, 4, 2, 64, torch.float16
    q, k, v, do = _make(gpu, (b, s, h, d), (b, s, hk, d), dt, 6)
    if kind == "fused":
        qkv = torch.cat([t.reshape(b, s, -1) for t in (q, k, v)], -1)
        lq, lk, lv = (t.unflatten(-1, (-1, d)) for t in qkv.split([h * d, hk * d, hk * d], -1))
    elif kind == "heads_first":
        lq, lk, lv = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    elif kind == "misaligned":
        def shift(t):
            flat = torch.empty(t.numel() + 1, device=gpu, dtype=dt)[1:]
            return flat.copy_(t.reshape(-1)).view(t.shape)
        lq, lk, lv = shift(q), shift(k), shift(v)
    elif kind == "odd_rows":
        def pad(t):
            wide = torch.zeros(*t.shape[:-1], d + 3, device=gpu, dtype=dt)
            wide[..., :d] = t
            return wide[..., :d]
        lq, lk, lv = pad(q), pad(k), pad(v)
    elif kind == "expanded":
        k, v = k[:, :, :1].expand(b, s, hk, d), v[:, :1].expand(b, s, hk, d)
        lq, lk, lv = q[:, :1].expand(b, s, h, d), k, v
        q = lq
    else:
        lq, lk, lv = (torch._neg_view(-t) for t in (q, k, v))
    dos = torch.empty(b, h, s, d, device=gpu, dtype=dt).copy_(do.transpose(1, 2)).transpose(1, 2)
    want = _grads(q.contiguous(), k.contiguous(), v.contiguous(), do)
    got = _grads(lq, lk, lv, dos)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu):
    """A cache whose last tokens lie more than 2^32 bytes behind its first ones."""
    sk, d, dt = 70001, 64, torch.bfloat16
    room = torch.empty(2, sk, 16384, device=gpu, dtype=dt)       # 2.3 GB a half
    q, k, v, do = _make(gpu, (2, 40, 4, d), (2, sk, 1, d), dt, 7)
    far = [room[:, :, i * d:(i + 1) * d].unsqueeze(2) for i in (0, 250)]
    for t, s in zip(far, (k, v)):
        t.copy_(s)
    want, got = _grads(q, k, v, do), _grads(q, *far, do)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
def test_nothing_to_see_and_nothing_to_do(gpu, dt):
    for b, sq, sk in ((2, 5, 0), (2, 0, 5), (0, 5, 5), (1, 0, 0)):
        q, k, v, do = _make(gpu, (b, sq, 4, 64), (b, sk, 2, 64), dt)
        for t, like in zip(_grads(q, k, v, do), (q, q, k, v)):
            assert t.shape == like.shape and not bool(t.any())
    q, k, v, do = _make(gpu, (6, 2, 64), (9, 2, 64), dt)
    none = torch.tensor([4], device=gpu)
    for t, like in zip(_grads(q, k, v, do, q_starts=none, kv_starts=none), (q, q, k, v)):
        assert t.shape == like.shape and not bool(t.any())


@pytest.mark.gpu
def test_wanted_gradients_only(gpu):
    q, k, v, do = _make(gpu, (1, 100, 4, 64), (1, 100, 2, 64), torch.bfloat16, 8)
    want = _grads(q, k, v, do)[1:]
    for mask in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((q, k, v))]
        dmuon.attention(*leaves).backward(do)
        for i, t in enumerate(leaves):
            assert (t.grad is None) if not mask >> i & 1 else torch.equal(t.grad, want[i])


@pytest.mark.gpu
def test_gradient_against_differences(gpu):
    """A step along the gradient changes a 64-bit loss as much as the gradient says."""
    q, k, v, do = _make(gpu, (1, 37, 2, 64), (1, 53, 1, 64), torch.float16, 9)
    got = _grads(q, k, v, do)[1:]
    step = [t.double() / t.double().norm() for t in got]

    def value(e):
        x = [t[0].double() + e * s[0] for t, s in zip((q, k, v), step)]
        total = 0.0
        for h in range(2):
            out = _one_head(x[0][:, h], x[1][:, 0], x[2][:, 0], None, 0.125, True, None, None)[0][0]
            total += float((out * do[0, :, h].double()).sum())
        return total
    slope = (value(1e-4) - value(-1e-4)) / 2e-4
    along = sum(float((t.double() * s).sum()) for t, s in zip(got, step))
    # each gradient is within 2^-11 of its size of the formula's, and a few times that from P and dS
    assert abs(along - slope) <= 2.0 ** -8 * along


@pytest.mark.gpu
def test_same_bits_every_time_on_any_stream_and_in_a_graph(gpu):
    starts = torch.tensor([0, 70, 300, 431], device=gpu)
    for dt, kw, shapes in ((torch.float16, {}, ((2, 200, 4, 128), (2, 200, 2, 128))),
                           (torch.bfloat16, dict(q_starts=starts, kv_starts=starts),
                            ((431, 4, 64), (431, 2, 64))),
                           (torch.bfloat16, {}, ((1, 2, 8, 128), (1, 5000, 2, 128)))):
        q, k, v, do = _make(gpu, *shapes, dt, 10)
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]

        def step():
            out = dmuon.attention(*leaves, **kw)
            return (out.detach(), *torch.autograd.grad(out, leaves, do))
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
            new = _make(gpu, *shapes, dt, 30 + seed)
            with torch.no_grad():
                for leaf, t in zip(leaves, new):
                    leaf.copy_(t)
            want = step()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, held))


@pytest.mark.gpu
def test_calls_at_once(gpu):
    """Calls on two streams, with nothing between them: each has its own workspace."""
    sets = [_make(gpu, (1, 300, 8, 64), (1, 2000, 2, 64), torch.float16, 40 + i) for i in range(6)]
    want = [_grads(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i, s in enumerate(sets):
        with torch.cuda.stream(streams[i % 2]):
            got.append(_grads(*s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_a_cache_that_grows_under_a_graph(gpu):
    """One captured call of a decoding loop: the token, the cache and its lengths change between replays."""
    b, room, h, hk, d = 3, 200, 8, 2, 64
    q, k, v, _ = _make(gpu, (b, 1, h, d), (b, room, hk, d), torch.bfloat16, 50)
    lengths = torch.tensor([0, 63, 199], device=gpu)
    with torch.no_grad():
        dmuon.attention(q, k, v, kv_lengths=lengths)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = dmuon.attention(q, k, v, kv_lengths=lengths)
        for step in range(4):
            q.copy_(_make(gpu, (b, 1, h, d), (b, 1, hk, d), torch.bfloat16, 60 + step)[0])
            lengths += 1
            graph.replay()
            torch.cuda.synchronize()
            n = lengths.clamp(max=room).tolist()
            _check([held], [((i,), (i, slice(0, m))) for i, m in enumerate(n)], q, k, v, None, True, None)
            assert torch.equal(held, dmuon.attention(q, k, v, kv_lengths=lengths))


@pytest.mark.gpu
def test_a_kept_graph_gives_its_gradients_again(gpu):
    q, k, v, do = _make(gpu, (1, 90, 4, 64), (1, 90, 2, 64), torch.float16, 51)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = dmuon.attention(*leaves)
    first = torch.autograd.grad(out, leaves, do, retain_graph=True)
    # a sum's gradient is one value seen everywhere
    torch.autograd.grad(out.sum(), leaves, retain_graph=True)
    again = torch.autograd.grad(out, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    ones = _grads(q, k, v, torch.ones_like(do))
    seen = [t.clone().requires_grad_(True) for t in (q, k, v)]
    total = torch.autograd.grad(dmuon.attention(*seen).sum(), seen)
    assert all(torch.equal(a, b) for a, b in zip(total, ones[1:]))


@pytest.mark.gpu
def test_one_tensor_in_all_places(gpu):
    x, _, _, do = _make(gpu, (1, 70, 2, 64), (1, 70, 2, 64), torch.bfloat16, 52)
    one = x.clone().requires_grad_(True)
    (got,) = torch.autograd.grad(dmuon.attention(one, one, one), one, do)
    parts = _grads(x, x, x, do)[1:]
    assert torch.equal(got, parts[0] + parts[1] + parts[2]) or \
        torch.equal(got, parts[2] + parts[1] + parts[0]) or torch.equal(got, parts[0] + parts[2] + parts[1])


@pytest.mark.gpu
def test_operands_written_to_in_between_are_refused(gpu):
    q, k, v, do = _make(gpu, (1, 10, 2, 64), (1, 10, 2, 64), torch.bfloat16)
    for i in range(3):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        held = [t * 1 for t in leaves]
        out = dmuon.attention(*held)
        with torch.no_grad():
            held[i].mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            out.backward(do)


@pytest.mark.gpu
def test_no_second_gradient(gpu):
    q, k, v, do = _make(gpu, (1, 10, 2, 64), (1, 10, 2, 64), torch.bfloat16)
    q.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        torch.autograd.grad(dmuon.attention(q, k, v), q, do, create_graph=True)


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
@pytest.mark.parametrize("which", range(4))
def test_tensors_without_memory_are_refused(gpu, which):
    q, k, v, _ = _make(gpu, (1, 10, 2, 64), (1, 10, 2, 64), torch.bfloat16)
    ops = [q, k, v, torch.tensor([7], device=gpu)]
    ops[which] = _Wrapped(ops[which])
    with pytest.raises(RuntimeError, match="memory"):
        dmuon.attention(*ops[:3], kv_lengths=ops[3])


def _refuse(match, *args, kind=ValueError, **kw):
    with pytest.raises(kind, match=match):
        dmuon.attention(*args, **kw)


def test_refusals_without_gpu():
    q, k = torch.zeros(2, 3, 4, 64).bfloat16(), torch.zeros(2, 5, 2, 64).bfloat16()
    n, s = torch.tensor([1, 2]), torch.tensor([0, 2])
    _refuse("do not fit", q[0], k, k)
    _refuse("do not fit", q, k, k[:, :4])
    _refuse("do not fit", q, k[:1], k[:1])
    _refuse("do not fit", q, k, k, q_starts=s, kv_starts=s)
    _refuse("do not fit", q[..., :32], k, k)
    _refuse("dim must", q[..., :60], k[..., :60], k[..., :60])
    _refuse("dim must", torch.zeros(1, 1, 1, 136), torch.zeros(1, 1, 1, 136), torch.zeros(1, 1, 1, 136))
    _refuse("multiple of kv_heads", q[:, :, :3], k, k)
    _refuse("bfloat16 or float16", q.float(), k.float(), k.float())
    _refuse("bfloat16 or float16", q, k.half(), k)
    _refuse("window", q, k, k, window=0)
    _refuse("window", q, k, k, causal=False, window=4)
    for bad in (0.0, -1.0, float("inf"), float("nan"), 1e39, 1e-39):
        _refuse("scale", q, k, k, scale=bad)
    _refuse("come together", q[0], k[0], k[0], q_starts=s)
    _refuse("not packed", q[0], k[0], k[0], q_starts=s, kv_starts=s, kv_lengths=n)
    _refuse("GPU", q, k, k, kind=RuntimeError)


@pytest.mark.gpu
def test_refusals_of_lengths_and_starts(gpu):
    q, k, v, _ = _make(gpu, (2, 3, 4, 64), (2, 5, 2, 64), torch.bfloat16)
    _refuse("kv_lengths must be integers", q, k, v, kv_lengths=torch.ones(2, device=gpu))
    _refuse("kv_lengths must have", q, k, v, kv_lengths=torch.ones(3, device=gpu, dtype=torch.long))
    _refuse("kv_lengths must live", q, k, v, kv_lengths=torch.ones(2, dtype=torch.long), kind=RuntimeError)
    s = torch.tensor([0, 3], device=gpu)
    _refuse("kv_starts must have", q[0], k[0], v[0], q_starts=s, kv_starts=s[:1])
    _refuse("q_starts must have", q[0], k[0], v[0], q_starts=s[:0], kv_starts=s[:0])


def test_c_entry_refusals_without_gpu():
    import ctypes

    from dmuon_amd import _C
    lib, need = _C.lib(), ctypes.c_int64()
    good = dict(q=4096, k=4096, v=4096, out=4096, rest=4096, lse=4096, dout=4096, dq=4096, dk=4096, dv=4096,
                batch=2, q_len=40, kv_len=50, heads=4, kv_heads=2, dim=64, q_batch=40 * 256, q_token=256,
                q_head=64, k_batch=50 * 128, k_token=128, k_head=64, v_batch=50 * 128, v_token=128,
                v_head=64, do_batch=40 * 256, do_token=256, do_head=64, scale=0.125, causal=1, dtype=1)

    def says(rc, text):
        assert rc != 0 and text in lib.dmuon_last_error().decode()

    def args(**kw):
        return ctypes.byref(_C.AttentionArgs(**{**good, **kw}))

    forward = lambda a: lib.dmuon_attention(a, None, 0, None)
    size = lambda a: lib.dmuon_attention_workspace_size(a, ctypes.byref(need))
    grad_size = lambda a: lib.dmuon_attention_grad_workspace_size(a, ctypes.byref(need))
    grad = lambda a: lib.dmuon_attention_grad(a, 4096, 1 << 40, None)
    assert size(args()) == 0 and grad_size(args()) == 0 and need.value >= 40 * 2 * 4 * 4
    for fn in (forward, size, grad_size, grad):
        says(fn(args(dtype=0)), "dtype")
        says(fn(args(dim=60)), "dim")
        says(fn(args(dim=256)), "dim")
        says(fn(args(q_len=-1)), "lengths")
        says(fn(args(kv_len=1 << 31)), "lengths")
        says(fn(args(q_len=1 << 30)), "2^30")
        says(fn(args(heads=5)), "multiple of kv_heads")
        says(fn(args(scale=0.0)), "scale")
        says(fn(args(scale=float("nan"))), "scale")
        says(fn(args(window=-1)), "window")
        says(fn(args(window=3, causal=0)), "window")
        says(fn(args(q_starts=4096)), "together")
        says(fn(args(q_starts=4096, kv_starts=4096, kv_lengths=4096)), "not packed")
        says(fn(args(k=None)), "NULL")
        says(fn(args(q=4104)), "aligned")
        says(fn(args(k_head=60)), "multiples of 8")
        says(fn(args(k_token=56)), "apart")
        says(fn(args(v_token=1 << 25)), "apart")
        says(fn(args(q_token=1 << 25)), "span")
    says(forward(args(out=None)), "out is NULL")
    says(forward(args(kv_len=5000)), "workspace")
    says(lib.dmuon_attention_grad(args(), 4096, 16, None), "workspace")
    says(lib.dmuon_attention_grad(args(), 4097, 1 << 40, None), "aligned")
    says(grad(args(lse=None)), "lse")
    says(grad(args(dq=4104)), "aligned")
    says(grad(args(rest=4104)), "aligned")
    says(grad(args(do_head=4)), "multiples of 8")
    says(grad(args(do_token=1 << 25)), "span")


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_tangents_and_tracers_are_refused(dev):
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    v = [torch.ones(1, 3, 2, 64, device=dev).half() for _ in range(3)]
    for k in range(3):
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(t, t) if i == k else t for i, t in enumerate(v)]
            with pytest.raises(RuntimeError, match="forward-mode"):
                dmuon.attention(*dual)
    with pytest.raises(RuntimeError, match="tracer"):
        torch.jit.trace(lambda *x: dmuon.attention(*x), tuple(v), check_trace=False)
    with pytest.raises(RuntimeError, match="tracer"):
        make_fx(lambda *x: dmuon.attention(*x))(*v)


def _own_peaks(q, k, v, do, causal):
    """[tokens, heads, dim] of one sequence as many heads as key heads in fp16, where dS is held times a power
    of two of its own for each row (dq) and each key (dk): (dq, dk) and their bounds. A row's (a key's) dS is at
    most ``2 |do| max|v|`` over what it has to do with, and is held with an absolute error of at most 2^-38 of
    its largest one (2^-25 under the normal range, where the largest has reached 2^13)."""
    d, scale, u = q.shape[-1], q.shape[-1] ** -0.5, U[torch.float16]
    want, bound = ([], []), ([], [])
    for h in range(q.shape[1]):
        x = [t[:, h].double() for t in (q, k, v, do)]
        (_, dq, dk, _), (_, bq, bk, _) = _one_head(*x, scale, causal, None, 0.0)
        seen = torch.ones(q.shape[0], k.shape[0], dtype=torch.bool, device=q.device)
        if causal:
            seen = seen.tril(k.shape[0] - q.shape[0])
        most = seen * (2 * x[3].norm(dim=1)[:, None] * x[2].norm(dim=1).max())
        bq = bq + scale * 2.0 ** -38 * (most.amax(1, keepdim=True) * (seen.double() @ x[1].abs()))
        bk = bk + scale * 2.0 ** -38 * (most.amax(0)[:, None] * (seen.double().t() @ x[0].abs()))
        for pair, add in ((want, (dq, dk)), (bound, (bq, bk))):
            for to, t in zip(pair, add):
                to.append(t)
    return tuple(tuple(torch.stack(t, 1) for t in pair) for pair in (want, bound))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("packed", [True, False])
def test_gradients_of_one_sequence_do_not_depend_on_another(gpu, packed, d):
    """fp16 gradients 2^24 apart, as of losses that are averaged over documents of very different lengths."""
    n, dt = 200, torch.float16
    q, k, v, do = _make(gpu, (2, n, 2, d), (2, n, 2, d), dt, 70)
    do[0] *= 4096
    do[1] *= 2.0 ** -12
    kw = {}
    if packed:
        q, k, v, do = (t.flatten(0, 1) for t in (q, k, v, do))
        kw = {"q_starts": torch.tensor([0, n, 2 * n], device=gpu)}
        kw["kv_starts"] = kw["q_starts"]
    halves = lambda t: t.reshape(2, n, 2, d)
    got = [halves(t) for t in _grads(q, k, v, do, **kw)]
    for i in range(2):
        want, bound = _own_peaks(*(halves(t)[i] for t in (q, k, v, do)), True)
        for name, g, w, b in zip(("dq", "dk"), got[1:], want, bound):
            _within(f"{name} of sequence {i}", g[i], w, b, dt)
    # the first one's values and gradients are nothing to the second one
    first = slice(0, n) if packed else 0
    other_v, other_do = v.clone(), do.clone()
    other_v[first] *= 16
    other_do[first] = 0
    again = [halves(t) for t in _grads(q, k, other_v, other_do, **kw)]
    assert all(torch.equal(a[1], b[1]) for a, b in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("which", ["early", "late", "every_other", "rising"])
def test_gradients_of_rows_of_very_different_sizes(gpu, which, d):
    """A row's dq and the dk of keys that only small rows see keep their own accuracy in fp16."""
    n, dt = 330, torch.float16
    q, k, v, do = _make(gpu, (1, n, 2, d), (1, n, 2, d), dt, 71)
    at = torch.arange(n, device=gpu)
    small = {"early": at < n // 2, "late": at >= n // 2, "every_other": at % 2 == 1}.get(which)
    size = torch.where(small, 2.0 ** -12, 4096.0) if small is not None else 2.0 ** (-12 + 24 * at / n).floor()
    do *= size[None, :, None, None].to(dt)
    got = _grads(q, k, v, do)
    want, bound = _own_peaks(q[0], k[0], v[0], do[0], True)
    for name, g, w, b in zip(("dq", "dk"), got[1:], want, bound):
        _within(name, g[0], w, b, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("sq,sk,h,hk,d", [(1, 40, 2, 1, 64), (1, 5000, 8, 2, 128), (100, 300, 2, 2, 128),
                                          (100, 5000, 4, 1, 64), (70, 70, 1, 1, 72)])
def test_scores_of_minus_infinity(gpu, sq, sk, h, hk, d, dt):
    """A key whose score is minus infinity has no share; a row that sees only such keys has no numbers, as
    the formula has it, and is not one that sees nothing."""
    q, k, v, do = _make(gpu, (1, sq, h, d), (1, sk, hk, d), dt, 72)
    q[..., 0] = -q[..., 0].abs() - 1
    k[..., 0] = float("inf")
    got = _grads(q, k, v, do, causal=False)
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        assert bool(torch.isnan(t).all()), name
    # one key of numbers among them takes the whole row, wherever it stands
    for one in (0, sk // 2, sk - 1):
        single = k.clone()
        single[:, one, :, 0] = 1
        with torch.no_grad():
            out = dmuon.attention(q, single, v, causal=False)
        assert torch.equal(out, v[:, one, None].repeat_interleave(h // hk, 2).expand_as(out))


@pytest.mark.gpu
def test_rows_of_minus_infinity_beside_others(gpu):
    """Under a causal mask, lengths and starts: rows that see nothing are 0 and have no gradient, rows that
    see only minus infinities are no numbers, the others are as without those keys."""
    d, dt = 64, torch.bfloat16
    q, k, v, do = _make(gpu, (3, 50, 2, d), (3, 40, 2, d), dt, 73)
    q[..., 0] = -q[..., 0].abs() - 1
    k[:, :8, :, 0] = float("inf")
    lengths = torch.tensor([40, 0, 40], device=gpu)
    # query i sees the keys up to i - 10; those of the second sequence see none
    got = _grads(q, k, v, do, kv_lengths=lengths)
    for b in (0, 2):
        out, dv = got[0][b], got[3][b]
        assert not bool(out[:10].any()) and bool(torch.isnan(out[10:18]).all())
        assert bool(torch.isfinite(out[18:]).all())
        assert bool(torch.isnan(dv[:8]).all()) and bool(torch.isfinite(dv[8:]).all())
        assert not bool(got[1][b][:10, :, 1:].any())           # (a key's infinity may reach rows near its own)
        want = _one_head(q[b, 18:, 0].double(), k[b, 8:, 0].double(), v[b, 8:, 0].double(), None, d ** -0.5, True,
                         None, None)
        _within("out", out[18:, 0], want[0][0], want[1][0], dt)
    assert all(not bool(t[1].any()) for t in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 40)])
def test_waves_of_none_to_several_tiles(gpu, dt, d):
    """Single tokens whose waves have no, one, two and more tiles of keys, whole ones and ends."""
    lens = [0, 1, 31, 32, 33, 64, 65, 96, 1000, 1024, 1025, 2047, 2048, 2080, 3071, 4000]
    b = len(lens)
    for sk in (4000, 40000):              # few and many keys a wave
        q, k, v, _ = _make(gpu, (b, 1, 4, d), (b, sk, 2, d), dt, 76)
        lengths = torch.tensor(lens, device=gpu) * (sk // 4000)
        with torch.no_grad():
            got = dmuon.attention(q, k, v, kv_lengths=lengths)
        _check([got], [((i,), (i, slice(0, int(n)))) for i, n in enumerate(lengths)], q, k, v, None, True, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("sq,sk,h,hk", [(700, 700, 2, 2), (8, 512, 4, 1), (2, 4096, 8, 1), (60, 3000, 4, 1)])
def test_gradients_take_in_what_the_rounding_of_the_result_left(gpu, sq, sk, h, hk, dt):
    """delta = sum do o stands in every dS of a row. Keys and values with a large common part make its error
    show: the exact dS of a row add up to 0, so the keys' common part c drops out of dq, where an error e of
    delta stays as scale e c. With o rounded, its values of 8 .. 16 are off by up to half a step, of even
    spread: e of sqrt(d) half / sqrt(3) on average, for dout of size 1. What else there is: P in o is
    rounded, by up to u of each term, which moves a row's values together by 8 u sqrt(sum P^2 / 3), e by sqrt(d)
    times that, for rows of some hundred keys a twentieth of the former; dS is rounded, u of terms that
    are as small as P |v - o|, and dq itself. A quarter holds all of these."""
    d, common = 128, 4.0
    q, k, v, do = _make(gpu, (1, sq, h, d), (1, sk, hk, d), dt, 75)
    q, k, v = (0.25 * q.float()).to(dt), (common + 0.3 * k.float()).to(dt), (10 + 0.5 * v.float()).to(dt)
    dq = _grads(q, k, v, do)[1][0].double()
    rows = slice(0, sq) if sq + 400 < sk else slice(400, sq)          # rows that see some hundred keys
    errors = []
    for i in range(h):
        at = i * hk // h
        want = _one_head(q[0, :, i].double(), k[0, :, at].double(), v[0, :, at].double(), do[0, :, i].double(),
                         d ** -0.5, True, None, None)[0][1]
        errors.append((dq[:, i] - want)[rows])
    rms = float(torch.stack(errors).pow(2).mean().sqrt())
    half = 8 * U[dt]                      # half a step of values of 8 .. 16
    assert rms <= 0.25 * d ** -0.5 * common * d ** 0.5 * half / 3 ** 0.5, rms


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_gradients_of_rows_that_see_nothing_are_not_read(gpu, dt, bad):
    """Queries before the first key, of an empty cache and outside of the sequences: whatever their gradient
    and they themselves hold."""
    q, k, v, do = _make(gpu, (2, 90, 6, 64), (2, 40, 2, 64), dt, 74)
    lengths = torch.tensor([40, 0], device=gpu)
    # sequence 0: queries under 50; sequence 1: all
    blind = torch.ones(2, 90, dtype=torch.bool, device=gpu)
    blind[0, 50:] = False
    for window in (None, 30):
        want = _grads(q, k, v, do.masked_fill(blind[..., None, None], 0), kv_lengths=lengths, window=window)
        no_q, no_do = (t.masked_fill(blind[..., None, None], bad) for t in (q, do))
        got = _grads(no_q, k, v, no_do, kv_lengths=lengths, window=window)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    starts, kstarts = torch.tensor([30, 90, 150], device=gpu), torch.tensor([5, 25, 75], device=gpu)
    flat = [t.flatten(0, 1) for t in (q, k, v, do)]
    at = torch.arange(180, device=gpu)
    # sequence 0: 60 queries of 20 keys; sequence 1: 60 of 50
    blind = ((at < 70) | ((at >= 90) & (at < 100)) | (at >= 150))[:, None, None]
    kw = {"q_starts": starts, "kv_starts": kstarts}
    want = _grads(*flat[:3], flat[3].masked_fill(blind, 0), **kw)
    got = _grads(flat[0].masked_fill(blind, bad), *flat[1:3], flat[3].masked_fill(blind, bad), **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_c_entry_refuses_scales_that_leave_fp32():
    """The kernels multiply scores by scale log2(e) in fp32."""
    import ctypes

    from dmuon_amd import _C
    lib, need = _C.lib(), ctypes.c_int64()
    good = dict(q=4096, k=4096, v=4096, batch=1, q_len=4, kv_len=4, heads=1, kv_heads=1, dim=64, q_batch=256,
                q_token=64, q_head=64, k_batch=256, k_token=64, k_head=64, v_batch=256, v_token=64, v_head=64,
                causal=1, dtype=1)

    def size(scale):
        return lib.dmuon_attention_workspace_size(ctypes.byref(_C.AttentionArgs(**good, scale=scale)),
                                                  ctypes.byref(need))
    assert size(2.0 ** -126) == 0 and size(2.0 ** 126) == 0
    for bad in (2.0 ** -127, 3e38, float("inf")):
        assert size(bad) != 0 and "scale" in lib.dmuon_last_error().decode()
