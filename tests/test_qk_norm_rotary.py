"""Norms of queries and keys for each head with the position rotation in the same pass: values and all gradients
against the formula in float64, over types, sizes, pairings, axes and kinds of positions, strided and unaligned
arrays; against differences; far positions; streams and captured graphs; and the refusals.

Tolerances are bounds on each value. With u the type's unit roundoff, e = 2^-24 and t the error of a cosine or sine
(2^-20 for 16-bit results, 2^-22 for float32, the angle's own rounding in it): r = 1 / sqrt(mean + eps) is off by
(dim + 8) e of itself, a turned value by u of itself and ((dim + 12) e + t) of the magnitudes of its pair; dx likewise
with the two terms it is made of; a weight's gradient by ((dim + rows + 12) e + t) of its terms' magnitudes."""

import decimal
import math

import pytest
import torch

from spectral import native
from spectral.nn import qk_norm_rotary

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
E = 2.0 ** -24


def turn_by(t, positions, rotated, pairs, theta, sign=1.0):
    """The rotation, in the type of t (64 bits)."""
    if positions is None or rotated == 0:
        return t
    axes = positions.shape[-1]
    span, n, out = rotated // axes, rotated // axes // 2, t.clone()
    for a in range(axes):
        angle = positions[..., a, None].double() * theta ** (-torch.arange(n, device=t.device).double() / n)
        c, s = torch.cos(angle).unsqueeze(-2), sign * torch.sin(angle).unsqueeze(-2)
        one = slice(a * span, a * span + n) if pairs == "halves" else slice(a * span, (a + 1) * span, 2)
        two = slice(a * span + n, (a + 1) * span) if pairs == "halves" else slice(a * span + 1, (a + 1) * span, 2)
        out[..., one] = t[..., one] * c - t[..., two] * s
        out[..., two] = t[..., one] * s + t[..., two] * c
    return out


def spread(t, positions, rotated, pairs):
    """For each value the magnitudes of its pair."""
    if positions is None or rotated == 0:
        return t.abs()
    axes, out = positions.shape[-1], t.abs().clone()
    span, n = rotated // axes, rotated // axes // 2
    for a in range(axes):
        one = slice(a * span, a * span + n) if pairs == "halves" else slice(a * span, (a + 1) * span, 2)
        two = slice(a * span + n, (a + 1) * span) if pairs == "halves" else slice(a * span + 1, (a + 1) * span, 2)
        both = t[..., one].abs() + t[..., two].abs()
        out[..., one] = both
        out[..., two] = both
    return out


def formula(x, weight, positions, dy, rotated, pairs, theta, eps, dtype):
    """y, dx, dweight in float64, each with its bound."""
    x, dy = x.detach().double(), dy.detach().double()
    dim = x.shape[-1]
    w = torch.ones(dim, dtype=torch.float64, device=x.device) if weight is None else weight.detach().double()
    u, t = torch.finfo(dtype).eps / 2, 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -20
    least = 2.0 ** -25 if dtype == torch.float16 else 1e-38
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x * r * w
    y = turn_by(n, positions, rotated, pairs, theta)
    slack = (dim + 12) * E + t
    g = turn_by(dy, positions, rotated, pairs, theta, -1.0)
    ga = spread(dy, positions, rotated, pairs)
    dw = (g * x * r).sum((0, 1, 2))
    rows = x.shape[0] * x.shape[1] * x.shape[2]
    dw_e = ((slack + rows * E) * ga * x.abs() * r).sum((0, 1, 2)) + 1e-38
    mean = (g * w * x).mean(-1, keepdim=True)
    dx = r * (g * w - x * r * r * mean)
    parts = r * (ga * w.abs() + x.abs() * r * r * (ga * w.abs() * x.abs()).mean(-1, keepdim=True))
    return (y, u * y.abs() + slack * spread(n, positions, rotated, pairs) + least), (dx, u * dx.abs() + 3 * slack * parts + least), (dw, dw_e)


def within(got, want, name):
    value, bound = want
    assert got.shape == value.shape, name
    if got.numel():
        worst = float(((got.detach().double() - value).abs() / bound).max())
        assert worst <= 1.0, f"{name}: {worst:.3g} of the bound"


def place(kind, batch, tokens, axes, seed=0):
    g = torch.Generator().manual_seed(seed + tokens)
    if kind == "none":
        return None
    if kind == "float":
        return (200 * torch.rand(batch, tokens, axes, generator=g) - 50).cuda()
    if kind == "shared":
        return (200 * torch.rand(tokens, axes, generator=g)).cuda()
    p = torch.randint(-1000, 1 << 20, (batch, tokens, axes), generator=g)
    return p.cuda() if kind == "int64" else p.int().cuda()


def inputs(batch, tokens, heads, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 3 * tokens + dim)
    x, dy = (torch.randn(batch, tokens, heads, dim, generator=g).to(dtype).cuda() for _ in range(2))
    return x, (1 + 0.3 * torch.randn(dim, generator=g)).cuda(), dy


def check(batch, queries, keys, heads, kv_heads, dim, axes, rotated, pairs, kind, dtype, weighted=True, theta=10000.0, eps=1e-6):
    q, wq, dq = inputs(batch, queries, heads, dim, dtype)
    k, wk, dk = inputs(batch, keys, kv_heads, dim, dtype, 1)
    if not weighted:
        wq = wk = None
    pq, pk = place(kind, batch, queries, axes), place(kind, batch, keys, axes, 1)
    options = dict(eps=eps, theta=theta, rotated=rotated, pairs=pairs)
    plain = qk_norm_rotary(q, k, wq, wk, pq, pk, **options)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, wq, wk) if t is not None]
    out = qk_norm_rotary(leaves[0], leaves[1], *(leaves[2:] or (None, None)), pq, pk, **options)
    got = torch.autograd.grad(out, leaves, (dq, dk))
    if rotated is None:
        rotated = dim // (2 * axes) * (2 * axes)
    for i, (x, w, p, d) in enumerate(((q, wq, pq, dq), (k, wk, pk, dk))):
        y, dx, dw = formula(x, w, p, d, rotated, pairs, theta, eps, dtype)
        assert out[i].dtype == dtype and out[i].is_contiguous() and torch.equal(out[i], plain[i])
        within(out[i], y, "y")
        within(got[i], dx, "dx")
        if w is not None:
            within(got[2 + i], dw, "dweight")
    only, none = qk_norm_rotary(q, None, wq, None, pq, None, **options)
    assert none is None and torch.equal(only, plain[0])
    return out, got


# batch, queries, keys, heads, kv_heads, dim, axes, rotated: one of everything; one token; whole and part heads;
# spans that are whole 16-byte pieces, 8, 4, and none; every width of a lane group; more heads than a CTA holds.
SIZES = [(1, 1, 1, 1, 1, 1, 1, None), (2, 3, 1, 2, 1, 2, 1, None), (1, 1, 4, 8, 2, 64, 2, None), (2, 37, 50, 4, 2, 32, 2, None),
         (3, 11, 70, 6, 3, 40, 1, 20), (1, 129, 5, 3, 3, 128, 1, None), (2, 20, 9, 5, 1, 13, 3, None), (1, 33, 17, 2, 2, 48, 3, None),
         (1, 300, 7, 1, 1, 16, 1, 8), (2, 5, 6, 300, 2, 24, 2, 12), (1, 2, 3, 2, 2, 100, 1, 0), (1, 3000, 40, 2, 2, 32, 2, None),
         (1, 9, 8, 4, 4, 36, 1, None), (1, 40, 30, 7, 7, 109, 3, None), (70, 2, 3, 2, 1, 8, 1, None), (1, 50, 60, 2, 1, 4, 2, None)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("kind", ["none", "float", "shared", "int32", "int64"])
@pytest.mark.parametrize(("batch", "queries", "keys", "heads", "kv_heads", "dim", "axes", "rotated"), SIZES)
def test_values_and_gradients(batch, queries, keys, heads, kv_heads, dim, axes, rotated, kind, pairs, dtype):
    check(batch, queries, keys, heads, kv_heads, dim, axes, rotated, pairs, kind, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
def test_settings(pairs, dtype):
    check(2, 9, 12, 2, 2, 64, 2, 32, pairs, "float", dtype, weighted=False, theta=100.0, eps=0.0)
    check(2, 9, 12, 2, 2, 64, 2, None, pairs, "int64", dtype, weighted=False, eps=10.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("dim", [8, 64, 36, 50, 70, 109, 128])
def test_no_epsilon(dim, pairs, dtype):
    # Every width of a piece, rows that do not fill a CTA's last turn: what lies behind them has no part in dweight.
    check(2, 9, 13, 2, 1, dim, 1, None, pairs, "float", dtype, eps=0.0)
    check(1, 301, 1, 3, 1, dim, 1, None, pairs, "none", dtype, eps=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
def test_far_positions_keep_their_angles(pairs):
    # Positions next to each other far out: 2^40 + i. Whole turns are taken off in 64 bits, so the turned vectors'
    # inner products depend on the distance alone, to float32's accuracy.
    x = torch.randn(1, 1, 1, 64, generator=torch.Generator().manual_seed(0)).cuda().expand(1, 50, 1, 64)
    near = torch.arange(50, device="cuda")[:, None]
    (a, _), (b, _) = (qk_norm_rotary(x, None, None, None, p, pairs=pairs) for p in (near, near + (1 << 40)))
    a, b = a[0, :, 0].double(), b[0, :, 0].double()
    # 2^40 turns in 64 bits leave 2^-13 of a turn's fraction: 2^40 x 2^-53 x 2 pi.
    assert float((a @ a.T - b @ b.T).abs().max()) <= 64 * 2.0 ** -10
    (c, _), = (qk_norm_rotary(x, None, None, None, near + (1 << 20), pairs=pairs),)
    c = c[0, :, 0].double()
    assert float((a @ a.T - c @ c.T).abs().max()) <= 64 * 4 * 2.0 ** -21


PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def exact_angles(positions, n, theta):
    """Angles less whole turns, and the whole angles' sizes and frequencies, of (position, pair), by 60 digits."""
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        frequencies = [decimal.Decimal(theta) ** (decimal.Decimal(-i) / n) for i in range(n)]
        rest = [[float((decimal.Decimal(p) * f).remainder_near(2 * PI)) for f in frequencies] for p in positions]
    f = torch.tensor([float(f) for f in frequencies], dtype=torch.float64)
    return torch.tensor(rest, dtype=torch.float64), torch.tensor(positions, dtype=torch.float64)[:, None].abs() * f, f


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize(("kind", "theta"), [("float", 1e4), ("float", 2.0 ** -20), ("int", 1e4)])
def test_angles_of_far_positions(kind, theta, pairs, dtype):
    # Heads (1, 0) in every pair come out as (cos, sin), times sqrt(2). A frequency f in 64 bits is off by (4 + |ln f|) 2^-53 of
    # itself (the exponent, the power, the division), its product with the position by another 2^-53; then t as above.
    n = 16
    places = [0, 1, -77, 5000, 400000, 500000, (1 << 23) + 1, -(1 << 26), (1 << 30) + 128, (1 << 36) + (1 << 13), -(1 << 40), (1 << 41) + (1 << 18)]
    if kind == "float":
        places += [0.25, 1000.5, 262143.96875]
    x = torch.zeros(1, len(places), 1, 2 * n, dtype=dtype, device="cuda")
    first = slice(0, n) if pairs == "halves" else slice(0, 2 * n, 2)
    second = slice(n, 2 * n) if pairs == "halves" else slice(1, 2 * n, 2)
    x[..., first] = 1
    p = torch.tensor(places, dtype=torch.float32 if kind == "float" else torch.int64, device="cuda")[:, None]
    y, _ = qk_norm_rotary(x, None, None, None, p, eps=0.0, theta=theta, pairs=pairs)
    y = y[0, :, 0].double().cpu() / math.sqrt(2.0)
    angle, size, f = exact_angles(places, n, theta)
    bound = torch.finfo(dtype).eps / 2 + (2.0 ** -21 if dtype == torch.float32 else 2.0 ** -19) + size * (5 + f.log().abs()) * 2.0 ** -53
    for got, want in ((y[:, first], torch.cos(angle)), (y[:, second], torch.sin(angle))):
        worst = ((got - want).abs() / bound).max(1)[0]
        assert float(worst.max()) <= 1.0, worst.tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("dim", [64, 24, 7])
def test_strided_broadcast_and_unaligned_arrays(dim, pairs, dtype):
    x, w, dy = inputs(2, 30, 4, dim, dtype)
    p = place("float", 2, 30, 1)

    def step(x, p, dy):
        leaf, weight = x.detach().requires_grad_(True), w.clone().requires_grad_(True)
        y, _ = qk_norm_rotary(leaf, None, weight, None, p, pairs=pairs)
        return (y.detach(), *torch.autograd.grad(y, (leaf, weight), dy))

    want = step(x, p, dy)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    def interleaved(t):
        return torch.stack([t, torch.full_like(t, 7.0)], 2).flatten(2, 3)[:, :, :t.shape[2]]

    u = torch.finfo(dtype).eps
    forms = [interleaved, lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), lambda t: t.transpose(2, 3).contiguous().transpose(2, 3),
             shifted, lambda t: t.flip(0).flip(0)]
    for form in forms:
        # Other widths of a lane's piece sum in another order: float32's last bits, and so one rounding to the type.
        for g, v in zip(step(form(x), p.transpose(0, 1).contiguous().transpose(0, 1), form(dy)), want):
            assert float((g.double() - v.double()).norm()) <= max(u, 2.0 ** -20) * float(v.double().norm())
    one = x[:1].clone().requires_grad_(True)
    (total,) = torch.autograd.grad(qk_norm_rotary(one.expand(2, -1, -1, -1), None, w, None, p, pairs=pairs)[0], one, dy)
    each = step(x[:1].repeat(2, 1, 1, 1), p, dy)[1]
    assert float((total - each.sum(0, keepdim=True)).abs().max()) <= 2 * u * float(each.abs().max())


@pytest.mark.gpu
def test_gradients_against_differences():
    x, w, dy = inputs(2, 20, 3, 24, torch.float32)
    p = place("float", 2, 20, 2)
    leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
    grads = torch.autograd.grad(qk_norm_rotary(leaves[0], None, leaves[1], None, p)[0], leaves, dy)
    step = 1e-2
    for i, grad in enumerate(grads):
        direction = torch.randn(grad.shape, generator=torch.Generator().manual_seed(i)).cuda()
        ends = []
        for sign in (1.0, -1.0):
            moved = [x, w]
            moved[i] = moved[i] + sign * step * direction
            ends.append((qk_norm_rotary(moved[0], None, moved[1], None, p)[0].double() * dy.double()).sum())
        slope = float(ends[0] - ends[1]) / (2 * step)
        # The remainder is of order step^2, the values' rounding 1e-5 / step.
        assert abs(slope - float((grad.double() * direction.double()).sum())) <= 3e-3 * float(grad.double().norm() * direction.double().norm())


@pytest.mark.gpu
def test_one_result_alone_has_its_own_gradients():
    q, wq, dq = inputs(2, 5, 4, 16, torch.float32)
    k, wk, _ = inputs(2, 7, 2, 16, torch.float32, 1)
    leaves = [t.requires_grad_(True) for t in (q, k, wq, wk)]
    qt, kt = qk_norm_rotary(*leaves)
    assert qt.shape == q.shape and kt.shape == k.shape
    got = torch.autograd.grad(qt, leaves, dq, allow_unused=True)
    assert got[1] is None and got[3] is None
    want = formula(q, wq, None, dq, 0, "halves", 1.0, 1e-6, torch.float32)
    within(got[0], want[1], "dx")
    within(got[2], want[2], "dweight")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_no_tokens(dtype):
    x, w, dy = inputs(2, 0, 4, 16, dtype)
    leaf, weight = x.requires_grad_(True), w.requires_grad_(True)
    y, none = qk_norm_rotary(leaf, None, weight, None, torch.zeros(0, 1, device="cuda"))
    dx, dw = torch.autograd.grad(y, (leaf, weight), dy)
    assert none is None and y.shape == x.shape and dx.shape == x.shape and float(dw.abs().sum()) == 0.0


@pytest.mark.gpu
def test_non_finite_heads_stay_by_themselves():
    x, w, _ = inputs(1, 40, 4, 32, torch.bfloat16)
    p = place("float", 1, 40, 2)
    clean, _ = qk_norm_rotary(x, None, w, None, p)
    x[0, 3, 2, 5] = float("nan")
    y, _ = qk_norm_rotary(x, None, w, None, p)
    assert y[0, 3, 2].isnan().all()
    y[0, 3, 2] = clean[0, 3, 2]
    assert torch.equal(y, clean)


@pytest.mark.gpu
def test_a_far_position_does_not_change_its_neighbours():
    x, w, _ = inputs(1, 60000, 1, 64, torch.float32)
    p = place("float", 1, 60000, 1) * 1000
    clean, _ = qk_norm_rotary(x, None, w, None, p)
    p[0, ::50] = 1e9
    y, _ = qk_norm_rotary(x, None, w, None, p)
    same = torch.arange(60000) % 50 != 0
    assert torch.equal(y[0, same], clean[0, same])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("dim", [64, 36, 70, 109])
def test_a_position_that_is_no_number_leaves_what_is_not_turned(dim, pairs, dtype):
    x, w, _ = inputs(1, 40, 2, dim, dtype)
    p = place("float", 1, 40, 1)
    clean, _ = qk_norm_rotary(x, None, w, None, p, rotated=4, pairs=pairs)
    for junk in (float("nan"), float("inf")):
        p[0, 7] = junk
        y, _ = qk_norm_rotary(x, None, w, None, p, rotated=4, pairs=pairs)
        assert y[0, 7, :, :4].isnan().all() and torch.equal(y[..., 4:], clean[..., 4:])
        y[0, 7] = clean[0, 7]
        assert torch.equal(y, clean)


@pytest.mark.gpu
def test_the_same_bits_every_time_on_a_side_stream_and_from_a_graph():
    q, wq, dq = inputs(4, 900, 4, 64, torch.bfloat16)
    k, wk, dk = inputs(4, 100, 2, 64, torch.bfloat16, 1)
    pq, pk = place("float", 4, 900, 2), place("float", 4, 100, 2, 1)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
        out = qk_norm_rotary(*leaves, pq, pk)
        return (*(o.detach() for o in out), *torch.autograd.grad(out, leaves, (dq, dk)))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    pq.add_(1.0)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(step(), third))


@pytest.mark.gpu
def test_past_two_to_the_31_values():
    tokens = (1 << 25) + 77
    x = torch.zeros(1, tokens, 1, 64, dtype=torch.bfloat16, device="cuda")
    tail, w, _ = inputs(1, 200, 1, 64, torch.bfloat16)
    x[:, -200:] = tail
    p = torch.zeros(tokens, 1, device="cuda")
    p[-200:] = place("shared", 1, 200, 1)
    y, _ = qk_norm_rotary(x, None, w, None, p)
    assert torch.equal(y[:, -200:], qk_norm_rotary(tail, None, w, None, p[-200:])[0]) and float(y[:, :1000].abs().max()) == 0.0


@pytest.mark.gpu
def test_more_than_once_is_refused():
    q, w, dq = inputs(1, 5, 2, 16, torch.float32)
    q.requires_grad_(True)
    (dx,) = torch.autograd.grad(qk_norm_rotary(q, None, w)[0], q, dq, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable itself"):
        torch.autograd.grad(dx.sum(), q)


def side(**change):
    a = dict(x=1 << 20, stride=(64, 32, 16), weight=None, positions=None, position_stride=(0, 1, 1), position_type=0, heads=2, tokens=2,
             out=1 << 21, dy=1 << 22, dweight=None)
    a.update(change)
    s = native.Heads(**{n: v for n, v in a.items() if not n.endswith("stride")})
    s.stride[:] = a["stride"]
    s.position_stride[:] = a["position_stride"]
    return s


@pytest.mark.parametrize(
    ("change", "call", "message"),
    [({}, dict(dtype=3), "dtype must be"), ({}, dict(dim=0), "dim <= 128"), ({}, dict(dim=129), "dim <= 128"), ({}, dict(rotated=6, axes=2), "multiple of 2"),
     ({}, dict(rotated=18), "multiple of 2"), ({}, dict(axes=0), "multiple of 2"), ({}, dict(pairs=2), "pairs must be"), ({}, dict(eps=-1.0), "eps >= 0"),
     ({}, dict(theta=0.0), "theta > 0"), ({}, dict(theta=float("inf")), "theta > 0"), (dict(heads=0), {}, "heads from 1"), (dict(tokens=-1), {}, "tokens"),
     (dict(x=None), {}, "null array"), (dict(out=None), {}, "null array"), (dict(x=(1 << 20) + 1), {}, "aligned"), (dict(weight=6), {}, "aligned"),
     (dict(positions=4096, position_type=3), {}, "position_type"), (dict(positions=4100, position_type=2), {}, "positions must be aligned"),
     (dict(out=(1 << 20) + 64), {}, "must not overlap"), ({}, dict(batch=-1), "batch")])
def test_the_c_abi_refuses(change, call, message):
    a = dict(dtype=1, batch=2, dim=16, rotated=16, axes=1, pairs=0, eps=1e-6, theta=1e4)
    a.update(call)
    with pytest.raises(ValueError, match=message):
        native.call("spectral_qk_norm_rotary", side(**change), None, *a.values(), None)


@pytest.mark.parametrize("axes", [(1 << 30) + 1, (1 << 31) - 1])
def test_the_c_abi_refuses_more_axes_than_pairs(axes):
    # Twice as many wrap in 32 bits: to 2 and to -2, which divide the head.
    keys = side(positions=4096)
    for name, work in (("spectral_qk_norm_rotary", ()), ("spectral_qk_norm_rotary_backward", (1 << 30,))):
        with pytest.raises(ValueError, match="multiple of 2"):
            native.call(name, keys, None, 1, 2, 16, 16, axes, 0, 1e-6, 1e4, *work, None)


@pytest.mark.gpu
def test_more_axes_than_pairs():
    q, w, _ = inputs(1, 3, 2, 16, torch.float32)
    many = torch.ones(3, 1, device="cuda").expand(3, (1 << 31) - 1)
    with pytest.raises(ValueError, match="multiple of 2"):
        qk_norm_rotary(q, None, w, None, many, rotated=16)
    # As many values as whole pairs of every axis: none.
    assert torch.equal(qk_norm_rotary(q, None, w, None, many)[0], qk_norm_rotary(q, None, w)[0])


def test_the_c_abi_refuses_backward():
    args = (1, 2, 16, 16, 1, 0, 1e-6, 1e4)
    for change, message in ((dict(dy=None), "null array"), (dict(dweight=4096), "workspace"), (dict(out=(1 << 22) + 64), "must not overlap")):
        with pytest.raises(ValueError, match=message):
            native.call("spectral_qk_norm_rotary_backward", side(**change), None, *args, None, None)
    with pytest.raises(ValueError, match="needs q or k"):
        native.call("spectral_qk_norm_rotary", None, None, *args, None)


@pytest.mark.parametrize(
    "change", [dict(x=(1 << 21) + 64), dict(out=(1 << 20) + 64), dict(out=(1 << 21) + 64), dict(out=1 << 22), dict(out=1 << 24), dict(dweight=1 << 22),
               dict(dweight=1 << 23), dict(weight=(1 << 21) + 64), dict(positions=(1 << 21) + 64), dict(dy=1 << 21)])
def test_the_c_abi_refuses_keys_over_the_queries(change):
    # The queries' arrays: x at 2^20, out 2^21, dy 2^22, dweight 2^23, weight 2^24.
    q = side(weight=1 << 24, dweight=1 << 23)
    k = side(**(dict(x=1 << 25, out=1 << 26, dy=1 << 27) | change))
    with pytest.raises(ValueError, match="must not overlap"):
        native.call("spectral_qk_norm_rotary_backward", q, k, 1, 2, 16, 16, 1, 0, 1e-6, 1e4, 1 << 30, None)


def test_cpu_tensors_and_wrong_counts_are_refused():
    with pytest.raises(NotImplementedError, match="CPU"):
        qk_norm_rotary(torch.zeros(1, 2, 2, 8))
    with pytest.raises(ValueError, match="must not be negative"):
        qk_norm_rotary(torch.zeros(1, 2, 2, 8), rotated=-2)


@pytest.mark.gpu
def test_wrong_arguments_are_refused():
    q, k = torch.zeros(2, 3, 4, 16, device="cuda"), torch.zeros(2, 5, 2, 16, device="cuda")
    p = torch.zeros(3, 2, device="cuda")
    with pytest.raises(RuntimeError, match="must be \\(batch, tokens, heads, dim\\)"):
        qk_norm_rotary(q[0])
    with pytest.raises(RuntimeError, match="k must be"):
        qk_norm_rotary(q, k.bfloat16())
    with pytest.raises(RuntimeError, match="agree in batch and dim"):
        qk_norm_rotary(q, k[:1])
    with pytest.raises(RuntimeError, match="q_weight must be"):
        qk_norm_rotary(q, None, torch.ones(8, device="cuda"))
    with pytest.raises(RuntimeError, match="k_weight must be"):
        qk_norm_rotary(q, k, None, torch.ones(16, device="cuda").bfloat16())
    with pytest.raises(RuntimeError, match="q_positions must be"):
        qk_norm_rotary(q, None, None, None, p[:2])
    with pytest.raises(RuntimeError, match="must be float32, int32 or int64"):
        qk_norm_rotary(q, None, None, None, p.double())
    with pytest.raises(RuntimeError, match="same axes"):
        qk_norm_rotary(q, k, None, None, p, torch.zeros(5, 1, device="cuda"))
    with pytest.raises(ValueError, match="multiple of 2"):
        qk_norm_rotary(q, None, None, None, p, rotated=6)
    with pytest.raises(RuntimeError, match="pairs must be"):
        qk_norm_rotary(q, pairs="thirds")
    with pytest.raises(RuntimeError, match="no gradient"):
        qk_norm_rotary(q.requires_grad_(True), None, None, None, p.requires_grad_(True))
