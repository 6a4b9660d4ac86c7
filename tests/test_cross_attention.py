"""Attention to states of another length: values and all gradients against the formula in float64, over types,
shared heads, sizes around the kernels' tiles, one query to many rows, cut keys (lengths, masks, rows left empty,
infinities and NaN in masked places), strided, broadcast and unaligned arrays; against differences; streams and
captured graphs; the refusals; CrossAttention, and FNOBlock with a context.

Tolerances are bounds on each value. With u the type's unit roundoff (2^-8 bf16, 2^-11 f16, 2^-24 float32) and
e = 2^-24, in the order the kernels compute:
  scores     off by dim e S, S the largest sum of |q k| scale, so weights by a factor 1 + p, p = 2 e ((dim + 4) S + 8)
  weights    16-bit: rounded once before they meet v, another u
  out        u |out| for its rounding, (p + u + 2 keys e) sum p |v|; the tensor cores cut a sum once per 16 keys, not more
  delta      its out is rounded: u sum |dout out|, and 2 dim e (sum |dout v| + sum |dout out|) with dp - delta
  dv, dk, dq their terms' errors, 2 n e of the sum of n magnitudes, u of the result for its rounding
float16 weights and gradients below its smallest normal number lose relative accuracy: 2^-25 of the scale they are
held in, at least 1 for weights (the largest is 1 or more), and 2^-40 of the largest product for gradients."""

import ctypes
import itertools
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from spectral import native
from spectral.nn import CrossAttention, FNOBlock, cross_attention, qk_norm_rotary

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
E = 2.0 ** -24


def inputs(batch, queries, keys, heads, kv_heads, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 3 * queries + 5 * keys + 7 * dim)
    shapes = [(batch, queries, heads, dim), (batch, keys, kv_heads, dim), (batch, keys, kv_heads, dim), (batch, queries, heads, dim)]
    return [torch.randn(*s, generator=g).to(dtype).cuda() for s in shapes]


def cuts(kind, batch, keys, seed=0):
    """lengths, mask, and the two together as a bool (batch, keys)."""
    g = torch.Generator().manual_seed(seed + keys)
    lengths = mask = None
    keep = torch.ones(batch, keys, dtype=torch.bool)
    if kind in ("lengths", "both"):
        lengths = torch.randint(0, keys + 1, (batch,), generator=g)
        lengths[0] = keys
        if batch > 1:
            lengths[1] = 0
        keep &= torch.arange(keys)[None] < lengths[:, None]
    if kind in ("mask", "both"):
        mask = torch.rand(batch, keys, generator=g) < 0.6
        if batch > 1:
            mask[-1] = False
        keep &= mask
    return (None if lengths is None else lengths.int().cuda(), None if mask is None else mask.cuda(), keep.cuda())


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def formula(q, k, v, dout, keep, scale, dtype):
    """out, dq, dk, dv in float64 and the bounds above, heads of k and v repeated for their queries."""
    q, k, v, dout = (t.detach().double().transpose(1, 2) for t in (q, k, v, dout))
    group, dim, keys, rows = q.shape[1] // k.shape[1], q.shape[-1], k.shape[2], q.shape[2] * (q.shape[1] // k.shape[1])
    keep = keep[:, None, None]
    wipe = keep.transpose(-1, -2)
    k, v = (torch.where(wipe, t, torch.zeros_like(t)).repeat_interleave(group, 1) for t in (k, v))
    u = unit(dtype)
    soft = u if dtype != torch.float32 else 0.0
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    s = torch.where(keep, q @ k.transpose(-1, -2) * scale, torch.full((), -math.inf, dtype=torch.float64, device=q.device))
    p = torch.softmax(s, -1).nan_to_num(0.0)
    size = float((q.abs() @ k.abs().transpose(-1, -2)).max()) * abs(scale) if keys else 0.0
    slack = 2 * E * ((dim + 4) * size + 8)
    out = p @ v
    most = float(v.abs().max()) if v.numel() else 0.0
    out_e = u * out.abs() + (slack + soft + 2 * keys * E) * (p @ v.abs()) + tiny * keys * most
    dp, delta = dout @ v.transpose(-1, -2), (dout * out).sum(-1, keepdim=True)
    dp_a = dout.abs() @ v.abs().transpose(-1, -2)
    delta_a = (dout.abs() * out.abs()).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    ds_e = (2 * slack + soft) * ds.abs() + p * (2 * dim * E * (dp_a + delta_a) + u * delta_a + (dout.abs() * out_e).sum(-1, keepdim=True))
    ds_e = ds_e + tiny * 2.0 ** -15 * float(dp_a.max() if dp_a.numel() else 0.0)
    a = abs(scale)
    dq, dq_e = ds @ k * scale, (ds_e + 2 * keys * E * ds.abs()) @ k.abs() * a
    t = lambda m: m.transpose(-1, -2)
    dk, dk_e = t(ds) @ q * scale, t(ds_e + 2 * rows * E * ds.abs()) @ q.abs() * a
    dv, dv_e = t(p) @ dout, t((slack + soft + 2 * rows * E) * p + tiny) @ dout.abs()

    def shared(m):
        return m.unflatten(1, (-1, group)).sum(2)

    dk, dk_e, dv, dv_e = map(shared, (dk, dk_e, dv, dv_e))
    results = [(out, out_e), (dq, dq_e + u * dq.abs()), (dk, dk_e + u * dk.abs()), (dv, dv_e + u * dv.abs())]
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return [(w.transpose(1, 2), b.transpose(1, 2) + least + 1e-30) for w, b in results]


def within(got, want, name):
    value, bound = want
    assert got.shape == value.shape, name
    if got.numel() == 0:
        return
    ratio = ((got.detach().double() - value).abs() / bound)
    assert got.isfinite().all(), f"{name}: not finite"
    worst = float(ratio.max())
    assert worst <= 1.0, f"{name}: {worst:.3g} of the bound at {ratio.flatten().argmax().item()}"


def run(q, k, v, dout, **options):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves, **options)
    assert out.dtype == q.dtype and out.is_contiguous()
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


def check(q, k, v, dout, keep=None, scale=None, **options):
    if keep is None:
        keep = torch.ones(k.shape[0], k.shape[1], dtype=torch.bool, device=k.device)
    got = run(q, k, v, dout, scale=scale, **options)
    want = formula(q, k, v, dout, keep, 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale, q.dtype)
    for g, w, name in zip(got, want, ("out", "dq", "dk", "dv")):
        within(g, w, name)
    assert torch.equal(cross_attention(q, k, v, scale=scale, **options), got[0])
    return got


# batch, queries, keys, heads, kv_heads, dim: one of everything; rows around tiles of 64, 128 and 256; keys around 64
# and 128; shared heads that divide a tile and that do not; heads that are no 16-byte pieces; few rows over many
# keys and the other way round.
SIZES = [(1, 1, 1, 1, 1, 1), (2, 1, 5, 2, 1, 8), (1, 3, 64, 4, 4, 16), (2, 64, 65, 2, 2, 32), (1, 65, 63, 3, 1, 24), (1, 127, 128, 2, 2, 64),
         (2, 128, 129, 4, 2, 64), (1, 129, 127, 2, 1, 128), (3, 40, 300, 6, 3, 40), (1, 257, 257, 2, 2, 80), (1, 300, 40, 5, 1, 13),
         (2, 1, 5000, 8, 2, 64), (1, 2, 3000, 6, 3, 48), (1, 17, 2500, 16, 1, 128), (1, 2600, 100, 4, 2, 32), (2, 700, 130, 2, 2, 96),
         (1, 50, 90, 128, 1, 8), (1, 260, 140, 24, 2, 36), (70, 3, 9, 2, 1, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["none", "lengths", "mask", "both"])
@pytest.mark.parametrize(("batch", "queries", "keys", "heads", "kv_heads", "dim"), SIZES)
def test_values_and_gradients(batch, queries, keys, heads, kv_heads, dim, kind, dtype):
    q, k, v, dout = inputs(batch, queries, keys, heads, kv_heads, dim, dtype)
    lengths, mask, keep = cuts(kind, batch, keys)
    got = check(q, k, v, dout, keep, lengths=lengths, mask=mask)
    for t in got[2:]:  # gradients of keys that do not count are zeros, not small numbers
        assert t[~keep].abs().sum() == 0
    empty = ~keep.any(1)
    assert got[0][empty].abs().sum() == 0 and got[1][empty].abs().sum() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["none", "both"])
@pytest.mark.parametrize(("batch", "queries", "keys", "heads", "kv_heads", "dim"),
                         [(2, 9, 65, 1, 1, 24), (1, 12, 1500, 2, 2, 64), (2, 3, 130, 8, 2, 40), (3, 16, 70, 2, 2, 128), (2, 2, 3000, 16, 2, 80),
                          (2, 5, 150, 128, 1, 64), (2, 3, 270, 130, 2, 128), (2, 1, 200, 100, 1, 50), (2, 20, 90, 96, 1, 96), (2, 300, 40, 66, 1, 33)])
def test_a_dozen_rows_and_many_heads_over_one(batch, queries, keys, heads, kv_heads, dim, kind, dtype):
    q, k, v, dout = inputs(batch, queries, keys, heads, kv_heads, dim, dtype)
    lengths, mask, keep = cuts(kind, batch, keys)
    check(q, k, v, dout, keep, lengths=lengths, mask=mask)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("queries", "keys"), [(1, 700), (12, 300), (200, 300)])
def test_the_operators_without_autograd(queries, keys, dtype):
    q, k, v, dout = inputs(2, queries, keys, 4, 2, 64, dtype)
    lengths, mask, keep = cuts("both", 2, keys)
    lengths[1], mask[1, :9] = keys, True
    keep = (torch.arange(keys, device="cuda")[None] < lengths[:, None]) & mask
    want = run(q, k, v, dout, lengths=lengths, mask=mask)
    ops = torch.ops.spectral
    out, stats, rest = ops.cross_attention(q, k, v, lengths, mask)
    assert torch.equal(out, want[0]) and rest.numel() == (0 if dtype == torch.float32 else out.numel())
    got = ops.cross_attention_backward(dout, q, k, v, out, stats, rest, lengths, mask)
    assert all(torch.equal(g, w) for g, w in zip(got, want[1:]))
    # Without what out's rounding took: the bounds count a rounded out.
    got = ops.cross_attention_backward(dout, q, k, v, out, stats, rest[:0].reshape(-1), lengths, mask)
    for g, w, name in zip(got, formula(q, k, v, dout, keep, 0.125, dtype)[1:], ("dq", "dk", "dv")):
        within(g, w, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("queries", "keys"), [(1, 700), (200, 300)])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf"), "largest"])
def test_what_lies_in_masked_places_has_no_effect(queries, keys, junk, dtype):
    q, k, v, dout = inputs(3, queries, keys, 4, 2, 64, dtype)
    lengths, mask, keep = cuts("both", 3, keys)
    want = run(q, k, v, dout, lengths=lengths, mask=mask)
    for t in (k, v):
        t[~keep] = -torch.finfo(dtype).max if junk == "largest" else junk
    got = run(q, k, v, dout, lengths=lengths, mask=mask)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_values_reach_what_reads_them_and_nothing_else(dtype):
    q, k, v, dout = inputs(2, 150, 200, 2, 2, 32, dtype)
    want = run(q, k, v, dout)
    q[0, 7, 1, 3] = float("nan")
    got = run(q, k, v, dout)
    rest = torch.ones(2, 150, 2, dtype=torch.bool)
    rest[0, 7, 1] = False
    for i in (0, 1):
        assert got[i][0, 7, 1].isnan().all() and torch.equal(got[i][rest.cuda()], want[i][rest.cuda()])
    for i in (2, 3):
        assert got[i][0, :, 1].isnan().all() and torch.equal(got[i][1], want[i][1]) and torch.equal(got[i][0, :, 0], want[i][0, :, 0])
    q, k, v, dout = inputs(2, 150, 200, 2, 2, 32, dtype)
    v[1, 5, 0, 4] = float("inf")
    got = run(q, k, v, dout)
    assert not got[0][1, :, 0, 4].isfinite().any() and torch.equal(got[0][0], want[0][0]) and torch.equal(got[0][1, :, 1], want[0][1, :, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("queries", "heads", "dim"), [(1, 2, 64), (8, 2, 64), (9, 2, 64), (16, 2, 64), (17, 2, 64), (100, 2, 64), (100, 2, 128), (40, 4, 20),
                                                 (3, 130, 32)])
def test_infinities_that_count(queries, heads, dim, dtype):
    # What the formula gives, whichever kernel a call's size takes. An infinite value: its weights are positive, so infinite results.
    q, k, v, dout = inputs(2, queries, 90, heads, 2, dim, dtype)
    clean, group, rest = cross_attention(q, k, v), heads // 2, torch.arange(dim) != 4
    for sign in (1.0, -1.0):
        v[1, 5, 0, 4] = sign * float("inf")
        out = cross_attention(q, k, v)
        assert bool((out[1, :, :group, 4] == sign * float("inf")).all())
        assert torch.equal(out[0], clean[0]) and torch.equal(out[1, :, group:], clean[1, :, group:]) and torch.equal(out[..., rest], clean[..., rest])
    # An infinite key: scores of either infinity by the query's sign. A weight of 0, as if the key did not count, or no number.
    q, k, v, dout = inputs(2, queries, 90, heads, 2, dim, dtype)
    k[1, 5, 0, 4] = float("inf")
    out = cross_attention(q, k, v)
    keep = torch.ones(2, 90, dtype=torch.bool, device="cuda")
    keep[1, 5] = False
    k[1, 5, 0, 4] = 0.0
    want, bound = formula(q, k, v, dout, keep, 1.0 / math.sqrt(dim), dtype)[0]
    positive = q[1, :, :group, 4] > 0
    assert bool(out[1, :, :group][positive].isnan().all())
    ratio = ((out.double() - want).abs() / bound)[1, :, :group][~positive]
    assert ratio.numel() == 0 or float(ratio.max()) <= 1.0
    assert torch.equal(out[0], clean[0]) and torch.equal(out[1, :, group:], clean[1, :, group:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("queries", "keys", "dim"), [(33, 70, 64), (33, 70, 20), (1, 900, 64), (200, 200, 128)])
def test_strided_broadcast_and_unaligned_arrays(queries, keys, dim, dtype):
    q, k, v, dout = inputs(2, queries, keys, 4, 2, dim, dtype)
    want = check(q, k, v, dout)

    def same(got, tolerance=0.0):
        for g, w in zip(got, want):
            assert float((g.double() - w.double()).norm()) <= tolerance * float(w.double().norm())

    def shifted(t):  # the same values one element off
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    def interleaved(t):  # next to other values of the same tokens
        return torch.stack([t, torch.full_like(t, 7.0)], 2).flatten(2, 3)[:, :, :t.shape[2]]

    def heads_first(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def dim_strided(t):
        return t.transpose(2, 3).contiguous().transpose(2, 3)

    for form in (interleaved, heads_first, dim_strided):
        same(run(form(q), form(k), form(v), form(dout)))
    # Off a 16-byte boundary a few rows' dot products add up in another order of lanes: the same bounds, not the same bits.
    check(shifted(q), shifted(k), shifted(v), shifted(dout))
    # Keys and values of one sample for all, of one head for all: broadcast arrays, whose gradients add up.
    got = run(q, k[:1].expand(2, -1, -1, -1), v[:, :, :1].expand(-1, -1, 2, -1), dout)
    full = run(q, k[:1].repeat(2, 1, 1, 1), v[:, :, :1].repeat(1, 1, 2, 1), dout)
    assert all(torch.equal(a, b) for a, b in zip(got, full))
    one = k[:1].clone().requires_grad_(True)
    (total,) = torch.autograd.grad(cross_attention(q, one.expand(2, -1, -1, -1), v), one, dout)
    each = run(q, k[:1].repeat(2, 1, 1, 1), v, dout)[2]
    assert float((total - each.sum(0, keepdim=True)).abs().max()) <= 2 * unit(dtype) * float(each.abs().max()) * 2
    same([cross_attention(q, k, v)], 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_scale_and_sharp_scores(dtype):
    q, k, v, dout = inputs(1, 100, 150, 2, 2, 32, dtype)
    check(q, k, v, dout, scale=0.0)
    check(q, k, v, dout, scale=-0.3)
    check(4 * q, k, v, dout, scale=1.0)
    # Scores in rising order, so that the largest so far changes all the way along, and in falling order.
    order = torch.argsort((q[0, 0, 0].float() * k[0, :, 0].float()).sum(-1))
    for o in (order, order.flip(0)):
        check(8 * q, k[:, o].contiguous(), v[:, o].contiguous(), dout)
    # One score far above the rest: its value, exactly.
    k[:, 77] = 30 * torch.sign(q[:, 3])
    out = cross_attention(q[:, 3:4], k, v, scale=1.0)
    assert torch.equal(out[:, 0], v[:, 77])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_small_and_large_gradients_keep_their_accuracy(dtype):
    q, k, v, dout = inputs(1, 300, 2000, 2, 2, 64, dtype)
    for size in (2.0 ** -10, 2.0 ** 8):
        check(q, k, v, (dout.float() * size).to(dtype))
    check(q, k, 64 * v, dout * 16)


@pytest.mark.gpu
@pytest.mark.parametrize(("queries", "keys", "dim"), [(1, 900, 64), (40, 300, 64), (300, 200, 32), (30, 100, 20), (200, 300, 128), (12000, 70, 16)])
def test_the_size_of_the_values_does_not_change_the_accuracy(queries, keys, dim):
    # bf16 values times a power of two give out, dq and dk times it, bit for bit: what out's rounding took is kept relative to out.
    q, k, v, dout = inputs(1, queries, keys, 4, 2, dim, torch.bfloat16)
    want = run(q, k, v, dout)
    for size in (2.0 ** -40, 2.0 ** -20, 2.0 ** -7, 2.0 ** 15, 2.0 ** 40):
        got = run(q, k, v * size, dout)
        for g, w, by in zip(got, want, (size, size, size, 1.0)):
            assert torch.equal(g.float(), w.float() * by), size


@pytest.mark.gpu
def test_sums_of_one_sign_over_many_keys_and_rows():
    # Terms that do not cancel: what a sum loses on the way shows here.
    for dtype, (queries, keys) in itertools.product([torch.bfloat16, torch.float16], [(2, 60000), (60000, 40)]):
        q, k, v, dout = inputs(1, queries, keys, 1, 1, 16, dtype)
        q, v, dout = 0.1 * q, v.abs() + 1, dout.abs() + 1
        check(q, k, v, dout)


@pytest.mark.gpu
def test_gradients_against_differences():
    q, k, v, dout = inputs(2, 30, 70, 4, 2, 24, torch.float32)
    lengths, mask, _ = cuts("both", 2, 70)
    lengths[1], mask[1, :9] = 50, True
    grads = run(q, k, v, dout, lengths=lengths, mask=mask)[1:]
    step = 1e-2
    for i, grad in enumerate(grads):
        direction = torch.randn(grad.shape, generator=torch.Generator().manual_seed(i)).cuda()
        ends = []
        for sign in (1.0, -1.0):
            moved = [q, k, v]
            moved[i] = moved[i] + sign * step * direction
            ends.append((cross_attention(*moved, lengths=lengths, mask=mask).double() * dout.double()).sum())
        slope = float(ends[0] - ends[1]) / (2 * step)
        # The remainder is of order step^2 (third derivatives of order one), the values' rounding 1e-5 / step.
        assert abs(slope - float((grad.double() * direction.double()).sum())) <= 3e-3 * float(grad.double().norm() * direction.double().norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_to_attend_to(dtype):
    q, k, v, dout = inputs(2, 5, 0, 4, 2, 16, dtype)
    out, dq, dk, dv = run(q, k, v, dout)
    assert out.shape == q.shape and out.abs().sum() == 0 and dq.abs().sum() == 0 and dk.shape == k.shape and dv.shape == v.shape
    for empty in (inputs(2, 0, 7, 4, 2, 16, dtype), inputs(0, 5, 7, 4, 2, 16, dtype)):
        out, dq, dk, dv = run(*empty)
        assert out.shape == empty[0].shape and dk.abs().sum() == 0 and dv.abs().sum() == 0
    q, k, v, dout = inputs(2, 5, 9, 4, 2, 16, dtype)
    for none in (dict(lengths=torch.zeros(2, dtype=torch.int64, device="cuda")), dict(mask=torch.zeros(1, 9, dtype=torch.bool, device="cuda"))):
        assert all(t.abs().sum() == 0 for t in run(q, k, v, dout, **none))


@pytest.mark.gpu
def test_lengths_beyond_the_keys_and_below_zero():
    q, k, v, dout = inputs(3, 9, 40, 2, 2, 32, torch.bfloat16)
    clear = run(q, k, v, dout, lengths=torch.tensor([40, 0, 17], device="cuda"))
    odd = run(q, k, v, dout, lengths=torch.tensor([1 << 40, -(1 << 40), 17], device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(clear, odd))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("queries", "keys"), [(1, 6000), (700, 400)])
def test_the_same_bits_every_time_on_a_side_stream_and_from_a_graph(queries, keys, dtype):
    q, k, v, dout = inputs(2, queries, keys, 4, 2, 64, dtype)
    lengths, mask, _ = cuts("both", 2, keys)
    lengths[1] = keys // 2
    step = lambda: run(q, k, v, dout, lengths=lengths, mask=mask)
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step())
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in results for a, b in zip(first, r))
    # Other inputs in the same places: a captured pass reads them, and the lengths, as they are then.
    q.mul_(0.5)
    lengths.copy_(torch.tensor([keys // 3, keys], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(results[0], step()))


@pytest.mark.gpu
def test_calls_on_several_streams_at_once():
    # Kernels that share SMs and their tensor memory: one sample's worth each, so that they run side by side.
    cases = [inputs(1, queries, keys, heads, 2, dim, dtype)
             for dtype, (queries, keys, heads, dim) in zip(DTYPES * 2, [(300, 700, 2, 64), (500, 300, 4, 32), (200, 900, 2, 128), (100, 400, 2, 96),
                                                                       (1, 5000, 4, 64), (700, 130, 2, 64)])]
    want = [run(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for c, stream in zip(cases, streams):
            with torch.cuda.stream(stream):
                got.append(run(*c))
    torch.cuda.synchronize()
    for i, results in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(results, want[i % len(cases)]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 40])
def test_lengths_outside_the_keys(queries, dtype):
    # Longer than the keys: all of them count. Negative: none.
    q, k, v, dout = inputs(3, queries, 333, 4, 2, 64, dtype)
    within_keys = torch.tensor([333, 0, 100], device="cuda")
    for kind in (torch.int32, torch.int64):
        least, most = torch.iinfo(kind).min, torch.iinfo(kind).max
        for low, high in ((-1, 334), (least, most)):
            got = run(q, k, v, dout, lengths=torch.tensor([high, low, 100], dtype=kind, device="cuda"))
            assert all(torch.equal(a, b) for a, b in zip(got, run(q, k, v, dout, lengths=within_keys.to(kind))))


@pytest.mark.gpu
@pytest.mark.parametrize("queries", [1, 20])
def test_the_last_of_the_most_keys(queries):
    # As many keys as a call may have, all the same one: where only the last 100 count the answer is their value, with weights
    # of one exactly, and a sum of 100 equal terms is off by far less than half a step of bf16.
    keys = (1 << 31) - 256
    q, k, v, _ = inputs(1, queries, 1, 1, 1, 8, torch.bfloat16)
    mask = torch.zeros(1, keys, dtype=torch.bool, device="cuda")
    mask[:, -100:] = True
    out = cross_attention(q, k.expand(1, keys, 1, 8), v.expand(1, keys, 1, 8), mask=mask)
    assert torch.equal(out, v.expand_as(out))


@pytest.mark.gpu
def test_past_two_to_the_31_values():
    keys = (1 << 25) + 77
    k = torch.zeros(1, keys, 1, 64, dtype=torch.bfloat16, device="cuda")
    q, k1, _, _ = inputs(1, 1, 200, 1, 1, 64, torch.bfloat16)
    mask = torch.zeros(1, keys, dtype=torch.bool, device="cuda")
    mask[:, -200:] = True
    k[:, -200:] = k1
    # Which keys share a tile differs from that of the 200 alone, and with it where a running maximum moves: not the
    # same bits, the same bounds.
    all_count = torch.ones(1, 200, dtype=torch.bool, device="cuda")
    within(cross_attention(q, k, k, mask=mask), formula(q, k1, k1, q, all_count, 0.125, torch.bfloat16)[0], "out")


@pytest.mark.gpu
def test_more_than_once_is_refused():
    q, k, v, dout = inputs(1, 5, 9, 2, 2, 16, torch.float32)
    q.requires_grad_(True)
    (dq,) = torch.autograd.grad(cross_attention(q, k, v), q, dout, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable itself"):
        torch.autograd.grad(dq.sum(), q)
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        cross_attention(fwad.make_dual(q.detach(), torch.ones_like(q)), k, v)


def module_inputs(dtype, channels=32, context_channels=24):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 6, 10, channels, generator=g).to(dtype).cuda()
    context = torch.randn(2, 30, context_channels, generator=g).to(dtype).cuda()
    return x, context, 40 * torch.rand(60, 2, generator=g).cuda(), 40 * torch.rand(2, 30, 2, generator=g).cuda()


def module64(m, x, context, positions, places, keep):
    """CrossAttention in float64."""
    b, d = x.shape[0], m.head_dim
    w = {n: p.detach().double() for n, p in m.named_parameters()}

    def turned(t, weight, pos):
        y = t / torch.sqrt((t * t).mean(-1, keepdim=True) + m.eps) * weight
        span, out = d // pos.shape[-1], []
        for a in range(pos.shape[-1]):
            n = span // 2
            angle = pos[..., a, None].double() * m.theta ** (-torch.arange(n, device=t.device).double() / n)
            one, two = y[..., a * span:a * span + n], y[..., a * span + n:(a + 1) * span]
            c, s = torch.cos(angle).unsqueeze(-2), torch.sin(angle).unsqueeze(-2)
            out += [one * c - two * s, one * s + two * c]
        return torch.cat(out, -1)

    q = turned((x @ w["w_q"].T).reshape(b, -1, m.heads, d), w["q_norm"], positions)
    k = turned((context @ w["w_k"].T).reshape(b, -1, m.kv_heads, d), w["k_norm"], places)
    v = (context @ w["w_v"].T).reshape(b, -1, m.kv_heads, d)
    k, v = (t.repeat_interleave(m.heads // m.kv_heads, 2) for t in (k, v))
    s = torch.einsum("bthd,bshd->bhts", q, k) / math.sqrt(d)
    p = torch.softmax(s.masked_fill(~keep[:, None, None], -math.inf), -1)
    out = torch.einsum("bhts,bshd->bthd", p, v).reshape(*x.shape[:-1], m.heads * d)
    return out @ w["w_out"].T


@pytest.mark.gpu
# A chain of four roundings to 16 bits (projection, turning, attention, projection) and products in between.
@pytest.mark.parametrize(("dtype", "tol"), [(torch.float32, 2e-5), (torch.bfloat16, 3e-2), (torch.float16, 4e-3)])
def test_module(dtype, tol):
    torch.manual_seed(0)
    m = CrossAttention(32, 24, 4, kv_heads=2, device="cuda", dtype=dtype)
    x, context, positions, places = module_inputs(dtype)
    lengths = torch.tensor([30, 11], device="cuda")
    keep = torch.arange(30, device="cuda")[None] < lengths[:, None]
    leaves = [x.requires_grad_(True), context.requires_grad_(True), *m.parameters()]
    y = m(x, context, positions=positions, context_positions=places, lengths=lengths)
    up = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    got = torch.autograd.grad(y, leaves, up)
    ref = CrossAttention(32, 24, 4, kv_heads=2, device="cuda", dtype=torch.float64).double()
    ref.load_state_dict({n: p.double() for n, p in m.state_dict().items()})
    x64, c64 = x.detach().double().requires_grad_(True), context.detach().double().requires_grad_(True)
    want = module64(ref, x64, c64, positions, places, keep)
    assert float((y.double() - want).norm()) <= tol * float(want.norm())
    for g, w in zip(got[:2], torch.autograd.grad(want, (x64, c64), up.double())):
        assert float((g.double() - w).norm()) <= tol * float(w.norm())
    assert all(g.isfinite().all() and float(g.abs().sum()) > 0 for g in got)
    assert "32, 24, heads=4, kv_heads=2, head_dim=8" in repr(m)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(0, 6, 10), (2, 0, 10), (2,)])
def test_module_over_no_samples_no_points_and_one_point_each(shape, dtype):
    torch.manual_seed(0)
    m = CrossAttention(32, 24, 4, kv_heads=2, device="cuda", dtype=dtype)
    x = torch.randn(*shape, 32, device="cuda").to(dtype).requires_grad_(True)
    context = torch.randn(shape[0], 30, 24, device="cuda").to(dtype)
    points = math.prod(shape[1:])
    places = torch.rand(points, 2, device="cuda"), torch.rand(30, 2, device="cuda")
    y = m(x, context, positions=places[0], context_positions=places[1])
    assert y.shape == x.shape
    y.sum().backward()
    assert x.grad.shape == x.shape and all(p.grad is not None and bool(p.grad.isfinite().all()) for p in m.parameters())
    if points == 1:
        assert torch.equal(y, m(x[:, None], context, positions=places[0], context_positions=places[1])[:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_the_passes_together(dtype):
    """Norm and rotation, then attention, and back, as a layer runs them: against the same in float64."""
    q, k, v, dout = inputs(2, 90, 140, 4, 2, 32, dtype)
    g = torch.Generator().manual_seed(3)
    wq, wk = (1 + 0.2 * torch.randn(32, generator=g).cuda() for _ in range(2))
    pq, pk = 60 * torch.rand(90, 2, generator=g).cuda(), 60 * torch.rand(2, 140, 2, generator=g).cuda()
    leaves = [t.requires_grad_(True) for t in (q, k, v, wq, wk)]
    qt, kt = qk_norm_rotary(q, k, wq, wk, pq, pk)
    got = torch.autograd.grad(cross_attention(qt, kt, v), leaves, dout)

    def turned(t, w, pos):
        y = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w
        angle = (pos.double()[..., None] * 1e4 ** (-torch.arange(8, device="cuda").double() / 8)).unsqueeze(-3)
        one, two = y.unflatten(-1, (2, 2, 8)).unbind(-2)
        c, s = torch.cos(angle), torch.sin(angle)
        return torch.stack([one * c - two * s, one * s + two * c], -2).flatten(-3)

    ref = [t.detach().double().requires_grad_(True) for t in leaves]
    q64, k64 = turned(ref[0], ref[3], pq), turned(ref[1], ref[4], pk)
    s = torch.einsum("bthd,bshd->bhts", q64, k64.repeat_interleave(2, 2)) / math.sqrt(32)
    out = torch.einsum("bhts,bshd->bthd", torch.softmax(s, -1), ref[2].repeat_interleave(2, 2))
    # The turned queries and keys, the weights, out and the gradients between are rounded: six roundings at most.
    tol = {torch.float32: 1e-5, torch.bfloat16: 6 * 2.0 ** -8, torch.float16: 6 * 2.0 ** -11}[dtype]
    for g, w in zip(got, torch.autograd.grad(out, ref, dout.double())):
        assert float((g.double() - w).norm()) <= tol * float(w.norm())


@pytest.mark.gpu
def test_fno_block_with_a_context():
    torch.manual_seed(1)
    plain = FNOBlock(16, 32, 4, 4, groups=4, device="cuda")
    torch.manual_seed(1)
    block = FNOBlock(16, 32, 4, 4, groups=4, device="cuda", context_channels=12, heads=2)
    u, context = torch.randn(2, 16, 16, 16, device="cuda"), torch.randn(2, 21, 12, device="cuda")
    places = torch.rand(2, 21, 2, device="cuda")
    for (_, a), (_, b) in zip(plain.named_parameters(), block.named_parameters()):
        assert torch.equal(a, b)
    # Without states the block is the plain one.
    none = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert torch.equal(block(u, context, context_positions=places, lengths=none), plain(u))
    y = block(u, context, context_positions=places)
    h = plain.norm(plain.conv(u).permute(0, 2, 3, 1))
    grid = torch.cartesian_prod(*[torch.arange(16, device="cuda", dtype=torch.float32) * 8] * 2)
    keep = torch.ones(2, 21, dtype=torch.bool, device="cuda")
    h = h.double() + module64(block.attention, h.double(), context.double(), grid, 128 * places, keep)
    want = u + plain.mlp(h.float()).permute(0, 3, 1, 2)
    assert float((y - want).norm()) <= 1e-5 * float(want.norm())
    y.square().mean().backward()
    assert all(p.grad is not None and p.grad.abs().isfinite().all() for p in block.parameters())
    with pytest.raises(ValueError, match="context"):
        block(u)
    with pytest.raises(ValueError, match="context"):
        plain(u, context)


def arguments(**change):
    a = dict(q=1 << 20, k=1 << 21, v=1 << 22, strides=None, lengths=None, lengths64=0, mask=None, out=1 << 23, rest=None, stats=1 << 24, dtype=1, batch=2,
             queries=4, keys=8, heads=4, kv_heads=2, dim=16, scale=1.0, work=1 << 25, stream=None)
    a.update(change)
    return tuple(a.values())


@pytest.mark.parametrize(
    ("change", "message"),
    [(dict(dtype=3), "dtype must be"), (dict(batch=-1), "need batch"), (dict(queries=-1), "need batch"), (dict(keys=1 << 31), "need batch"),
     (dict(dim=0), "dim <= 128"), (dict(dim=129), "dim <= 128"), (dict(heads=3), "multiple of kv_heads"), (dict(kv_heads=0), "multiple of kv_heads"),
     (dict(heads=258), "may share"), (dict(batch=40000), "need batch"), (dict(q=None), "null array"), (dict(v=None), "null array"),
     (dict(out=None), "null array"), (dict(k=(1 << 21) + 1), "aligned"), (dict(stats=(1 << 24) + 4), "aligned"), (dict(lengths=2), "aligned"),
     (dict(lengths=4100, lengths64=1), "aligned"), (dict(out=(1 << 20) + 64), "must not overlap"), (dict(out=(1 << 22) + 64), "must not overlap"),
     (dict(stats=(1 << 23) + 64), "must not overlap"), (dict(rest=(1 << 23) + 64), "must not overlap"), (dict(rest=1 << 24), "must not overlap"),
     (dict(stats=1 << 20), "must not overlap"), (dict(mask=1 << 23), "must not overlap"), (dict(lengths=(1 << 23) + 8), "must not overlap")])
def test_the_c_abi_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        native.call("spectral_cross_attention", *arguments(**change))


@pytest.mark.parametrize(
    ("change", "message"),
    [(dict(dout=None), "null array"), (dict(stats=None), "null array"), (dict(dk=None), "null array"), (dict(work=None), "null array"),
     (dict(dq=(1 << 27) + 1), "aligned"), (dict(dq=(1 << 20) + 64), "must not overlap"), (dict(dv=(1 << 19) + 64), "must not overlap"),
     (dict(dk=(1 << 27) + 64), "must not overlap"), (dict(dv=1 << 28), "must not overlap"), (dict(dq=1 << 24), "must not overlap"),
     (dict(rest=1 << 28), "must not overlap"), (dict(mask=1 << 29), "must not overlap"), (dict(work=1 << 27), "must not overlap"),
     (dict(dtype=-1), "dtype must be")])
def test_the_c_abi_refuses_backward(change, message):
    a = dict(dout=1 << 19, q=1 << 20, k=1 << 21, v=1 << 22, strides=None, out=1 << 23, rest=None, stats=1 << 24, lengths=None, lengths64=0, mask=None,
             dq=1 << 27, dk=1 << 28, dv=1 << 29, dtype=1, batch=2, queries=4, keys=8, heads=4, kv_heads=2, dim=16, scale=1.0, work=1 << 30,
             stream=None)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        native.call("spectral_cross_attention_backward", *a.values())


def host_program(tmp_path, source):
    """Compiles and runs a C++ program over the kernels' host headers; its output."""
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    headers = Path(__file__).resolve().parent.parent / "gpu-spectral-stack_b200" / "csrc"
    (tmp_path / "main.cpp").write_text(source)
    subprocess.run(["g++", "-std=c++17", "-I", str(headers), str(tmp_path / "main.cpp"), "-o", str(tmp_path / "main")], check=True)
    return subprocess.run([str(tmp_path / "main")], check=True, capture_output=True, text=True).stdout


def test_a_workspace_starts_on_whole_256s_and_has_room_for_that(tmp_path):
    source = """
        #include "workspace.hpp"
        #include <cstdio>
        #include <initializer_list>
        int main()
        {
            using namespace spectral;
            Arena arena;
            for (std::size_t bytes : {1, 256, 300, 0, 8}) {
                const std::size_t at = arena.take(bytes);
                if (at % 256 != 0) return 1;
            }
            if (arena.size() != 256 * 5 || work_bytes(0) != 0) return 2;
            for (std::size_t bytes : {1, 8, 256, 1280}) {
                for (std::uintptr_t at = 1 << 20; at < (1 << 20) + 512; at += 8) {
                    const auto from = reinterpret_cast<std::uintptr_t>(work_base(reinterpret_cast<void*>(at)));
                    if (from % 256 != 0 || from < at || from + bytes > at + work_bytes(bytes)) return 3;
                }
            }
            std::puts("whole");
        }
    """
    assert host_program(tmp_path, source) == "whole\n"


def test_row_constants_past_two_to_the_32_floats(tmp_path):
    # As many tiles as 2^25 tokens of 33 heads make (and twice as many of twice the rows): the last one's place, and its neighbour's.
    source = """
        #include "workspace.hpp"
        #include <cstdio>
        int main()
        {
            const unsigned tile = (1u << 25) + 3;  // as the kernel counts them
            const int width = 64;
            std::printf("%lld %lld %lld\\n", spectral::row_constants_at(tile, width), spectral::row_constants_at(tile - 1, width),
                        spectral::row_constants_at(2LL * tile, 2 * width));
        }
    """
    last = ((1 << 25) + 3) * 128
    assert host_program(tmp_path, source).split() == [str(last), str(last - 128), str(4 * last)]


def workspace(name, size, arrays, strides=None):
    """Bytes that a workspace query asks for; size: dtype, batch, queries, keys, heads, kv_heads, dim."""
    count = ctypes.c_size_t()
    native.call(name, *arrays, strides, *size, ctypes.byref(count))
    return 8 * count.value


def test_workspaces_hold_their_arrays_at_any_alignment():
    whole = lambda n: (n + 255) // 256 * 256
    # 16-bit arrays of unknown alignment are copied: 3 samples, 40 queries of 4 heads, 70 keys of 2, 24 values; 9 rows or more
    # and one split, so the copies are all there is.
    size = (1, 3, 40, 70, 4, 2, 24)
    copies = whole(3 * 40 * 4 * 24 * 2) + 2 * whole(3 * 70 * 2 * 24 * 2)
    assert workspace("spectral_cross_attention_workspace", size, [None] * 3) == copies + 256
    # Three bf16 parts of each in float32.
    assert workspace("spectral_cross_attention_workspace", (0, *size[1:]), [None] * 3) >= 3 * (3 * 40 * 4 + 2 * 3 * 70 * 2) * 24 * 2 + 256
    # Few rows over one range of keys, and a call without rows: nothing.
    assert workspace("spectral_cross_attention_workspace", (1, 3, 1, 70, 4, 2, 24), [None] * 3) == 0
    assert workspace("spectral_cross_attention_workspace", (1, 3, 0, 70, 4, 2, 24), [None] * 3) == 0
    assert workspace("spectral_cross_attention_backward_workspace", size, [None] * 4) >= copies + whole(3 * 40 * 4 * 24 * 2) + 256


@pytest.mark.parametrize("at", [8, 256])
def test_a_workspace_over_an_array_is_refused_at_any_alignment(at):
    # The arrays of a workspace start on the next whole 256 bytes, so the last of them ends past `count` values less 256 bytes.
    q = 1 << 20
    size = dict(dtype=0, batch=3, queries=40, keys=70, heads=4, kv_heads=2, dim=24)
    bytes_ = workspace("spectral_cross_attention_workspace", tuple(size.values()), [q, 1 << 21, 1 << 22])
    work = (1 << 25) + at
    for out in (work + bytes_ - 8, work - 8):
        with pytest.raises(ValueError, match="must not overlap"):
            native.call("spectral_cross_attention", *arguments(**size, out=out, work=work, stats=1 << 27))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("queries", "keys", "heads", "kv_heads", "dim"), [(1, 5000, 4, 2, 64), (12, 700, 2, 2, 64), (40, 2500, 4, 2, 64), (200, 300, 2, 2, 36),
                                                                    (33, 70, 2, 1, 13), (300, 150, 2, 2, 128), (2, 200, 130, 2, 32)])
@pytest.mark.parametrize("off", [8, 136])
def test_workspaces_of_any_alignment(off, queries, keys, heads, kv_heads, dim, dtype):
    q, k, v, dout = inputs(2, queries, keys, heads, kv_heads, dim, dtype)
    want = run(q, k, v, dout)
    size = (DTYPES.index(dtype), 2, queries, keys, heads, kv_heads, dim)
    p = lambda t: t.data_ptr() if t.numel() else None
    stream = torch.cuda.current_stream().cuda_stream

    def work(name, *arrays):  # 8 bytes past a multiple of 128, junk in it
        bytes_ = workspace(name, size, [p(t) for t in arrays])
        whole = torch.full((bytes_ + 512,), 255, dtype=torch.uint8, device="cuda")
        first = -whole.data_ptr() % 256 + off
        return whole, (whole.data_ptr() + first if bytes_ else None), first, first + bytes_

    out, dq, dk, dv = (torch.empty_like(t) for t in (q, q, k, v))
    stats = torch.empty(2, kv_heads, queries * (heads // kv_heads), 2, device="cuda")
    rest = torch.empty(0 if dtype == torch.float32 else q.numel(), dtype=torch.int8, device="cuda")
    scale = 1.0 / math.sqrt(dim)
    whole, at, first, last = work("spectral_cross_attention_workspace", q, k, v)
    native.call("spectral_cross_attention", p(q), p(k), p(v), None, None, 0, None, p(out), p(rest), p(stats), *size, scale, at, stream)
    assert torch.equal(out, want[0]) and bool((whole[:first] == 255).all()) and bool((whole[last:] == 255).all())
    whole, at, first, last = work("spectral_cross_attention_backward_workspace", dout, q, k, v)
    native.call("spectral_cross_attention_backward", p(dout), p(q), p(k), p(v), None, p(out), p(rest), p(stats), None, 0, None, p(dq), p(dk), p(dv),
                *size, scale, at, stream)
    assert all(torch.equal(g, w) for g, w in zip((dq, dk, dv), want[1:])) and bool((whole[:first] == 255).all()) and bool((whole[last:] == 255).all())


def test_cpu_tensors_are_refused():
    t = torch.zeros(1, 2, 2, 8)
    with pytest.raises(NotImplementedError, match="CPU"):
        cross_attention(t, t, t)


def test_a_module_without_whole_heads_is_refused():
    with pytest.raises(ValueError, match="do not divide"):
        CrossAttention(10, 8, 4)


@pytest.mark.gpu
def test_wrong_arguments_are_refused():
    q, k, v, _ = inputs(2, 5, 9, 4, 2, 16, torch.float32)
    with pytest.raises(RuntimeError, match="do not match"):
        cross_attention(q, k, v[:, :8])
    with pytest.raises(RuntimeError, match="do not match"):
        cross_attention(q, k[..., :8], v[..., :8])
    with pytest.raises(RuntimeError, match="do not match"):
        cross_attention(q[0], k, v)
    with pytest.raises(RuntimeError, match="v must be"):
        cross_attention(q, k, v.bfloat16())
    with pytest.raises(RuntimeError, match="must be float32"):
        cross_attention(q.double(), k.double(), v.double())
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        cross_attention(q[:, :, :3], k, v)
    with pytest.raises(ValueError, match="dim <= 128"):
        cross_attention(*[torch.zeros(1, 2, 1, 130, device="cuda")] * 3)
    with pytest.raises(RuntimeError, match="lengths must be"):
        cross_attention(q, k, v, lengths=torch.zeros(2, device="cuda"))
    with pytest.raises(RuntimeError, match="lengths must be"):
        cross_attention(q, k, v, lengths=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="lengths must be"):
        cross_attention(q, k, v, lengths=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="mask must be"):
        cross_attention(q, k, v, mask=torch.ones(2, 9, device="cuda"))
    with pytest.raises(RuntimeError, match="mask must be"):
        cross_attention(q, k, v, mask=torch.ones(2, 5, 9, dtype=torch.bool, device="cuda"))
