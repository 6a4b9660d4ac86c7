"""Group norm with an activation on channels-last fields: values, statistics and all gradients against
the formula in float64 (differentiated by torch's autograd), over types, group sizes that do not
fill a vector, sizes of both kernel forms (a group kept on chip, and read twice), checkpoints in 8
bits, strided and unaligned inputs, empty and non-finite ones; against differences; and the refusals.

Tolerances, relative to the result's norm: a 16-bit type rounds each value once, at most 2^-9
(bf16) or 2^-12 (f16) of it; float32 outputs carry a few roundings of the statistics (2^-24 each,
times 1 + |mean| / std for the difference from the mean) and about 4 units of the fast exponential:
64 units in all."""

import math

import pytest
import torch

import spectral
from spectral import native
from spectral.nn import GroupNormAct, group_norm_act

TOL = {torch.float32: 64 * 2.0 ** -24, torch.bfloat16: 2.0 ** -9 * 1.05, torch.float16: 2.0 ** -12 * 1.05}
DTYPES = list(TOL)


def act64(z, activation):
    if activation == "silu":
        return z * torch.sigmoid(z)
    if activation == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z / math.sqrt(2.0)))
    return z


def formula(x, groups, weight, bias, eps, activation, at=None):
    """The definition on float64 tensors; statistics of x, values at `at` (x if not given)."""
    b, c = x.shape[0], x.shape[-1]
    v = x.reshape(b, -1, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt(((v - mean) ** 2).mean((1, 3), keepdim=True) + eps)
    xhat = (v - mean) * rstd
    z = xhat.reshape(b, -1, c)
    if weight is not None:
        z = z * weight
    if bias is not None:
        z = z + bias
    return act64(z, activation).reshape(x.shape)


def gradients_at(x8, x, groups, weight, bias, eps, activation, dy):
    """dx, dweight, dbias at the restored input x8 with the statistics of x, in float64."""
    b, c = x.shape[0], x.shape[-1]
    v = x.reshape(b, -1, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt(((v - mean) ** 2).mean((1, 3), keepdim=True) + eps)
    xhat = ((x8.reshape(v.shape) - mean) * rstd).reshape(b, -1, c)
    z = (xhat * weight + bias).requires_grad_(True)
    (slope,) = torch.autograd.grad(act64(z, activation).sum(), z)
    dz = dy.reshape(b, -1, c) * slope
    t = (dz * weight).reshape(v.shape)
    h = xhat.reshape(v.shape)
    dx = rstd * (t - t.mean((1, 3), keepdim=True) - h * (t * h).mean((1, 3), keepdim=True))
    return dx.reshape(x.shape), (dz * xhat).sum((0, 1)), dz.sum((0, 1))


def close(got, want, tol, name=""):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    err, size = float((got - want).norm()), float(want.norm())
    assert err <= tol * size, f"{name}: {err / max(size, 1e-300):.3g} > {tol:.3g}"


def inputs(shape, dtype, seed, offset=1.0):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]
    x = torch.randn(*shape, generator=g) * torch.exp(0.5 * torch.randn(c, generator=g)) + offset * torch.randn(c, generator=g)
    weight, bias = 1.0 + 0.2 * torch.randn(c, generator=g), 0.3 * torch.randn(c, generator=g)
    dy = torch.randn(*shape, generator=g)
    return x.to(dtype).cuda(), weight.cuda(), bias.cuda(), dy.to(dtype).cuda()


# shape (batch, ..., channels), groups. Whole vectors and not; one point; one channel a group; a
# group of everything; several CTAs a cluster; the two-pass form (more than a cluster holds, or
# a group wider than a CTA's threads).
SHAPES = [((2, 1, 16), 4), ((3, 5, 7, 24), 3), ((1, 16, 16, 32), 8), ((2, 33, 30), 6), ((2, 19, 7), 7), ((4, 9, 64), 64),
          ((2, 300, 12), 1), ((1, 70, 70, 64), 8), ((2, 4000, 60), 6), ((1, 20000, 48), 2), ((2, 3, 4608), 2),
          ((1, 70000, 64), 1), ((1, 5, 5, 1), 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["none", "silu", "gelu"])
@pytest.mark.parametrize(("shape", "groups"), SHAPES)
def test_values_and_gradients(shape, groups, activation, dtype):
    x, weight, bias, dy = inputs(shape, dtype, sum(shape) + groups)
    leaves = [t.clone().requires_grad_(True) for t in (x, weight, bias)]
    y = group_norm_act(leaves[0], groups, leaves[1], leaves[2], eps=1e-5, activation=activation)
    got = torch.autograd.grad(y, leaves, dy)
    ref = [t.double().requires_grad_(True) for t in (x, weight, bias)]
    want_y = formula(ref[0], groups, ref[1], ref[2], 1e-5, activation)
    want = torch.autograd.grad(want_y, ref, dy.double())
    assert y.dtype == dtype and y.is_contiguous()
    v = x.double().reshape(shape[0], -1, groups, shape[-1] // groups)
    std = (v.var((1, 3), unbiased=False) + 1e-5).sqrt()
    worst = 1.0 + float((v.mean((1, 3)).abs() / std).max())
    single = TOL[torch.float32] * worst
    tol = TOL[dtype] + single
    close(y, want_y, tol, "y")
    # A group of few values has dx near zero against its terms: rstd (t - mean(t) - xhat mean(t xhat)).
    terms = float(((1.0 / std)[:, None, :, None] * (dy.double() * weight.double()).reshape(v.shape)).norm())
    err = float((got[0].double() - want[0]).norm())
    assert err <= tol * float(want[0].norm()) + single * 2 * terms, f"dx: {err:.3g}"
    # The parameters' gradients are float32 sums; bound by the sums of magnitudes.
    for name, g, w, size in (("dweight", got[1], want[1], (dy.double().abs() * 4).sum()),
                             ("dbias", got[2], want[2], (dy.double().abs() * 2).sum())):
        assert float((g.double() - w).abs().max()) <= single * float(w.abs().max()) + single * float(size) / shape[-1] ** 0.5, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("shape", "groups"), [((3, 5, 7, 24), 3), ((2, 33, 30), 6), ((1, 70, 70, 64), 8), ((2, 11, 136), 2),
                                               ((1, 70000, 64), 1), ((2, 500, 4608), 3)])
def test_gradients_from_an_8_bit_checkpoint(shape, groups, dtype):
    x, weight, bias, dy = inputs(shape, dtype, sum(shape) + groups)
    leaves = [t.clone().requires_grad_(True) for t in (x, weight, bias)]
    y = group_norm_act(leaves[0], groups, leaves[1], leaves[2], activation="gelu", checkpoint8=True)
    assert torch.equal(y, group_norm_act(x, groups, weight, bias, activation="gelu"))
    got = torch.autograd.grad(y, leaves, dy)
    restored = spectral.unpack8(*spectral.pack8(x), dtype=dtype)
    want = gradients_at(restored.double(), x.double(), groups, weight.double(), bias.double(), 1e-5, "gelu", dy.double())
    v = x.double().reshape(shape[0], -1, groups, shape[-1] // groups)
    worst = 1.0 + float((v.mean((1, 3)).abs() / (v.var((1, 3), unbiased=False) + 1e-5).sqrt()).max())
    single = TOL[torch.float32] * worst
    close(got[0], want[0], TOL[dtype] + single, "dx")
    for name, g, w, factor in (("dweight", got[1], want[1], 4), ("dbias", got[2], want[2], 2)):
        size = float((dy.double().abs() * factor).sum()) / shape[-1] ** 0.5
        assert float((g.double() - w).abs().max()) <= single * (float(w.abs().max()) + size), name


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_gradients_against_differences(activation):
    x, weight, bias, dy = inputs((2, 40, 24), torch.float32, 3)
    args = [x, weight, bias]
    leaves = [t.clone().requires_grad_(True) for t in args]
    grads = torch.autograd.grad(group_norm_act(leaves[0], 4, leaves[1], leaves[2], activation=activation), leaves, dy)
    step = 1e-2
    for i, grad in enumerate(grads):
        direction = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).cuda()
        ends = []
        for sign in (1.0, -1.0):
            moved = list(args)
            moved[i] = args[i] + sign * step * direction
            ends.append((group_norm_act(moved[0], 4, moved[1], moved[2], activation=activation).double() * dy.double()).sum())
        slope = float(ends[0] - ends[1]) / (2 * step)
        # Second-order remainder step^2 and rounding 1e-6 / step, against gradients of this norm.
        assert abs(slope - float((grad.double() * direction.double()).sum())) <= 2e-3 * float(grad.double().norm() * direction.double().norm())


@pytest.mark.gpu
def test_statistics_of_a_large_mean_do_not_cancel():
    # Offsets of 3000 standard deviations: the one-pass form sum x^2 - n mean^2 would lose the variance.
    for shape in [(2, 600, 16), (1, 70000, 64)]:
        g = torch.Generator().manual_seed(7)
        x = (torch.randn(*shape, generator=g) + 3000.0).cuda()
        y = group_norm_act(x, 1)
        close(y, formula(x.double(), 1, None, None, 1e-5, "none"), 64 * 3001 * 2.0 ** -24)


@pytest.mark.gpu
def test_optional_parameters_constant_inputs_and_eps():
    x = torch.full((2, 7, 8), 3.0, device="cuda")
    bias = torch.arange(8.0, device="cuda")
    assert torch.equal(group_norm_act(x, 2, None, bias), bias.expand(2, 7, 8))
    x = inputs((2, 9, 8), torch.float32, 1)[0]
    close(group_norm_act(x, 2, eps=0.5), formula(x.double(), 2, None, None, 0.5, "none"), 1e-5)
    leaf = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(group_norm_act(leaf, 2, eps=0.5).sum(), leaf)
    assert float(dx.abs().max()) < 1e-5  # a sum over a group of normalised values does not move


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["resident", "two passes"])
def test_non_finite_values_stay_in_their_group(form):
    shape, groups = ((2, 50, 16), 2) if form == "resident" else ((2, 70000, 128), 2)
    x, weight, bias, dy = inputs(shape, torch.float32, 11)
    clean = group_norm_act(x, groups, weight, bias, activation="silu")
    x[0, 3, 1] = float("nan")
    x[1, 4, shape[-1] - 1] = float("inf")
    leaf = x.clone().requires_grad_(True)
    y = group_norm_act(leaf, groups, weight, bias, activation="silu")
    half = shape[-1] // 2
    assert y[0, :, :half].isnan().all() and y[1, :, half:].isnan().all()
    assert torch.equal(y[0, :, half:], clean[0, :, half:]) and torch.equal(y[1, :, :half], clean[1, :, :half])
    (dx,) = torch.autograd.grad(y, leaf, dy)
    assert dx[0, :, half:].isfinite().all() and dx[1, :, :half].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_unaligned_inputs(dtype):
    g = torch.Generator().manual_seed(2)
    first = torch.randn(3, 24, 10, 9, generator=g).to(dtype).cuda()  # channels first in memory
    weight, bias = torch.randn(24, generator=g).cuda(), torch.randn(24, generator=g).cuda()
    flat = torch.randn(2 * 24 * 11 + 1, generator=g).to(dtype).cuda()
    for x in (first.permute(0, 2, 3, 1), first[:, :, ::2].permute(0, 2, 3, 1), flat[1:].view(2, 11, 24),
              first.permute(0, 2, 3, 1)[..., 8:16].repeat(1, 1, 1, 3)):
        leaf = x.detach().requires_grad_(True)
        y = group_norm_act(leaf, 4, weight, bias, activation="gelu")
        same = x.contiguous().clone().requires_grad_(True)
        want = group_norm_act(same, 4, weight, bias, activation="gelu")
        close(y, want, TOL[torch.float32] + (0 if dtype == torch.float32 else TOL[dtype]))
        dy = torch.randn(y.shape, generator=g).to(dtype).cuda()
        close(torch.autograd.grad(y, leaf, dy)[0], torch.autograd.grad(want, same, dy)[0],
              4 * TOL[torch.float32] + (0 if dtype == torch.float32 else TOL[dtype]))


@pytest.mark.gpu
def test_empty_inputs():
    weight = torch.ones(8, device="cuda", requires_grad=True)
    for shape in [(0, 5, 8), (2, 0, 8)]:
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = group_norm_act(x, 2, weight, activation="silu")
        assert y.shape == shape
        dx, dw = torch.autograd.grad(y.sum(), (x, weight))
        assert dx.shape == shape and torch.equal(dw, torch.zeros_like(dw))


@pytest.mark.gpu
def test_the_same_bits_every_time_and_on_a_side_stream():
    for shape, groups in [((4, 4000, 64), 8), ((1, 70000, 64), 1)]:
        x, weight, bias, dy = inputs(shape, torch.bfloat16, 4)

        def step():
            leaves = [t.clone().requires_grad_(True) for t in (x, weight, bias)]
            y = group_norm_act(leaves[0], groups, leaves[1], leaves[2], activation="gelu", checkpoint8=True)
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))

        first = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = step()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.gpu
def test_past_two_to_the_31_values():
    points = (1 << 24) + 5
    x = torch.zeros(2, points, 64, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(1)
    x[1, -1000:] = torch.randn(1000, 64, generator=g).to(torch.bfloat16).cuda()
    y = group_norm_act(x, 2)
    v = x[1, -1000:].double().reshape(1000, 2, 32)
    n = points * 32
    mean = v.sum((0, 2)) / n
    var = (v ** 2).sum((0, 2)) / n - mean ** 2
    want = (v - mean[:, None]) / torch.sqrt(var[:, None] + 1e-5)
    close(y[1, -1000:].reshape(1000, 2, 32), want, TOL[torch.bfloat16] + 2.0 ** -20)
    assert float(y[0].abs().max()) == 0.0


@pytest.mark.gpu
def test_module():
    norm = GroupNormAct(4, 16, activation="silu", checkpoint8=True, device="cuda")
    x = inputs((2, 6, 6, 16), torch.bfloat16, 8)[0]
    assert torch.equal(norm(x), group_norm_act(x, 4, norm.weight, norm.bias, activation="silu"))
    norm(x).float().square().mean().backward()
    assert norm.weight.grad.shape == (16,) and norm.bias.grad.shape == (16,)
    assert "checkpoint8=True" in repr(norm)


def forward_args(**change):
    a = dict(x=4096, weight=None, bias=None, y=8192, mean=None, rstd=None, codes=None, scales=None, dtype=0, channels_first=0, batch=1,
             points=4, channels=8, groups=2, eps=1e-5, activation=0, work=65536, stream=None)
    a.update(change)
    return tuple(a.values())


@pytest.mark.parametrize(
    ("change", "message"),
    [(dict(dtype=5), "dtype must be"), (dict(activation=9), "activation must be"), (dict(groups=3), "groups dividing channels"),
     (dict(groups=0), "groups dividing channels"), (dict(eps=-1.0), "eps must be"), (dict(eps=math.nan), "eps must be"), (dict(batch=-1), "batch >= 0"), (dict(work=None), "must be given"),
     (dict(mean=4096), "mean with rstd"), (dict(codes=4096), "codes with scales"), (dict(x=4098), "aligned"),
     (dict(y=4096 + 64), "must not overlap"), (dict(channels_first=1, points=5), "channels first needs"),
     (dict(channels_first=1, codes=1 << 20, scales=1 << 21), "channels first needs"), (dict(batch=1 << 31, x=1 << 60), "at most 2\\^30 samples")])
def test_the_c_abi_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        native.call("spectral_group_norm_act", *forward_args(**change))


@pytest.mark.parametrize(
    ("change", "message"),
    [(dict(x=None), "either x or codes"), (dict(codes=4096, scales=4096), "either x or codes"), (dict(mean=None), "must be given"),
     (dict(dx=1 << 20), "must not overlap"), (dict(groups=5), "groups dividing channels"), (dict(dy=(1 << 20) + 1), "aligned")])
def test_the_c_abi_refuses_backward(change, message):
    a = dict(dy=1 << 20, x=1 << 21, codes=None, scales=None, weight=None, bias=None, mean=4096, rstd=8192, dx=1 << 22,
             dweight=None, dbias=None, dtype=0, batch=1, points=4, channels=8, groups=2, activation=0, work=65536, stream=None)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        native.call("spectral_group_norm_act_backward", *a.values())


def test_cpu_tensors_are_refused():
    with pytest.raises(NotImplementedError, match="CPU"):
        group_norm_act(torch.zeros(2, 4, 8), 2)


@pytest.mark.gpu
def test_wrong_arguments_are_refused():
    x = torch.zeros(2, 4, 8, device="cuda")
    with pytest.raises(RuntimeError, match="groups must divide"):
        group_norm_act(x, 3)
    with pytest.raises(RuntimeError, match="activation must be"):
        group_norm_act(x, 2, activation="relu")
    with pytest.raises(RuntimeError, match="weight must be a float32 tensor of 8"):
        group_norm_act(x, 2, torch.ones(4, device="cuda"))
    with pytest.raises(RuntimeError, match="weight must be a float32 tensor of 8"):
        group_norm_act(x, 2, torch.ones(8, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        group_norm_act(x.double(), 2)
    with pytest.raises(RuntimeError, match="must be \\(batch"):
        group_norm_act(x[0, 0], 2)


# Fields with the channels first in memory, as a convolution leaves them: (batch, channels, points along two axes), groups.
FIRST = [((2, 16, 8, 8), 4), ((3, 24, 12, 16), 3), ((2, 8, 1, 8), 1), ((1, 72, 64, 96), 72), ((1, 136, 50, 40), 2), ((2, 64, 72, 1000), 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("checkpoint8", [False, True])
@pytest.mark.parametrize(("shape", "groups"), FIRST)
def test_channels_first_in_memory(shape, groups, checkpoint8, dtype):
    b, c, *points = shape
    x, weight, bias, dy = inputs((b, *points, c), dtype, sum(shape) + groups)
    first = x.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)  # the same values, channels first
    dy_first = dy.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    leaves = [t.detach().requires_grad_(True) for t in (first, weight, bias)]
    y = group_norm_act(leaves[0], groups, leaves[1], leaves[2], activation="gelu", checkpoint8=checkpoint8)
    assert y.is_contiguous() and y.shape == x.shape
    got = torch.autograd.grad(y, leaves, dy_first)
    close(group_norm_act(first, groups, weight, bias, activation="gelu"), y, TOL[torch.float32] + (0 if dtype == torch.float32 else TOL[dtype]))
    close(y, formula(x.double(), groups, weight.double(), bias.double(), 1e-5, "gelu"),
          TOL[dtype] + first_single(x, groups))
    at = spectral.unpack8(*spectral.pack8(x), dtype=dtype) if checkpoint8 else x
    want = gradients_at(at.double(), x.double(), groups, weight.double(), bias.double(), 1e-5, "gelu", dy.double())
    single = first_single(x, groups)
    v = x.double().reshape(b, -1, groups, c // groups)
    std = (v.var((1, 3), unbiased=False) + 1e-5).sqrt()
    terms = float(((1.0 / std)[:, None, :, None] * (dy.double() * weight.double()).reshape(v.shape)).norm())
    err = float((got[0].double() - want[0]).norm())
    assert err <= (TOL[dtype] + single) * float(want[0].norm()) + single * 2 * terms, f"dx: {err:.3g}"
    for name, g, w, factor in (("dweight", got[1], want[1], 4), ("dbias", got[2], want[2], 2)):
        size = float((dy.double().abs() * factor).sum()) / c ** 0.5
        assert float((g.double() - w).abs().max()) <= single * (float(w.abs().max()) + size), name


def first_single(x, groups):
    v = x.double().reshape(x.shape[0], -1, groups, x.shape[-1] // groups)
    std = (v.var((1, 3), unbiased=False) + 1e-5).sqrt()
    return TOL[torch.float32] * (1.0 + float((v.mean((1, 3)).abs() / std).max()))


@pytest.mark.gpu
def test_channels_first_statistics_of_a_large_mean_and_non_finite_values():
    g = torch.Generator().manual_seed(7)
    x = (torch.randn(2, 16, 40, 30, generator=g) + 3000.0).cuda().permute(0, 2, 3, 1)
    close(group_norm_act(x, 2), formula(x.double(), 2, None, None, 1e-5, "none"), 64 * 3001 * 2.0 ** -24)
    clean = group_norm_act(x, 2)
    x[0, 3, 1, 2] = float("nan")
    y = group_norm_act(x, 2)
    assert y[0, ..., :8].isnan().all() and torch.equal(y[0, ..., 8:], clean[0, ..., 8:]) and torch.equal(y[1], clean[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("batch", "points", "channels"), [(1, 8, 8), (3, 200, 24), (2, 5000, 136), (70000, 8, 8)])
def test_the_c_abi_lays_channels_last(batch, points, channels, dtype):
    x = torch.randn(batch, channels, points, generator=torch.Generator().manual_seed(points)).to(dtype).cuda()
    y = torch.empty(batch, points, channels, dtype=dtype, device="cuda")
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    native.call("spectral_channels_last", x.data_ptr(), y.data_ptr(), code, batch, points, channels, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(y, x.transpose(1, 2))


@pytest.mark.parametrize(
    ("change", "message"),
    [(dict(dtype=4), "dtype must be"), (dict(points=5), "points of 16 bytes"), (dict(channels=12), "multiple of 8"), (dict(x=4104), "aligned"),
     (dict(x=None), "needs"), (dict(y=4096 + 32), "must not overlap"), (dict(batch=-1), "batch >= 0")])
def test_the_c_abi_refuses_to_lay_channels_last(change, message):
    a = dict(x=4096, y=1 << 20, dtype=0, batch=2, points=8, channels=8, stream=None)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        native.call("spectral_channels_last", *a.values())


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint8", [False, True])
def test_gradients_of_gradients_under_a_constant_upstream_gradient_are_refused(checkpoint8):
    x, weight, bias, _ = inputs((2, 9, 16), torch.float32, 5)
    leaves = [t.requires_grad_(True) for t in (x, weight, bias)]

    def layer():
        return group_norm_act(leaves[0], 2, leaves[1], leaves[2], activation="gelu", checkpoint8=checkpoint8)

    y = layer()
    plain = torch.autograd.grad(y.sum(), leaves, retain_graph=True)
    grads = torch.autograd.grad(y.sum(), leaves, create_graph=True)
    for g, p in zip(grads, plain):  # the values are there, without a way back through them
        assert torch.equal(g, p)
        for wrt in leaves:
            with pytest.raises(RuntimeError, match="not differentiable itself"):
                torch.autograd.grad(y.mean() + g.pow(2).sum(), wrt, retain_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable itself"):
        (layer().mean() + grads[0].pow(2).sum()).backward()
    # Through two layers, and with an upstream gradient that depends on another tensor.
    scale = torch.ones((), device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad((group_norm_act(layer(), 4) * scale).sum(), leaves[0], create_graph=True)
    for wrt in (leaves[0], scale):
        with pytest.raises(RuntimeError, match="not differentiable itself"):
            torch.autograd.grad(g.sum(), wrt, retain_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_tangents_are_refused(which, grad_mode):
    args = list(inputs((2, 9, 16), torch.float32, 5)[:3])
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        args[which] = torch.autograd.forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            group_norm_act(args[0], 2, args[1], args[2], activation="gelu")


@pytest.mark.parametrize("change", [dict(weight=(1 << 20) + 2), dict(bias=(1 << 20) + 1), dict(mean=(1 << 20) + 2, rstd=1 << 21),
                                    dict(mean=1 << 20, rstd=(1 << 21) + 2), dict(codes=1 << 20, scales=(1 << 21) + 2)])
def test_the_c_abi_refuses_unaligned_float_arrays(change):
    with pytest.raises(ValueError, match="aligned"):
        native.call("spectral_group_norm_act", *forward_args(**change))


@pytest.mark.parametrize(
    ("change", "message"),
    [({name: (1 << 24) + 2}, "aligned") for name in ("weight", "bias", "mean", "rstd", "dweight", "dbias")]
    + [(dict(x=None, codes=1 << 21, scales=(1 << 23) + 2), "aligned"), (dict(dweight=(1 << 24) + 2, points=0), "aligned")])
def test_the_c_abi_refuses_unaligned_float_arrays_backward(change, message):
    backward_refuses(change, message)


@pytest.mark.parametrize("change", [dict(codes=(1 << 22) + 100, scales=1 << 23), dict(codes=1 << 23, scales=(1 << 22) + 124)])
def test_the_c_abi_refuses_dx_over_the_checkpoint(change):
    backward_refuses(dict(x=None, **change), "must not overlap the checkpoint")


def backward_refuses(change, message):
    a = dict(dy=1 << 20, x=1 << 21, codes=None, scales=None, weight=None, bias=None, mean=4096, rstd=8192, dx=1 << 22,
             dweight=None, dbias=None, dtype=0, batch=1, points=4, channels=8, groups=2, activation=0, work=65536, stream=None)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        native.call("spectral_group_norm_act_backward", *a.values())


# The two-pass form where rows are no whole 16-byte pieces (single values; pairs), and wide rows in tiles that hold whole groups.
TWO_PASS = [((2, 70001, 37), 1), ((2, 50001, 54), 6), ((2, 1100, 4608), 144)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("shape", "groups"), TWO_PASS)
def test_two_passes_over_odd_and_wide_rows(shape, groups, dtype):
    assert math.prod(shape) * (4 if dtype == torch.float32 else 2) > 8 << 20  # smaller arrays stay on chip
    test_values_and_gradients(shape, groups, "gelu", dtype)
    test_gradients_from_an_8_bit_checkpoint(shape, groups, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint8", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_two_passes_over_unaligned_views(dtype, checkpoint8):
    x, weight, bias, dy = inputs((2, 40001, 64), dtype, 6)

    def step(x, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, weight, bias)]
        y = group_norm_act(leaves[0], 8, leaves[1], leaves[2], activation="silu", checkpoint8=checkpoint8)
        return (y, *torch.autograd.grad(y, leaves, dy))

    def shifted(t, by):  # the same values a few elements off a 16-byte boundary
        flat = torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)
        flat[by:] = t.reshape(-1)
        return flat[by:].view(t.shape)

    want = step(x, dy)
    for by in (1, 2):
        for got, w in zip(step(shifted(x, by), shifted(dy, by)), want):
            # Sums in another order, and a rounding that may then fall the other way.
            close(got, w, 4 * TOL[torch.float32] + (0 if got.dtype == torch.float32 else TOL[dtype]))
