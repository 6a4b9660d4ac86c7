"""The gated feed-forward block: values and all gradients against the formula in float64
(differentiated by torch's autograd), over types, sizes that are no multiple of a tile, one token to
many, unaligned and strided operands, 8-bit checkpoints, non-finite values; against differences;
and the refusals; and FNOBlock, which runs the pointwise operators around the spectral convolution.

Tolerances, relative to the result's norm. 16-bit types round the hidden values and the result
once each. Over many values a rounding is 2^-9 (bf16) or 2^-12 (f16) of the norm or less, so twice
that bounds both; a result of a few values has to allow the worst case of each, 2^-8 or 2^-11, and
f16's subnormal unit 2^-24. float32 products accumulate passes of 128 values, cut at 2^-23 per 16 of them: at most
8 x 2^-23 a product, and a result is a chain of at most three."""

import math

import pytest
import torch

import spectral
from spectral import native
from spectral.nn import FNOBlock, GatedMLP, gated_mlp

TOL = {torch.float32: 24 * 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = list(TOL)


def act64(z, activation):
    if activation == "silu":
        return z * torch.sigmoid(z)
    if activation == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z / math.sqrt(2.0)))
    return z


def formula(x, w_gate, w_up, w_down, activation):
    return (act64(x @ w_gate.T, activation) * (x @ w_up.T)) @ w_down.T


def inputs(tokens, channels, hidden, outputs, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + tokens + 7 * channels + 11 * hidden)
    shapes = [(tokens, channels), (hidden, channels), (hidden, channels), (outputs, hidden), (tokens, outputs)]
    scale = [1.0, channels ** -0.5, channels ** -0.5, hidden ** -0.5, 1.0]
    return [(torch.randn(*s, generator=g) * k).to(dtype).cuda() for s, k in zip(shapes, scale)]


def close(got, want, tol, name=""):
    dtype, few = got.dtype, got.numel() < 16
    got, want = got.detach().double(), want.detach().double()
    err, size = float((got - want).norm()), float(want.norm())
    least = 0.0
    if few and dtype != torch.float32:
        tol, least = 2 * tol, 2.0 ** -22 if dtype == torch.float16 else 0.0
    assert err <= tol * size + least, f"{name}: {err / max(size, 1e-300):.3g} > {tol:.3g}"


# tokens, channels, hidden, outputs: one of everything; the few-token form and its edge; sizes around
# the tiles of 64, 128 and 256; unlike inputs and outputs; rows that are no 16-byte pieces.
SIZES = [(1, 1, 1, 1), (1, 64, 128, 64), (3, 50, 33, 70), (8, 512, 96, 200), (9, 64, 64, 64), (17, 24, 40, 8),
         (128, 64, 128, 64), (129, 65, 127, 33), (200, 130, 300, 129), (1000, 100, 270, 100), (513, 256, 512, 257),
         (300, 64, 1024, 320), (2048, 16, 16, 16), (640, 520, 72, 264)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["none", "silu", "gelu"])
@pytest.mark.parametrize(("tokens", "channels", "hidden", "outputs"), SIZES)
def test_values_and_gradients(tokens, channels, hidden, outputs, activation, dtype):
    *args, dy = inputs(tokens, channels, hidden, outputs, dtype)
    want_y = formula(*[a.double() for a in args], activation)
    close(gated_mlp(*args, activation=activation), want_y, TOL[dtype], "y without gradients")
    leaves = [a.clone().requires_grad_(True) for a in args]
    y = gated_mlp(*leaves, activation=activation)
    assert y.dtype == dtype and y.shape == (tokens, outputs)
    got = torch.autograd.grad(y, leaves, dy)
    ref = [a.double().requires_grad_(True) for a in args]
    want = torch.autograd.grad(formula(*ref, activation), ref, dy.double())
    close(y, want_y, TOL[dtype], "y")
    # dx adds two products and the gate's slope may cancel against 1: bounded by the two parts' norms.
    for name, g, w in zip(("dx", "dw_gate", "dw_up", "dw_down"), got, want):
        assert g.dtype == dtype and g.shape == w.shape
        close(g, w, TOL[dtype] * (2 if name == "dx" and channels * hidden < 64 else 1), name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("tokens", "channels", "hidden", "outputs"), [(5, 64, 96, 64), (700, 64, 128, 64), (333, 200, 130, 72),
                                                                       (150, 37, 50, 37)])
def test_gradients_from_an_8_bit_checkpoint(tokens, channels, hidden, outputs, dtype):
    *args, dy = inputs(tokens, channels, hidden, outputs, dtype)
    leaves = [a.clone().requires_grad_(True) for a in args]
    y = gated_mlp(*leaves, activation="gelu", checkpoint8=True)
    assert torch.equal(y, gated_mlp(*args, activation="gelu"))
    got = torch.autograd.grad(y, leaves, dy)
    restored = spectral.unpack8(*spectral.pack8(args[0]), dtype=dtype)
    ref = [a.double().requires_grad_(True) for a in (restored, *args[1:])]
    want = torch.autograd.grad(formula(*ref, "gelu"), ref, dy.double())
    for name, g, w in zip(("dx", "dw_gate", "dw_up", "dw_down"), got, want):
        close(g, w, TOL[dtype], name)


@pytest.mark.gpu
def test_gradients_against_differences():
    *args, dy = inputs(40, 24, 36, 20, torch.float32)
    leaves = [a.clone().requires_grad_(True) for a in args]
    grads = torch.autograd.grad(gated_mlp(*leaves), leaves, dy)
    step = 1e-2
    for i, grad in enumerate(grads):
        direction = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).cuda()
        direction /= direction.norm() / args[i].norm()
        ends = []
        for sign in (1.0, -1.0):
            moved = list(args)
            moved[i] = args[i] + sign * step * direction
            ends.append((gated_mlp(*moved).double() * dy.double()).sum())
        slope = float(ends[0] - ends[1]) / (2 * step)
        # The remainder is of order step^2, the values' rounding 1e-6 / step.
        assert abs(slope - float((grad.double() * direction.double()).sum())) <= 2e-3 * float(grad.double().norm() * direction.double().norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_unaligned_and_batched_operands(dtype):
    *args, dy = inputs(60, 40, 48, 40, dtype)
    want = gated_mlp(*args)

    def shifted(t):  # the same values one element off a 16-byte boundary
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    exact = 0.0 if dtype != torch.float32 else 1e-7
    for variant in ([shifted(a) for a in args], [a.t().contiguous().t() for a in args], [args[0].view(3, 4, 5, 40), *args[1:]]):
        close(gated_mlp(*variant).reshape(want.shape), want, exact)
        leaves = [a.detach().requires_grad_(True) for a in variant]
        y = gated_mlp(*leaves)
        plain = [a.clone().requires_grad_(True) for a in args]
        grads = torch.autograd.grad(y, leaves, dy.reshape(y.shape))
        for g, w in zip(grads, torch.autograd.grad(gated_mlp(*plain), plain, dy)):
            close(g.reshape(w.shape), w, exact)
    one = [a.clone() for a in args]
    close(gated_mlp(shifted(one[0][:2]), *map(shifted, one[1:])), gated_mlp(one[0][:2].clone(), *one[1:]), TOL[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [6, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_tokens_stay_in_their_rows(tokens, dtype):
    *args, dy = inputs(tokens, 64, 96, 64, dtype)
    clean = gated_mlp(*args)
    args[0][2, 5] = float("nan")
    args[0][4, 0] = float("inf")
    leaf = args[0].clone().requires_grad_(True)
    y = gated_mlp(leaf, *args[1:])
    rest = [i for i in range(tokens) if i not in (2, 4)]
    assert y[2].isnan().all() and not y[4].isfinite().any()
    assert torch.equal(y[rest], clean[rest])
    (dx,) = torch.autograd.grad(y, leaf, dy)
    assert dx[rest].isfinite().all() and dx[2].isnan().all()


@pytest.mark.gpu
def test_float32_beyond_the_16_bit_ranges():
    # The three parts of a float32 have its range: large and small operands keep float32's accuracy.
    *args, _ = inputs(100, 40, 48, 40, torch.float32)
    args[0] *= 1e18
    args[1] *= 1e-20
    args[2] *= 1e10
    args[3] *= 1e-12
    close(gated_mlp(*args, activation="none"), formula(*[a.double() for a in args], "none"), TOL[torch.float32])


@pytest.mark.gpu
def test_no_tokens():
    *args, dy = inputs(0, 8, 16, 24, torch.bfloat16)
    leaves = [a.requires_grad_(True) for a in args]
    y = gated_mlp(*leaves)
    assert y.shape == (0, 24)
    for g, a in zip(torch.autograd.grad(y, leaves, dy), leaves):
        assert g.shape == a.shape and float(g.abs().sum()) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_same_bits_every_time_and_on_a_side_stream(dtype):
    *args, dy = inputs(5000, 96, 160, 96, dtype)

    def step():
        leaves = [a.clone().requires_grad_(True) for a in args]
        y = gated_mlp(*leaves, activation="gelu", checkpoint8=True)
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
    tokens = (1 << 25) + 77
    x = torch.zeros(tokens, 64, dtype=torch.bfloat16, device="cuda")
    *args, dy = inputs(200, 64, 16, 8, torch.bfloat16)
    x[-200:] = args[0]
    y = gated_mlp(x, *args[1:])
    close(y[-200:], formula(*[a.double() for a in args], "silu"), TOL[torch.bfloat16])
    assert float(y[:1000].abs().max()) == 0.0


@pytest.mark.gpu
def test_module_and_training_step():
    torch.manual_seed(0)
    mlp = GatedMLP(16, 48, activation="silu", checkpoint8=True, device="cuda")
    x, target = torch.randn(500, 16, device="cuda"), torch.randn(500, 16, device="cuda")
    opt = torch.optim.SGD(mlp.parameters(), lr=0.05)
    losses = []
    for _ in range(3):
        loss = ((mlp(x) - target) ** 2).mean()
        losses.append(loss.item())
        opt.zero_grad()
        loss.backward()
        opt.step()
    assert losses[2] < losses[1] < losses[0]
    assert "16, 48, 16" in repr(mlp)


def block64(block, u):
    """FNOBlock in float64 with torch's FFT."""
    conv, norm, mlp = block.conv, block.norm, block.mlp
    n1, n2 = u.shape[-2:]
    spec = torch.fft.rfft2(u)
    modes = torch.cat([spec[..., :conv.m1, :conv.m2], spec[..., n1 - conv.m1:, :conv.m2]], dim=-2)
    out = torch.einsum("bikl,iokl->bokl", modes, conv.weight.to(torch.complex128))
    full = torch.zeros(*u.shape[:2], n1, n2 // 2 + 1, dtype=out.dtype, device=u.device)
    full[..., :conv.m1, :conv.m2] = out[..., :conv.m1, :]
    full[..., n1 - conv.m1:, :conv.m2] = out[..., conv.m1:, :]
    v = torch.fft.irfft2(full, s=(n1, n2)).permute(0, 2, 3, 1)
    g = v.reshape(v.shape[0], -1, norm.groups, v.shape[-1] // norm.groups)
    mean = g.mean((1, 3), keepdim=True)
    g = (g - mean) / torch.sqrt(((g - mean) ** 2).mean((1, 3), keepdim=True) + norm.eps)
    z = act64(g.reshape(v.shape) * norm.weight.double() + norm.bias.double(), norm.activation)
    z = formula(z, mlp.w_gate.double(), mlp.w_up.double(), mlp.w_down.double(), mlp.activation)
    return u + z.permute(0, 3, 1, 2)


@pytest.mark.gpu
@pytest.mark.parametrize(("dtype", "tol"), [(torch.float32, 2e-5), (torch.bfloat16, 2e-2)])
def test_fno_block(dtype, tol):
    torch.manual_seed(1)
    block = FNOBlock(16, 32, 8, 8, groups=4, device="cuda", dtype=dtype)
    u = torch.randn(2, 16, 32, 32, device="cuda")
    up = torch.randn_like(u)
    leaf = u.clone().requires_grad_(True)
    y = block(leaf)
    params = [block.norm.weight, block.norm.bias, block.mlp.w_gate, block.mlp.w_up, block.mlp.w_down]
    got = torch.autograd.grad(y, [leaf, *params], up)
    ref = u.double().requires_grad_(True)
    want_y = block64(block, ref)
    want = torch.autograd.grad(want_y, [ref, *params], up.double())
    close(y, want_y, tol)
    for g, w in zip(got, want):
        close(g, w, tol)


@pytest.mark.gpu
def test_fno_block_trains_with_8_bit_checkpoints():
    torch.manual_seed(2)
    block = FNOBlock(16, 32, 8, 8, groups=4, checkpoint8=True, device="cuda")
    u, target = torch.randn(4, 16, 32, 32, device="cuda"), torch.randn(4, 16, 32, 32, device="cuda")
    opt = torch.optim.SGD(block.parameters(), lr=0.05)
    losses = []
    for _ in range(3):
        loss = ((block(u) - target) ** 2).mean()
        losses.append(loss.item())
        opt.zero_grad()
        loss.backward()
        opt.step()
    assert losses[2] < losses[1] < losses[0]


def arguments(**change):
    a = dict(x=1 << 20, w_gate=1 << 21, w_up=1 << 22, w_down=1 << 23, y=1 << 24, dtype=1, tokens=4, channels=8, hidden=16,
             outputs=8, activation=1, work=1 << 25, stream=None)
    a.update(change)
    return tuple(a.values())


@pytest.mark.parametrize(
    ("change", "message"),
    [(dict(dtype=3), "dtype must be"), (dict(tokens=-1), "tokens"), (dict(hidden=0), "hidden"), (dict(activation=3), "activation must be"),
     (dict(w_up=None), "null array"), (dict(x=(1 << 20) + 1), "aligned"), (dict(y=(1 << 20) + 32), "must not overlap"),
     (dict(work=None), "null array"), (dict(tokens=1 << 31), "tokens")])
def test_the_c_abi_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        native.call("spectral_gated_mlp", *arguments(**change))


@pytest.mark.parametrize(
    ("change", "message"),
    [(dict(x=None), "either x or codes"), (dict(codes=4096, scales=4096), "either x or codes"), (dict(dw_up=None), "null array"),
     (dict(dx=1 << 20), "must not overlap"), (dict(dx=None), "must be given"), (dict(dtype=-1), "dtype must be"),
     (dict(dw_down=(1 << 29) + 1), "aligned")])
def test_the_c_abi_refuses_backward(change, message):
    a = dict(dy=1 << 20, x=1 << 21, codes=None, scales=None, w_gate=1 << 22, w_up=1 << 23, w_down=1 << 24, dx=1 << 25,
             dw_gate=1 << 26, dw_up=1 << 27, dw_down=1 << 29, dtype=1, tokens=4, channels=8, hidden=16, outputs=8, activation=1,
             work=1 << 30, stream=None)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        native.call("spectral_gated_mlp_backward", *a.values())


def test_cpu_tensors_are_refused():
    w = torch.zeros(16, 8)
    with pytest.raises(NotImplementedError, match="CPU"):
        gated_mlp(torch.zeros(2, 8), w, w, w.t())


@pytest.mark.gpu
def test_wrong_arguments_are_refused():
    x, w, d = torch.zeros(2, 8, device="cuda"), torch.zeros(16, 8, device="cuda"), torch.zeros(4, 16, device="cuda")
    with pytest.raises(RuntimeError, match="do not match"):
        gated_mlp(x, w, w[:8], d)
    with pytest.raises(RuntimeError, match="do not match"):
        gated_mlp(x[:, :4], w, w, d)
    with pytest.raises(RuntimeError, match="w_down must be"):
        gated_mlp(x, w, w, d.bfloat16())
    with pytest.raises(RuntimeError, match="activation must be"):
        gated_mlp(x, w, w, d, activation="tanh")
    with pytest.raises(RuntimeError, match="must be matrices"):
        gated_mlp(x, w[0], w, d)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        gated_mlp(x.double(), w.double(), w.double(), d.double())


@pytest.mark.gpu
def test_gradients_of_gradients_are_refused_and_unused_ones_cost_nothing_else():
    *args, dy = inputs(20, 16, 24, 16, torch.float32)
    leaves = [a.clone().requires_grad_(True) for a in args]
    up = dy.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable itself"):
        torch.autograd.grad(gated_mlp(*leaves), leaves, up, create_graph=True)
    with torch.no_grad():
        assert gated_mlp(*leaves).grad_fn is None
    # Only some inputs want gradients.
    frozen = [args[0].clone().requires_grad_(True), *args[1:]]
    (dx,) = torch.autograd.grad(gated_mlp(*frozen), frozen[:1], dy)
    assert torch.equal(dx, torch.autograd.grad(gated_mlp(*leaves), leaves[:1], dy)[0])


@pytest.mark.gpu
@pytest.mark.parametrize(("tokens", "channels"), [(4, 64), (1000, 64), (1000, 200)])
def test_a_captured_training_step_replays_with_new_inputs(tokens, channels):
    # Norm, feed-forward block and their backward passes in one CUDA graph, after a first call outside it.
    *args, dy = inputs(tokens, channels, 96, channels, torch.bfloat16)
    x = args[0].view(1, tokens, channels)
    weight = torch.ones(channels, device="cuda")

    def step(x, dy):
        leaves = [x.detach().requires_grad_(True), weight.detach().requires_grad_(True), *(a.detach().requires_grad_(True) for a in args[1:])]
        y = gated_mlp(spectral.nn.group_norm_act(leaves[0], 2, leaves[1], activation="gelu", checkpoint8=True), *leaves[2:])
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    static_x, static_dy = x.clone(), dy.view(1, tokens, channels).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static_x, static_dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static_x, static_dy)
    new_x, new_dy = x * 0.5 + 0.25, static_dy.flip(1)
    static_x.copy_(new_x)
    static_dy.copy_(new_dy)
    graph.replay()
    for a, b in zip(out, step(new_x, new_dy)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize(("tokens", "channels", "hidden"), [(300, 100, 270), (700, 240, 2000), (40, 16, 130)])
def test_float32_products_stay_at_float32_error(tokens, channels, hidden):
    # A pass of 128 values of K ends with eight products on the full-size sum, each cut by at most a unit in
    # the last place, 2^-23, half of it on average: 8 units of 2^-24; 4 more for the small products, the
    # operands' rounding and the sums of passes.
    *args, dy = inputs(tokens, channels, hidden, channels, torch.float32)
    leaves = [a.clone().requires_grad_(True) for a in args]
    y = gated_mlp(*leaves, activation="silu")
    wide = [a.double().requires_grad_(True) for a in args]
    want = formula(*wide, "silu")
    grads = torch.autograd.grad(y, leaves, dy)
    for got, exact in zip((y, *grads), (want, *torch.autograd.grad(want, wide, dy.double()))):
        assert float((got.detach().double() - exact.detach()).norm()) <= 12 * 2.0 ** -24 * float(exact.detach().norm())


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint8", [False, True])
def test_gradients_of_gradients_under_a_constant_upstream_gradient_are_refused(checkpoint8):
    *args, _ = inputs(20, 16, 24, 16, torch.float32)
    leaves = [a.requires_grad_(True) for a in args]

    def layer(x):
        return gated_mlp(x, *leaves[1:], checkpoint8=checkpoint8)

    y = layer(leaves[0])
    plain = torch.autograd.grad(y.sum(), leaves, retain_graph=True)
    grads = torch.autograd.grad(y.sum(), leaves, create_graph=True)
    for g, p in zip(grads, plain):  # the values are there, without a way back through them
        assert torch.equal(g, p)
        for wrt in leaves:
            with pytest.raises(RuntimeError, match="not differentiable itself"):
                torch.autograd.grad(y.mean() + g.pow(2).sum(), wrt, retain_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable itself"):
        (y.mean() + grads[0].pow(2).sum()).backward()
    # Through two layers, and with an upstream gradient that depends on another tensor.
    scale = torch.ones((), device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad((layer(layer(leaves[0])) * scale).sum(), leaves[0], create_graph=True)
    for wrt in (leaves[0], leaves[3], scale):
        with pytest.raises(RuntimeError, match="not differentiable itself"):
            torch.autograd.grad(g.sum(), wrt, retain_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_tangents_are_refused(which, grad_mode):
    *args, _ = inputs(20, 16, 24, 16, torch.float32)
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        args[which] = torch.autograd.forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            gated_mlp(*args)


# bf16: tokens, channels, hidden, outputs; a shape whose forward pass stays on chip, ones whose backward pass does not.
@pytest.mark.parametrize(("tokens", "channels", "hidden", "outputs"), [(262144, 64, 128, 64), (262144, 128, 256, 128), (8192, 512, 2048, 512),
                                                                       (8192, 1024, 4096, 1024), (8192, 4096, 11008, 4096),
                                                                       (32768, 4096, 14336, 4096), (100, 24, 40, 8)])
def test_workspaces_hold_what_a_call_uses(tokens, channels, hidden, outputs):
    small = 4096 + 512 * hidden  # roundings to 256 bytes, and a few rows
    operands = 2 * (tokens * channels + 2 * hidden * channels + hidden * outputs)
    hidden_values = 2 * tokens * (hidden + 15) // 16 * 16
    gradients = 4 * hidden * (2 * channels + outputs)
    on_chip = channels <= 64 and outputs <= 64 and hidden <= 128
    # Parts of the weight gradients: one per CTA on chip, else what fills a few whole waves of 148 SMs.
    tiles = 2 * -(-hidden // 256) * -(-channels // 256) + -(-outputs // 256) * -(-hidden // 256)
    parts = min(148, -(-tokens // 128)) if on_chip else 1 + 4 * 148 // tiles
    forward = 8 * native.workspace("spectral_gated_mlp_workspace", 1, tokens, channels, hidden, outputs)
    assert forward <= operands + (0 if channels <= 64 and hidden <= 256 else hidden_values) + small
    backward = 8 * native.workspace("spectral_gated_mlp_backward_workspace", 1, tokens, channels, hidden, outputs)
    most = 2 * tokens * outputs + operands + (0 if on_chip else 3 * hidden_values) + parts * gradients + small
    assert backward <= most
    # For arrays that are read in place: no copies of them, x restored only from a checkpoint.
    shape = (1, tokens, channels, hidden, outputs)
    at = 4096
    assert 8 * native.workspace("spectral_gated_mlp_workspace_for", at, at, at, at, *shape) <= forward - operands + small
    for packed in (0, 1):
        exact = 8 * native.workspace("spectral_gated_mlp_backward_workspace_for", at, None if packed else at, packed, at, at, at, *shape)
        assert exact <= backward - operands - 2 * tokens * outputs + packed * 2 * tokens * channels + small


def test_a_checkpoint_saves_memory_in_the_backward_pass():
    # What a backward pass from 8 bits needs beside its operands is no more than one restored x.
    for shape in [(1, 262144, 64, 128, 64), (1, 8192, 512, 2048, 512), (0, 8192, 512, 2048, 512), (2, 999, 37, 50, 37)]:
        plain, packed = (native.workspace("spectral_gated_mlp_backward_workspace_for", 4096, None if p else 4096, p, 4096, 4096, 4096, *shape)
                         for p in (0, 1))
        size = (4 if shape[0] == 0 else 2) * shape[1] * shape[2]
        assert 8 * (packed - plain) <= size + 4096


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint8", [False, True])
def test_a_training_step_allocates_what_it_needs(checkpoint8):
    tokens, channels, hidden = 8192, 512, 2048
    *args, dy = inputs(tokens, channels, hidden, channels, torch.bfloat16)
    leaves = [a.requires_grad_(True) for a in args]
    y = gated_mlp(*leaves, checkpoint8=checkpoint8)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(y, leaves, dy)
    peak = torch.cuda.max_memory_allocated() - before
    # The results, three hidden arrays, a restored x, and FP32 parts of the weight gradients (48 tiles: seven at most).
    assert peak <= sum(g.numel() * 2 for g in grads) + 3 * 2 * tokens * hidden + 2 * tokens * channels + 7 * 4 * 3 * hidden * channels + (1 << 22)


# Sums over many tokens, of terms of one sign: the wide kernels with 128 and with 256 columns a tile, and the narrow one.
@pytest.mark.gpu
@pytest.mark.parametrize(("tokens", "channels", "hidden", "outputs"), [(262144 + 77, 200, 401, 201), (262144, 320, 512, 320),
                                                                       ((1 << 24) + 77, 64, 128, 64)])
def test_weight_gradients_of_many_tokens_are_not_pulled_towards_zero(tokens, channels, hidden, outputs):
    dtype = torch.float16
    g = torch.Generator(device="cuda").manual_seed(1)

    def positive(rows, cols, scale):
        return torch.rand(rows, cols, generator=g, device="cuda").add_(0.5).mul_(scale).to(dtype)

    args = [positive(tokens, channels, 1.0), positive(hidden, channels, 1 / channels), positive(hidden, channels, 1 / channels),
            positive(outputs, hidden, 1 / hidden)]
    dy = positive(tokens, outputs, 64 / tokens)
    leaves = [a.requires_grad_(True) for a in args]
    got = torch.autograd.grad(gated_mlp(*leaves, activation="none"), leaves, dy)
    with torch.no_grad():
        wg, wu, wd = (a.double() for a in args[1:])
        want = [torch.zeros_like(w) for w in (wg, wu, wd)]
        for i in range(0, tokens, 1 << 17):
            x, d = args[0][i:i + (1 << 17)].double(), dy[i:i + (1 << 17)].double()
            gate, up, dh = x @ wg.T, x @ wu.T, d @ wd
            want[0] += (dh * up).T @ x
            want[1] += (dh * gate).T @ x
            want[2] += d.T @ (gate * up)
    # An MMA of 16 tokens cuts its sum by less than 2^-23 of what it ends up as, and 512 follow one another at most;
    # roundings to the type (of the hidden values, their gradients and the results) are to nearest and leave a mean of
    # 2^-17 at most over these many values.
    for name, a, b in zip(("dw_gate", "dw_up", "dw_down"), got[1:], want):
        mean = float(((a.double() - b) / b).mean())
        assert abs(mean) <= 512 * 2.0 ** -23 + 2.0 ** -17, f"{name}: {mean:.3g}"
    # dx, wherever the call was cut: the rows' own values.
    for i in (0, tokens // 14 // 128 * 128, tokens // 2, tokens - 301):
        rows = [args[0][i:i + 300].detach().requires_grad_(True), *leaves[1:]]
        (alone,) = torch.autograd.grad(gated_mlp(*rows, activation="none"), rows[:1], dy[i:i + 300])
        assert torch.equal(got[0][i:i + 300], alone)


def test_the_c_abi_refuses_unaligned_scales():
    a = dict(dy=1 << 20, x=None, codes=1 << 21, scales=(1 << 18) + 2, w_gate=1 << 22, w_up=1 << 23, w_down=1 << 24, dx=1 << 25,
             dw_gate=1 << 26, dw_up=1 << 27, dw_down=1 << 29, dtype=1, tokens=4, channels=8, hidden=16, outputs=8, activation=1,
             work=1 << 30, stream=None)
    with pytest.raises(ValueError, match="aligned"):
        native.call("spectral_gated_mlp_backward", *a.values())


# Enough tokens for the wide tiles: 256 columns down and to the input, 128 at the gate both ways, weight tiles of 256 x 256 in
# the 16-bit types; then 128 columns down and to the input, with weight tiles of 128 x 128.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize(("tokens", "channels", "hidden", "outputs"), [(8200, 520, 2050, 530), (12300, 120, 300, 120), (12289, 121, 299, 130)])
def test_wide_tiles(tokens, channels, hidden, outputs, activation, dtype):
    test_values_and_gradients(tokens, channels, hidden, outputs, activation, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_tiles_from_an_8_bit_checkpoint(dtype):
    test_gradients_from_an_8_bit_checkpoint(8200, 520, 2050, 530, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize(("dtype", "tol"), [(torch.float32, 2e-5), (torch.bfloat16, 2e-2), (torch.float16, 4e-3)])
def test_fno_block_at_its_own_size(dtype, tol):
    torch.manual_seed(3)
    block = FNOBlock(64, 128, 16, 16, groups=8, device="cuda", dtype=dtype)
    u, up = torch.randn(4, 64, 128, 128, device="cuda"), torch.randn(4, 64, 128, 128, device="cuda")
    params = [block.norm.weight, block.norm.bias, block.mlp.w_gate, block.mlp.w_up, block.mlp.w_down]
    leaf = u.clone().requires_grad_(True)
    y = block(leaf)
    got = torch.autograd.grad(y, [leaf, *params], up)
    ref = u.double().requires_grad_(True)
    want_y = block64(block, ref)
    for g, w in zip((y, *got), (want_y, *torch.autograd.grad(want_y, [ref, *params], up.double()))):
        close(g, w, tol)
    # With its inputs kept in 8 bits: values within the same bound (the norm then reads a copy with the channels last), and
    # gradients off by what the checkpoints are. Half a step is 1/254 of the largest of 64 values (some 2.7 standard
    # deviations), 0.6 % of the values in the mean square; two checkpoints, each through an operand and a slope or a product:
    # 2.4 % to first order, twice that here.
    block.norm.checkpoint8 = block.mlp.checkpoint8 = True
    packed = block(leaf)
    close(packed, want_y, tol)
    for g, w in zip(torch.autograd.grad(packed, [leaf, *params], up), got):
        close(g, w.double(), 0.05)


@pytest.mark.gpu
def test_mixed_types_are_refused_by_the_layers():
    # The norm's parameters are float32 whatever the fields are; the feed-forward weights have the fields' type. Autocast casts neither.
    x = torch.zeros(2, 3, 16, device="cuda")
    with pytest.raises(RuntimeError, match="weight must be a float32"):
        spectral.nn.GroupNormAct(4, 16, device="cuda").bfloat16()(x.bfloat16())
    mlp = GatedMLP(16, 32, device="cuda")
    with pytest.raises(RuntimeError, match="w_gate must be"):
        mlp(x.bfloat16())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert mlp(x).dtype == torch.float32
        with pytest.raises(RuntimeError, match="w_gate must be"):
            mlp(x.bfloat16())
