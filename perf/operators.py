"""Cases, plain forms and 64-bit results for the pointwise half of an FNO block.

Around its spectral convolution an FNO block normalises its fields (group norm with an
activation, channels last), mixes their channels pointwise (a gated feed-forward block), and
keeps what the backward pass needs (activation checkpoints, in 8 bits if asked). This file lists
real calls of those three operators, draws more of the same ranges, and computes each in a plain
form made of elementary torch operations in 32 bits.

    op "norm"  y = act(group_norm(x) * weight + bias), x (batch, n1, n2, channels)
    op "pack"  8-bit round trip: codes and scales of x (rows, width), and the values they stand for
    op "mlp"   y = (act(x w_gate^T) * (x w_up^T)) w_down^T, x (tokens, channels)

    mode "infer"   the forward pass
    mode "train"   the forward pass and every gradient for an upstream gradient dy
    mode "train8"  the same, the input kept for the backward pass as an 8-bit checkpoint
"""

import math
import sys

import torch

own = False  # True: run() calls this repository's operators instead of the plain forms

BLOCK = 64       # values along the last dimension that share one scale of an 8-bit checkpoint
TINY = 2.0 ** -100  # smallest magnitude a block's scale is made from
EPS = 1e-5
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZES = {"float32": 4, "bfloat16": 2, "float16": 2}


def listed():
    return [
        # One small latent field while serving: launch latency.
        dict(name="norm_small", op="norm", mode="infer", dtype="bfloat16", batch=1, n1=16, n2=16, channels=32,
             groups=8, act="silu", layout="last"),
        # The benchmark's FNO layer (64 samples, 64 channels, 128 x 128), as the spectral
        # convolution hands it over: float32, channels first in memory.
        dict(name="norm_layer", op="norm", mode="infer", dtype="float32", batch=64, n1=128, n2=128, channels=64,
             groups=8, act="gelu", layout="first"),
        # The same layer in a bfloat16 training step.
        dict(name="norm_layer_train", op="norm", mode="train", dtype="bfloat16", batch=64, n1=128, n2=128,
             channels=64, groups=8, act="gelu", layout="last"),
        # An irregular grid: odd extents, ten channels a group.
        dict(name="norm_odd_train", op="norm", mode="train", dtype="float32", batch=3, n1=97, n2=61, channels=60,
             groups=6, act="silu", layout="last"),
        # The layer's training step with its input kept in 8 bits.
        dict(name="norm_layer_train8", op="norm", mode="train8", dtype="bfloat16", batch=64, n1=128, n2=128,
             channels=64, groups=8, act="gelu", layout="last"),
        # Keeping and restoring the layer's activations.
        dict(name="pack_layer", op="pack", mode="infer", dtype="bfloat16", rows=1048576, width=64),
        # Rows that end inside a block of 64.
        dict(name="pack_odd", op="pack", mode="infer", dtype="float32", rows=1000, width=130),
        # One token through a wide block while serving: the weights are all there is to read.
        dict(name="mlp_token", op="mlp", mode="infer", dtype="bfloat16", tokens=1, channels=512, hidden=2048,
             act="silu"),
        # Every grid point of 16 samples of the FNO layer through its channel mixer.
        dict(name="mlp_layer", op="mlp", mode="infer", dtype="bfloat16", tokens=262144, channels=64, hidden=128,
             act="gelu"),
        # A training step of that mixer, its input kept in 8 bits.
        dict(name="mlp_layer_train8", op="mlp", mode="train8", dtype="bfloat16", tokens=262144, channels=64,
             hidden=128, act="gelu"),
        # A training step of a wide block over latent tokens: matrix products bound it.
        dict(name="mlp_wide_train", op="mlp", mode="train", dtype="bfloat16", tokens=8192, channels=512,
             hidden=2048, act="silu"),
        # Float32 with no size a multiple of a tile.
        dict(name="mlp_odd", op="mlp", mode="infer", dtype="float32", tokens=1000, channels=100, hidden=270,
             act="silu"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "pack", "mlp", "mlp"])
    dtype = rng.choice(["bfloat16", "float32", "float16"])
    if op == "pack":
        width = _log(rng, 1, 4096)
        rows = _log(rng, 1, max(1, (1 << 25) // max(width, 64)))
        return dict(op="pack", mode="infer", dtype=dtype, rows=rows, width=width)
    mode = rng.choice(["infer", "train", "train8"])
    act = rng.choice(["silu", "gelu", "none"])
    if op == "norm":
        channels = _log(rng, 1, 512)
        if rng.random() < 0.5:
            channels = max(8, channels // 8 * 8)
        groups = rng.choice([g for g in range(1, channels + 1) if channels % g == 0])
        n1, n2 = _log(rng, 1, 512), _log(rng, 1, 512)
        limit = max(1, (1 << (26 if mode == "infer" else 25)) // (n1 * n2 * channels))
        while n1 * n2 * channels > (1 << 25):
            n1 = max(1, n1 // 2)
        return dict(op="norm", mode=mode, dtype=dtype, batch=_log(rng, 1, min(64, limit)), n1=n1, n2=n2,
                    channels=channels, groups=groups, act=act, layout=rng.choice(["last", "last", "first"]))
    channels, hidden = _log(rng, 8, 1024), _log(rng, 8, 4096)
    if rng.random() < 0.5:
        channels, hidden = max(16, channels // 16 * 16), max(16, hidden // 16 * 16)
    passes = 1 if mode == "infer" else 3
    # No more products than the wide training step, and no more rows x (channels + hidden) than
    # the layer cases.
    limit = min(262144, int(0.9 * 1.5e11 / (6 * passes * channels * hidden)), (1 << 26) // (channels + hidden))
    return dict(op="mlp", mode=mode, dtype=dtype, tokens=_log(rng, 1, max(1, limit)), channels=channels,
                hidden=hidden, act=act)


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def prepare(case, seed):
    device, dtype = _device(), DTYPES[case["dtype"]]
    g = torch.Generator(device=device).manual_seed(1000003 * seed + 17)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    state = {"case": dict(case)}
    if case["op"] == "pack":
        # Activations: rows of different size, a few large channels.
        x = normal(case["rows"], case["width"]) * torch.exp(0.5 * normal(case["rows"], 1))
        state["x"] = (x * torch.exp(0.5 * normal(case["width"]))).to(dtype)
        return state
    if case["op"] == "norm":
        b, n1, n2, c = case["batch"], case["n1"], case["n2"], case["channels"]
        # Fields with an offset and a size of their own per channel.
        size, offset = torch.exp(0.5 * normal(c)), normal(c)
        if case["layout"] == "first":
            x = normal(b, c, n1, n2).mul_(size[:, None, None]).add_(offset[:, None, None]).to(dtype)
            x = x.permute(0, 2, 3, 1)
        else:
            x = normal(b, n1, n2, c).mul_(size).add_(offset).to(dtype)
        state["x"] = x
        state["weight"] = 1.0 + 0.2 * normal(c)
        state["bias"] = 0.2 * normal(c)
        if case["mode"] != "infer":
            state["dy"] = normal(b, n1, n2, c).to(dtype)
    else:
        m, c, f = case["tokens"], case["channels"], case["hidden"]
        state["x"] = normal(m, c).to(dtype)
        state["w_gate"] = (normal(f, c) / math.sqrt(c)).to(dtype)
        state["w_up"] = (normal(f, c) / math.sqrt(c)).to(dtype)
        state["w_down"] = (normal(c, f) / math.sqrt(f)).to(dtype)
        if case["mode"] != "infer":
            state["dy"] = normal(m, c).to(dtype)
    if case["mode"] != "infer":
        for key in ("x", "weight", "bias", "w_gate", "w_up", "w_down"):
            if key in state:
                state[key].requires_grad_(True)
    return state


# --- the framework's operators, as a user calls them ---------------------------------------------


def _run_own(state):
    if "gpu-spectral-stack_b200" not in sys.path:
        sys.path.insert(0, "gpu-spectral-stack_b200")
    import spectral

    case = state["case"]
    if case["op"] == "pack":
        codes, scales = spectral.pack8(state["x"])
        return spectral.unpack8(codes, scales, dtype=state["x"].dtype)
    keep8 = case["mode"] == "train8"
    if case["op"] == "norm":
        inputs = (state["x"], state["weight"], state["bias"])
        y = spectral.nn.group_norm_act(inputs[0], case["groups"], inputs[1], inputs[2], eps=EPS,
                                       activation=case["act"], checkpoint8=keep8)
    else:
        inputs = (state["x"], state["w_gate"], state["w_up"], state["w_down"])
        y = spectral.nn.gated_mlp(*inputs, activation=case["act"], checkpoint8=keep8)
    if case["mode"] == "infer":
        return y
    return (y.detach(), *torch.autograd.grad(y, inputs, state["dy"]))


# --- the plain forms -------------------------------------------------------------------------------


def _act(z, act):
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, act):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    return torch.ones_like(z)


def _plain_pack(x):
    """The values an 8-bit checkpoint of x holds, in x's type: per block of 64 along the last
    dimension, code = round(x * (127 / m)) and value = code * (m / 127), m the block's largest
    magnitude."""
    width = x.shape[-1]
    blocks = -(-width // BLOCK)
    v = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - width)).reshape(*x.shape[:-1], blocks, BLOCK)
    m = v.abs().amax(-1, keepdim=True).clamp_min(TINY)
    most = torch.full_like(m, 127.0)  # a tensor: torch turns divisions with a number into products
    code = torch.round(v * (most / m))
    value = (code * (m / most)).reshape(*x.shape[:-1], blocks * BLOCK)[..., :width]
    return value.to(x.dtype)


def _plain_norm(state):
    case, x = state["case"], state["x"]
    b, n1, n2, c = x.shape
    groups, act, dtype = case["groups"], case["act"], x.dtype
    shape = (b, n1 * n2, groups, c // groups)
    v = x.float().reshape(shape)
    mean = v.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt(((v - mean) ** 2).mean((1, 3), keepdim=True) + EPS)
    w, bias = state["weight"].reshape(1, 1, groups, -1), state["bias"].reshape(1, 1, groups, -1)
    y = _act((v - mean) * rstd * w + bias, act).reshape(x.shape).to(dtype)
    if case["mode"] == "infer":
        return y
    if case["mode"] == "train8":
        v = _plain_pack(x.contiguous()).float().reshape(shape)
    xhat = (v - mean) * rstd
    del v
    dz = state["dy"].float().reshape(shape) * _act_slope(xhat * w + bias, act)
    dbias = dz.sum((0, 1)).reshape(c)
    dweight = (dz * xhat).sum((0, 1)).reshape(c)
    dz = dz * w
    dx = rstd * (dz - dz.mean((1, 3), keepdim=True) - xhat * (dz * xhat).mean((1, 3), keepdim=True))
    return y, dx.reshape(x.shape).to(dtype), dweight, dbias


def _plain_mlp(state):
    case, x = state["case"], state["x"]
    act, dtype = case["act"], x.dtype
    wg, wu, wd = (state[k].float() for k in ("w_gate", "w_up", "w_down"))
    v = x.float()
    g, u = v @ wg.T, v @ wu.T
    y = ((_act(g, act) * u) @ wd.T).to(dtype)
    if case["mode"] == "infer":
        return y
    if case["mode"] == "train8":
        v = _plain_pack(x).float()
        g, u = v @ wg.T, v @ wu.T
    dy = state["dy"].float()
    dh = dy @ wd
    a = _act(g, act)
    dwd = dy.T @ (a * u)
    du = dh * a
    dg = dh * u * _act_slope(g, act)
    dx = dg @ wg + du @ wu
    return y, dx.to(dtype), (dg.T @ v).to(dtype), (du.T @ v).to(dtype), dwd.to(dtype)


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        if state["case"]["op"] == "pack":
            return _plain_pack(state["x"])
        return _plain_norm(state) if state["case"]["op"] == "norm" else _plain_mlp(state)


# --- what a pass cannot do without -----------------------------------------------------------------


def work(case):
    size = SIZES[case["dtype"]]
    train = case["mode"] != "infer"
    if case["op"] == "pack":
        n = case["rows"] * case["width"]
        scales = case["rows"] * -(-case["width"] // BLOCK)
        # x read, the checkpoint written and read back, the values written.
        return {"bytes": 2 * n * size + 2 * n + 8 * scales, "flops": 4 * n}
    if case["op"] == "norm":
        n = case["batch"] * case["n1"] * case["n2"] * case["channels"]
        # x and y, and dy and dx; a few operations per value and direction.
        return {"bytes": (4 if train else 2) * n * size + 8 * (2 if train else 1) * case["channels"],
                "flops": (30 if train else 10) * n}
    m, c, f = case["tokens"], case["channels"], case["hidden"]
    # Three products forward; two more of the same size for each in the backward pass.
    return {"bytes": (2 if train else 1) * (2 * m * c + 3 * c * f) * size,
            "flops": 6 * m * c * f * (3 if train else 1)}


# --- the definition in 64 bits ---------------------------------------------------------------------


def _exact_act(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z


def _exact_pack(x):
    """The restored values, block by block. The codes are whole numbers, so the two operations
    that decide them are the definition's own, in 32 bits."""
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    for start in range(0, x.shape[-1], BLOCK):
        piece = x[..., start:start + BLOCK].to(torch.float32)
        largest = torch.maximum(piece.max(-1, keepdim=True).values, -piece.min(-1, keepdim=True).values)
        largest = torch.maximum(largest, torch.full_like(largest, TINY))
        per_unit = torch.full_like(largest, 127.0) / largest
        codes = torch.special.round(piece * per_unit)
        out[..., start:start + BLOCK] = (codes * (largest / torch.full_like(largest, 127.0))).to(x.dtype)
    return out


def _exact_norm(case, state):
    x = state["x"].detach()
    b, n1, n2, c = x.shape
    groups, per = case["groups"], c // case["groups"]
    weight = state["weight"].detach().double().requires_grad_(True)
    bias = state["bias"].detach().double().requires_grad_(True)

    def rows(t):  # (batch, groups, values of a group)
        return t.reshape(b, n1 * n2, groups, per).permute(0, 2, 1, 3).reshape(b, groups, -1)

    v = rows(x.double())
    var, mean = torch.var_mean(v, dim=-1, unbiased=False, keepdim=True)
    inv = 1.0 / torch.sqrt(var + EPS)

    def affine(h):  # (batch, n1 n2, c) from normalised rows
        h = h.reshape(b, groups, n1 * n2, per).permute(0, 2, 1, 3).reshape(b, n1 * n2, c)
        return _exact_act(h * weight + bias, case["act"])

    if case["mode"] == "infer":
        with torch.no_grad():
            return affine((v - mean) * inv).reshape(x.shape)
    with torch.no_grad():
        y = affine((v - mean) * inv).reshape(x.shape)
    if case["mode"] == "train8":
        v = rows(_exact_pack(x.contiguous()).double())
    h = ((v - mean) * inv).requires_grad_(True)
    dh, dweight, dbias = torch.autograd.grad(affine(h), (h, weight, bias),
                                             state["dy"].double().reshape(b, n1 * n2, c))
    # The Jacobian of the normalisation: what is constant over a group and what is parallel to h drop out.
    h = h.detach()
    dv = inv * (dh - dh.mean(-1, keepdim=True) - h * (dh * h).mean(-1, keepdim=True))
    dx = dv.reshape(b, groups, n1 * n2, per).permute(0, 2, 1, 3).reshape(x.shape)
    return y, dx, dweight, dbias


def _exact_mlp(case, state):
    def block(x, w_gate, w_up, w_down):
        gate = torch.einsum("mc,fc->mf", x, w_gate)
        up = torch.einsum("mc,fc->mf", x, w_up)
        return torch.einsum("mf,cf->mc", _exact_act(gate, case["act"]) * up, w_down)

    keys = ("x", "w_gate", "w_up", "w_down")
    args = [state[k].detach().double() for k in keys]
    with torch.no_grad():
        y = block(*args)
    if case["mode"] == "infer":
        return y
    if case["mode"] == "train8":
        args[0] = _exact_pack(state["x"].detach()).double()
    for a in args:
        a.requires_grad_(True)
    return (y, *torch.autograd.grad(block(*args), args, state["dy"].double()))


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "pack":
        return _exact_pack(state["x"])
    return _exact_norm(case, state) if case["op"] == "norm" else _exact_mlp(case, state)
