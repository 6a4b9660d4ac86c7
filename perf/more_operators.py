"""Cases, plain forms and 64-bit results for the operators that condition a field on an encoder's states.

Next to its spectral convolution an operator network reads from states of another length: sensors, observations,
an encoder's tokens. Its grid points (or latent points, or single query points while serving) make queries, the
states make keys and values; queries and keys are normalised for each head and rotated by their positions first.
This file lists real calls of those two operators, draws more of the same ranges, and computes each in a plain form
made of elementary torch operations in 32 bits (angles in 64).

    op "rotary"     q, k (batch, tokens, heads, dim): x / sqrt(mean(x^2) + eps) * weight over each head, its first
                    `rotated` values turned by angles position * theta^(-i / n), in one pass over both
    op "attention"  out = softmax(scale q k^T) v, q (batch, queries, heads, dim), k and v (batch, keys, kv_heads, dim);
                    heads / kv_heads query heads share a head of k and v; keys cut off by a length per sample or by
                    a mask; a sample without keys gives zeros

    mode "infer"    the forward pass
    mode "train"    the forward pass and every gradient for upstream gradients
"""

import math
import sys

import torch

own = False  # True: run() calls this repository's operators instead of the plain forms

EPS = 1e-6
THETA = 10000.0
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZES = {"float32": 4, "bfloat16": 2, "float16": 2}


def listed():
    return [
        # One query point while serving, its keys kept from before: launch latency.
        dict(name="rotary_point", op="rotary", mode="infer", dtype="bfloat16", batch=1, queries=1, keys=0, heads=8,
             kv_heads=0, dim=64, rotated=64, axes=2, pairs="halves", positions="coordinates"),
        # Every grid point of the benchmark's FNO layer (64 samples, 128 x 128, 64 channels as two heads) and 256
        # states for each sample.
        dict(name="rotary_grid", op="rotary", mode="infer", dtype="bfloat16", batch=64, queries=16384, keys=256, heads=2,
             kv_heads=2, dim=32, rotated=32, axes=2, pairs="halves", positions="coordinates"),
        # The same layer in a training step.
        dict(name="rotary_grid_train", op="rotary", mode="train", dtype="bfloat16", batch=64, queries=16384, keys=256,
             heads=2, kv_heads=2, dim=32, rotated=32, axes=2, pairs="halves", positions="coordinates"),
        # A long series of samples in time: whole-number positions far out, odd sizes, half of each head rotated.
        dict(name="rotary_far_train", op="rotary", mode="train", dtype="float32", batch=3, queries=4099, keys=1001,
             heads=6, kv_heads=3, dim=40, rotated=20, axes=1, pairs="neighbours", positions="far"),
        # One query point of one sample: the states are all there is to read.
        dict(name="attention_point", op="attention", mode="infer", dtype="bfloat16", batch=1, queries=1, keys=4096,
             heads=8, kv_heads=2, dim=64, cut="none"),
        # Sixteen samples served together, one query point each, states of different lengths.
        dict(name="attention_points_ragged", op="attention", mode="infer", dtype="bfloat16", batch=16, queries=1,
             keys=16384, heads=16, kv_heads=4, dim=64, cut="lengths"),
        # Every grid point of the benchmark's FNO layer reads 256 states.
        dict(name="attention_grid", op="attention", mode="infer", dtype="bfloat16", batch=64, queries=16384, keys=256,
             heads=2, kv_heads=2, dim=32, cut="none"),
        # The same layer in a training step.
        dict(name="attention_grid_train", op="attention", mode="train", dtype="bfloat16", batch=64, queries=16384,
             keys=256, heads=2, kv_heads=2, dim=32, cut="none"),
        # 512 latent points gather a 128 x 128 field of which some points are missing, in a float16 training step.
        dict(name="attention_latents_train", op="attention", mode="train", dtype="float16", batch=8, queries=512,
             keys=16384, heads=8, kv_heads=8, dim=64, cut="mask"),
        # Wide heads, shared keys and values, long on both sides: matrix products bound it.
        dict(name="attention_wide", op="attention", mode="infer", dtype="bfloat16", batch=4, queries=4096, keys=4096,
             heads=16, kv_heads=4, dim=128, cut="none"),
        dict(name="attention_wide_train", op="attention", mode="train", dtype="bfloat16", batch=4, queries=4096,
             keys=4096, heads=16, kv_heads=4, dim=128, cut="none"),
        # Float32 with no size a multiple of a tile, a sample without keys.
        dict(name="attention_odd_train", op="attention", mode="train", dtype="float32", batch=3, queries=1000, keys=333,
             heads=6, kv_heads=3, dim=40, cut="mask"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "attention", "attention"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    mode = rng.choice(["infer", "train"])
    dim = _log(rng, 8, 128)
    if rng.random() < 0.6:
        dim = max(16, dim // 16 * 16)
    kv_heads, group = _log(rng, 1, 16), rng.choice([1, 1, 2, 3, 4, 8])
    heads = kv_heads * group
    queries = rng.choice([1, _log(rng, 1, 16384), _log(rng, 1, 16384)])
    keys = _log(rng, 1, 16384)
    if op == "rotary":
        axes = rng.choice([1, 2, 3])
        rotated = dim // (2 * axes) * (2 * axes)
        if rng.random() < 0.3:
            rotated = rotated // (4 * axes) * (2 * axes)
        limit = max(1, (1 << 26) // ((queries * heads + keys * kv_heads) * dim))
        while (queries * heads + keys * kv_heads) * dim > (1 << 26):
            queries, keys = max(1, queries // 2), max(1, keys // 2)
        return dict(op=op, mode=mode, dtype=dtype, batch=_log(rng, 1, min(64, limit)), queries=queries, keys=keys,
                    heads=heads, kv_heads=kv_heads, dim=dim, rotated=rotated, axes=axes if rotated else 1,
                    pairs=rng.choice(["halves", "neighbours"]), positions=rng.choice(["coordinates", "far"]))
    # No more products than the wide training step, no more scores than it holds at once in the plain form.
    most = min(4 * 16 * 4096 * 4096, 4 * 16 * 4096 * 4096 * 128 // dim)
    while queries * keys * heads > most:
        queries, keys = max(1, queries // 2), max(1, keys // 2)
    limit = max(1, min(most // (queries * keys * heads), (1 << 26) // ((queries * heads + keys * kv_heads) * dim)))
    return dict(op=op, mode=mode, dtype=dtype, batch=_log(rng, 1, min(64, limit)), queries=queries, keys=keys, heads=heads,
                kv_heads=kv_heads, dim=dim, cut=rng.choice(["none", "lengths", "mask"]))


def _lengths(case):
    """The samples' numbers of keys, before the seed shuffles them: from half of the states to all, and in a batch of
    three or more one sample without any."""
    batch, keys = case["batch"], case["keys"]
    lengths = [keys - i * keys // (2 * batch) for i in range(batch)]
    if batch >= 3:
        lengths[-1] = 0
    return lengths


def _valid(case):
    """How many keys each sample has, in some order."""
    batch, keys = case["batch"], case["keys"]
    if case["cut"] == "lengths":
        return _lengths(case)
    if case["cut"] == "mask":
        return [0 if batch >= 3 and i == 0 else keys - keys // 4 for i in range(batch)]
    return [keys] * batch


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def prepare(case, seed):
    device, dtype = _device(), DTYPES[case["dtype"]]
    g = torch.Generator(device=device).manual_seed(1000003 * seed + 29)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    b, tq, tk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    train = case["mode"] == "train"
    state = {"case": dict(case)}
    if case["op"] == "rotary":
        # Projections, each channel with a size of its own, views into one array with values the pass does not read
        # (queries next to gates, keys next to values), as one product leaves them.
        def half(tokens, count):
            return (normal(b, tokens, 2, count, d) * torch.exp(0.3 * normal(count, d))).to(dtype)[:, :, 0]

        def positions(tokens):
            if case["positions"] == "far":
                start = torch.randint(0, 1 << 20, (b, 1, 1), generator=g, device=device)
                return (start + torch.arange(tokens, device=device)[None, :, None]).expand(b, tokens, case["axes"])
            return 128.0 * torch.rand(b, tokens, case["axes"], generator=g, device=device)

        for name, tokens, count in (("q", tq, h), ("k", tk, hk)):
            state[name] = half(tokens, count) if tokens else None
            state[name + "_weight"] = 1.0 + 0.2 * normal(d) if tokens else None
            state[name + "_positions"] = positions(tokens) if tokens else None
            if train and tokens:
                state["d" + name] = normal(b, tokens, count, d).to(dtype)
        leaves = ("q", "k", "q_weight", "k_weight")
    else:
        # Queries and keys of unit size after their norm, some heads sharper than others.
        state["q"] = (normal(b, tq, h, d) * torch.exp(0.3 * normal(h, 1))).to(dtype)
        state["k"] = normal(b, tk, hk, d).to(dtype)
        state["v"] = (normal(b, tk, hk, d) + 0.3 * normal(hk, d)).to(dtype)
        state["lengths"] = state["mask"] = None
        order = torch.randperm(b, generator=g, device=device)
        if case["cut"] == "lengths":
            state["lengths"] = torch.tensor(_lengths(case), device=device, dtype=torch.int32)[order]
        elif case["cut"] == "mask":
            rank = torch.rand(b, tk, generator=g, device=device).argsort(-1).argsort(-1)
            state["mask"] = rank < torch.tensor(_valid(case), device=device)[order][:, None]
        if train:
            state["dout"] = normal(b, tq, h, d).to(dtype)
        leaves = ("q", "k", "v")
    if train:
        for name in leaves:
            if state[name] is not None:
                state[name].requires_grad_(True)
    return state


# --- the framework's operators, as a user calls them ---------------------------------------------


def _run_own(state):
    if "gpu-spectral-stack_b200" not in sys.path:
        sys.path.insert(0, "gpu-spectral-stack_b200")
    import spectral

    case = state["case"]
    if case["op"] == "rotary":
        q, k = spectral.nn.qk_norm_rotary(
            state["q"], state["k"], state["q_weight"], state["k_weight"], state["q_positions"], state["k_positions"],
            eps=EPS, theta=THETA, rotated=case["rotated"], pairs=case["pairs"])
        if case["mode"] == "infer":
            return q if k is None else (q, k)
        outputs, upstream = [q, k], [state["dq"], state["dk"]]
        inputs = [state[name] for name in ("q", "k", "q_weight", "k_weight")]
    else:
        out = spectral.nn.cross_attention(state["q"], state["k"], state["v"], lengths=state["lengths"], mask=state["mask"])
        if case["mode"] == "infer":
            return out
        outputs, upstream = [out], [state["dout"]]
        inputs = [state[name] for name in ("q", "k", "v")]
    return (*(o.detach() for o in outputs), *torch.autograd.grad(outputs, inputs, upstream))


# --- the plain forms -------------------------------------------------------------------------------


def _pair_indices(case, device):
    """The values that the rotation pairs up: indices of the first and second of each pair, the axis and the number of
    the pair within it."""
    axes, rotated = case["axes"], case["rotated"]
    per = rotated // axes
    n = per // 2
    axis = torch.arange(axes, device=device).repeat_interleave(n)
    i = torch.arange(n, device=device).repeat(axes)
    if case["pairs"] == "halves":
        return axis * per + i, axis * per + i + n, axis, i
    return axis * per + 2 * i, axis * per + 2 * i + 1, axis, i


def _angles(case, positions):
    """cos and sin (batch, tokens, 1, pairs), float32 from angles in 64 bits."""
    _, _, axis, i = _pair_indices(case, positions.device)
    n = max(1, case["rotated"] // case["axes"] // 2)
    frequency = THETA ** (-i.double() / n)
    angle = positions.double()[..., axis] * frequency
    return torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]


def _turn(case, x, cos, sin):
    first, second, _, _ = _pair_indices(case, x.device)
    a, b = x[..., first], x[..., second]
    y = x.clone()
    y[..., first] = a * cos - b * sin
    y[..., second] = a * sin + b * cos
    return y


def _plain_rotary(state):
    case = state["case"]
    results, gradients, weights = [], [], []
    for name in ("q", "k"):
        if state[name] is None:
            continue
        x, w = state[name].float(), state[name + "_weight"]
        cos, sin = _angles(case, state[name + "_positions"])
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        results.append(_turn(case, x * r * w, cos, sin).to(state[name].dtype))
        if case["mode"] == "train":
            g = _turn(case, state["d" + name].float(), cos, -sin)
            weights.append((g * x * r).sum((0, 1, 2)))
            g = g * w
            gradients.append((r * (g - x * r * r * (g * x).mean(-1, keepdim=True))).to(state[name].dtype))
    if case["mode"] == "train":
        return (*results, *gradients, *weights)
    return results[0] if len(results) == 1 else tuple(results)


def _plain_attention(state):
    case = state["case"]
    b, tq, tk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    group, dtype, scale = h // hk, state["q"].dtype, 1.0 / math.sqrt(d)

    def rows(t):  # (batch, kv_heads, group * queries, dim)
        return t.float().reshape(b, tq, hk, group, d).permute(0, 2, 3, 1, 4).reshape(b, hk, group * tq, d)

    def back(t):
        return t.reshape(b, hk, group, tq, d).permute(0, 3, 1, 2, 4).reshape(b, tq, h, d).to(dtype)

    q, k, v = rows(state["q"]), state["k"].float().transpose(1, 2), state["v"].float().transpose(1, 2)
    s = q @ k.transpose(-1, -2)
    s *= scale
    cut = None
    if state["lengths"] is not None:
        cut = torch.arange(tk, device=q.device)[None] >= state["lengths"][:, None]
    elif state["mask"] is not None:
        cut = ~state["mask"]
    if cut is not None:
        s.masked_fill_(cut[:, None, None], -math.inf)
    largest = s.amax(-1, keepdim=True)
    largest = torch.where(largest == -math.inf, torch.zeros_like(largest), largest)
    s -= largest
    p = s.exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0.0, torch.ones_like(total), total)
    o = p @ v
    if case["mode"] == "infer":
        return back(o)
    do = rows(state["dout"])
    dv = p.transpose(-1, -2) @ do
    ds = do @ v.transpose(-1, -2)
    ds -= (do * o).sum(-1, keepdim=True)
    ds *= p
    ds *= scale
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    return back(o), back(dq), dk.transpose(1, 2).to(dtype), dv.transpose(1, 2).to(dtype)


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_rotary(state) if state["case"]["op"] == "rotary" else _plain_attention(state)


# --- what a pass cannot do without -----------------------------------------------------------------


def work(case):
    size = SIZES[case["dtype"]]
    train = case["mode"] == "train"
    b, tq, tk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    if case["op"] == "rotary":
        values = b * (tq * h + tk * hk) * d
        position = 8 if case["positions"] == "far" else 4
        # Each value read and written, and its gradient again; a position for each token and axis.
        return {"bytes": (4 if train else 2) * values * size + b * (tq + tk) * case["axes"] * position + 8 * d,
                "flops": (25 if train else 10) * values}
    valid = sum(_valid(case))
    # Queries in, results out, the keys and values that count; and the same of their gradients (those of all keys).
    values = 2 * b * tq * h * d + 2 * valid * hk * d
    if train:
        values += 2 * b * tq * h * d + 2 * b * tk * hk * d
    # Two products forward; five backward, the scores again among them.
    return {"bytes": values * size + (b * tk if case["cut"] == "mask" else 0), "flops": 2 * (7 if train else 2) * valid * tq * h * d}


# --- the definition in 64 bits ---------------------------------------------------------------------


def _exact_rotary(case, state):
    """Pairs as complex numbers, each multiplied by exp(i angle)."""
    axes, rotated = case["axes"], case["rotated"]
    n = rotated // axes // 2
    outputs, inputs, upstream, weights = [], [], [], []
    for name in ("q", "k"):
        if state[name] is None:
            continue
        x = state[name].detach().double().requires_grad_(True)
        w = state[name + "_weight"].detach().double().requires_grad_(True)
        y = x / torch.sqrt(torch.sum(x ** 2, -1, keepdim=True) / case["dim"] + EPS) * w
        pieces = []
        for a in range(axes if rotated else 0):
            part = y[..., a * 2 * n:(a + 1) * 2 * n]
            part = part.unflatten(-1, (2, n)).transpose(-1, -2) if case["pairs"] == "halves" else part.unflatten(-1, (n, 2))
            powers = torch.logspace(0, -(n - 1) / n, n, base=THETA, dtype=torch.float64, device=x.device)
            angle = state[name + "_positions"][..., a, None].double() * powers
            turned = torch.view_as_complex(part.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, :, None]
            turned = torch.view_as_real(turned)
            pieces.append((turned.transpose(-1, -2) if case["pairs"] == "halves" else turned).flatten(-2))
        outputs.append(torch.cat([*pieces, y[..., rotated:]], -1))
        inputs.append(x)
        weights.append(w)
        upstream.append(state["d" + name].double() if case["mode"] == "train" else None)
    values = [o.detach() for o in outputs]
    if case["mode"] == "train":
        return (*values, *torch.autograd.grad(outputs, [*inputs, *weights], upstream))
    return values[0] if len(values) == 1 else tuple(values)


def _exact_attention(case, state):
    """Sample by sample and head by head, over the keys that count only."""
    train = case["mode"] == "train"
    group = case["heads"] // case["kv_heads"]
    q, k, v = (state[n].detach().double() for n in ("q", "k", "v"))
    out = torch.zeros_like(q)
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v)) if train else (None, None, None)
    keep = torch.ones(case["batch"], case["keys"], dtype=torch.bool, device=q.device)
    if state["lengths"] is not None:
        for i, length in enumerate(state["lengths"].tolist()):
            keep[i, length:] = False
    if state["mask"] is not None:
        keep = state["mask"]
    for i in range(case["batch"]):
        index = torch.nonzero(keep[i]).flatten()
        if index.numel() == 0:
            continue
        for head in range(case["kv_heads"]):
            span = slice(head * group, (head + 1) * group)
            args = [q[i, :, span], k[i, index, head], v[i, index, head]]
            if train:
                args = [a.clone().requires_grad_(True) for a in args]
            scores = torch.einsum("tgd,sd->tgs", args[0], args[1]) / math.sqrt(case["dim"])
            result = torch.einsum("tgs,sd->tgd", torch.softmax(scores, -1), args[2])
            out[i, :, span] = result.detach()
            if train:
                grads = torch.autograd.grad(result, args, state["dout"][i, :, span].double())
                dq[i, :, span] = grads[0]
                dk[i, index, head] = grads[1]
                dv[i, index, head] = grads[2]
    return (out, dq, dk, dv) if train else out


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_rotary(case, state) if case["op"] == "rotary" else _exact_attention(case, state)
