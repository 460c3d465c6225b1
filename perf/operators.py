"""The operators of a trainer's local step, as they are measured: layer norm, dropout, the gated
linear layer and the linear cross entropy, each with its gradient.

``run`` makes one pass of a training step through an operator (forward and backward).  With ``own``
false it is written in elementary torch operations in 32 bits; with ``own`` true it makes the calls of
``p2pdl_amd.training``.  ``exact`` gives the same values from the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IGNORE = -100


def _loss_scale(case):
    """Training in float16 scales the loss by a power of two, so that the gradient of a mean over many
    tokens stays among its normal numbers."""
    return 4.0 * 2.0 ** math.ceil(math.log2(case["rows"])) if case["dtype"] == "f16" else 1.0


def listed():
    return [
        # The hidden layer of the protocol's MLP at its batch of 32: launches and host time count.
        {"name": "norm mlp hidden", "op": "norm", "dtype": "f32", "rows": 32, "cols": 512},
        # A ragged batch (the last one of a shard) of a width that no vector load divides.
        {"name": "norm ragged", "op": "norm", "dtype": "f16", "rows": 4099, "cols": 1001},
        # A full device batch of a wide model.
        {"name": "norm wide", "op": "norm", "dtype": "bf16", "rows": 16384, "cols": 4096},
        # Dropout behind the MLP's hidden layer, batch of 32.
        {"name": "dropout mlp hidden", "op": "dropout", "dtype": "f32", "rows": 32, "cols": 512, "p": 0.5, "residual": False},
        # A ragged batch of an odd width.
        {"name": "dropout ragged", "op": "dropout", "dtype": "f16", "rows": 4099, "cols": 1001, "p": 0.2, "residual": False},
        # The end of a residual branch: dropout and the addition to the stream.
        {"name": "dropout residual wide", "op": "dropout", "dtype": "bf16", "rows": 16384, "cols": 4096, "p": 0.1, "residual": True},
        # A gated layer of the MLP's sizes (784 inputs, 512 units) at its batch of 32.
        {"name": "gated mlp", "op": "gated", "dtype": "f32", "rows": 32, "cols": 784, "units": 512, "act": "silu"},
        # Odd sizes everywhere: nothing is aligned.
        {"name": "gated ragged", "op": "gated", "dtype": "f16", "rows": 1023, "cols": 1001, "units": 2731, "act": "gelu"},
        # The feed-forward block of a wide model over a full device batch.
        {"name": "gated wide", "op": "gated", "dtype": "bf16", "rows": 8192, "cols": 4096, "units": 16384, "act": "silu"},
        # The protocol's MLP head: 256 features, 10 classes, a batch of 32.
        {"name": "loss mlp head", "op": "loss", "dtype": "f32", "rows": 32, "cols": 256, "units": 10},
        # A small language model's head, odd sizes.
        {"name": "loss ragged", "op": "loss", "dtype": "f16", "rows": 1023, "cols": 1001, "units": 32003},
        # A large vocabulary over a full device batch: the logits would be 2 GB in 16 bits.
        {"name": "loss large vocabulary", "op": "loss", "dtype": "bf16", "rows": 8192, "cols": 4096, "units": 131072},
    ]


def _spread(rng, low, high):
    """A size between low and high, even over its logarithm; every second one a multiple of 8."""
    n = min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))
    return max(low, n // 8 * 8) if n >= 16 and rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["norm", "dropout", "gated", "loss"])
    case = {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"])}
    if op in ("norm", "dropout"):
        case |= {"rows": _spread(rng, 1, 16384), "cols": _spread(rng, 16, 4096)}
        if op == "dropout":
            case |= {"p": round(rng.uniform(0.05, 0.6), 3), "residual": rng.random() < 0.5}
    else:
        case |= {"rows": _spread(rng, 1, 8192), "cols": _spread(rng, 64, 4096),
                 "units": _spread(rng, 64, 16384) if op == "gated" else _spread(rng, 10, 131072)}
        if op == "gated":
            case["act"] = rng.choice(["silu", "gelu", "relu"])
    return case


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    rows, cols, op = case["rows"], case["cols"], case["op"]

    def normal(*shape, scale=1.0, shift=0.0):
        # drawn in the type itself: a 32-bit draw of the largest weights would be made and thrown away
        return torch.randn(shape, generator=g, device=dev, dtype=dt).mul_(scale).add_(shift)

    s = {"case": dict(case)}
    if op == "norm":
        s |= {"x": normal(rows, cols, scale=1.5, shift=0.25), "w": normal(cols, scale=0.1, shift=1.0),
              "b": normal(cols, scale=0.1), "dy": normal(rows, cols)}
    elif op == "dropout":
        s |= {"x": normal(rows, cols), "dy": normal(rows, cols),
              "r": normal(rows, cols) if case["residual"] else None,
              # a trainer's seed, and a counter that has already passed 32 bits
              "seed": (seed * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 63), "offset": (1 << 32) - 1000 + seed % 512}
    elif op == "gated":
        s |= {"x": normal(rows, cols), "wg": normal(case["units"], cols, scale=cols ** -0.5),
              "wu": normal(case["units"], cols, scale=cols ** -0.5), "dh": normal(rows, case["units"])}
    else:
        t = torch.randint(0, case["units"], (rows,), generator=g, device=dev)
        # one token in eight is padding, which the loss leaves out; the first never is
        t[1:] = torch.where(torch.rand(rows - 1, generator=g, device=dev) < 0.125, IGNORE, t[1:])
        s |= {"x": normal(rows, cols), "w": normal(case["units"], cols, scale=1.5 * cols ** -0.5), "t": t,
              "dloss": torch.full((), _loss_scale(case), device=dev)}
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return {"norm": _norm, "dropout": _dropout, "gated": _gated, "loss": _loss}[s["case"]["op"]](s)


def _norm(s):
    if own:
        from p2pdl_amd import training
        y, mean, rstd = training.layer_norm_forward(s["x"], s["w"], s["b"], 1e-5)
        dx, dw, db = training.layer_norm_backward(s["dy"], s["x"], mean, rstd, s["w"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    dt = s["x"].dtype
    x, w, b, dy = (s[k].float() for k in ("x", "w", "b", "dy"))
    d = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5)
    n = d * rstd
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    return {"y": (n * w + b).to(dt), "dx": dx.to(dt), "dw": (dy * n).sum(0).to(dt), "db": dy.sum(0).to(dt)}


def _philox(index, seed):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011) of
    the counters (index mod 2^32, index / 2^32, 0, 0) under the key `seed`: four words each, as int64."""
    low = 0xFFFFFFFF
    c0, c1 = index & low, (index >> 32) & low
    c2 = c3 = torch.zeros_like(index)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the low 64 bits of each product, whatever their sign
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), 1)


def _dropout(s):
    c = s["case"]
    if own:
        from p2pdl_amd import training
        return {"y": training.dropout_forward(s["x"], c["p"], s["seed"], s["offset"], residual=s["r"]),
                "dx": training.dropout_backward(s["dy"], c["p"], s["seed"], s["offset"])}
    dt, n = s["x"].dtype, s["x"].numel()
    blocks = torch.arange(s["offset"], s["offset"] + (n + 3) // 4, device=s["x"].device)
    keep = (_philox(blocks, s["seed"]).reshape(-1)[:n] >= int(c["p"] * 2.0 ** 32)).reshape(s["x"].shape)
    scale = 1.0 / (1.0 - c["p"])
    y = torch.where(keep, s["x"].float() * scale, 0.0)
    if s["r"] is not None:
        y = y + s["r"].float()
    return {"y": y.to(dt), "dx": torch.where(keep, s["dy"].float() * scale, 0.0).to(dt)}


def _activation(name, g):
    """act(g) and its derivative."""
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if name == "gelu":
        phi = 0.5 * (1.0 + torch.erf(g * 0.5 ** 0.5))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (2.0 * math.pi) ** -0.5
    on = (g > 0).to(g.dtype)
    return g * on, on


def _gated(s):
    act = s["case"]["act"]
    if own:
        from p2pdl_amd import training
        h, gate, up = training.gated_linear_forward(s["x"], s["wg"], s["wu"], act)
        dx, dwg, dwu = training.gated_linear_backward(s["dh"], s["x"], s["wg"], s["wu"], gate, up, act)
        return {"h": h, "dx": dx, "dwg": dwg, "dwu": dwu}
    dt = s["x"].dtype
    x, wg, wu, dh = (s[k].float() for k in ("x", "wg", "wu", "dh"))
    up = x @ wu.t()
    a, da = _activation(act, x @ wg.t())
    dg, du = dh * up * da, dh * a
    return {"h": (a * up).to(dt), "dx": (dg @ wg + du @ wu).to(dt), "dwg": (dg.t() @ x).to(dt), "dwu": (du.t() @ x).to(dt)}


def _loss(s):
    if own:
        from p2pdl_amd import training
        loss, lse, norm = training.linear_cross_entropy_forward(s["x"], s["w"], s["t"], IGNORE)
        dx, dw = training.linear_cross_entropy_backward(s["x"], s["w"], s["t"], lse, norm, s["dloss"], IGNORE)
        return {"loss": loss, "dx": dx, "dw": dw}
    dt = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    seen = s["t"] != IGNORE
    t = torch.where(seen, s["t"], 0)
    z = x @ w.t()
    z = z - z.amax(1, keepdim=True)
    at = z.gather(1, t[:, None])[:, 0]
    z = z.exp_()
    total = z.sum(1)
    count = seen.sum()
    loss = torch.where(seen, total.log() - at, 0.0).sum() / count
    scale = torch.where(seen, s["dloss"] / count, 0.0)
    z = z.mul_((scale / total)[:, None])
    z.scatter_add_(1, t[:, None], -scale[:, None])
    return {"loss": loss, "dx": (z @ w).to(dt), "dw": (z.t() @ x).to(dt)}


# ------------------------------------------------------------------ the least it can do
def work(case):
    rows, cols = case["rows"], case["cols"]
    size = 4 if case["dtype"] == "f32" else 2
    n = rows * cols
    if case["op"] == "norm":  # x, dy, y, dx, and the weight, the bias and their gradients
        return {"bytes": size * (4 * n + 4 * cols), "flops": 20 * n}
    if case["op"] == "dropout":  # x, y, dy, dx (and the residual)
        return {"bytes": size * n * (5 if case["residual"] else 4), "flops": 3 * n}
    units = case["units"]
    if case["op"] == "gated":  # x, h, dh, dx, both weights and their gradients; two, two and two products
        return {"bytes": size * (2 * n + 2 * rows * units + 4 * units * cols), "flops": 12 * n * units}
    # x, dx, the weight and its gradient, the targets; three products
    return {"bytes": size * (2 * n + 2 * units * cols) + 8 * rows, "flops": 6 * n * units}


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    op = case["op"]
    if op == "norm":
        x, dy = d["x"], d["dy"]
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        std = (var + 1e-5).sqrt()
        xhat = (x - mean) / std
        gw = dy * d["w"]
        dx = (gw - (gw.sum(1, keepdim=True) + xhat * (gw * xhat).sum(1, keepdim=True)) / x.shape[1]) / std
        return {"y": xhat * d["w"] + d["b"], "dx": dx, "dw": (dy * xhat).sum(0), "db": dy.sum(0)}
    if op == "dropout":
        n = case["rows"] * case["cols"]
        place = torch.arange(n, device=d["x"].device)
        block, word = place // 4 + s["offset"], place % 4
        del place
        kept = _word(block, word, s["seed"]).double() / 2.0 ** 32 >= math.floor(case["p"] * 2 ** 32) / 2.0 ** 32
        m = kept.reshape(d["x"].shape).double() / (1.0 - case["p"])
        y = d["x"] * m
        return {"y": y if d["r"] is None else y + d["r"], "dx": d["dy"] * m}
    if op == "gated":
        gate = torch.matmul(d["x"], d["wg"].T).requires_grad_()
        up = torch.matmul(d["x"], d["wu"].T).requires_grad_()
        with torch.enable_grad():
            h = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu}[case["act"]](gate) * up
            dg, du = torch.autograd.grad(h, (gate, up), d["dh"])
        return {"h": h.detach(), "dx": torch.matmul(dg, d["wg"]) + torch.matmul(du, d["wu"]),
                "dwg": torch.matmul(dg.T, d["x"]), "dwu": torch.matmul(du.T, d["x"])}
    rows = torch.nonzero(s["t"] != IGNORE)[:, 0]  # only the tokens that count
    x, t = d["x"][rows], s["t"][rows]
    p = torch.log_softmax(torch.matmul(x, d["w"].T), 1)
    here = torch.arange(len(rows), device=x.device)
    loss = -p[here, t].mean()
    p = p.exp_()
    p[here, t] -= 1.0
    p *= d["dloss"] / len(rows)
    dx = torch.zeros_like(d["x"])
    dx[rows] = torch.matmul(p, d["w"])
    return {"loss": loss, "dx": dx, "dw": torch.matmul(p.T, x)}


def _word(block, word, seed):
    """Word `word` of Philox4x32-10's block `block`, products put together from 16-bit halves."""
    def product(a, m):
        lo, hi = a * (m & 0xFFFF), a * (m >> 16)  # each below 2^48
        t = lo + ((hi & 0xFFFF) << 16)
        return (hi >> 16) + (t >> 32), t & 0xFFFFFFFF

    c = [block % (1 << 32), block // (1 << 32), torch.zeros_like(block), torch.zeros_like(block)]
    k = [seed % (1 << 32), seed >> 32]
    for r in range(10):
        (h0, l0), (h2, l2) = product(c[0], 0xD2511F53), product(c[2], 0xCD9E8D57)
        k0, k1 = (k[0] + r * 0x9E3779B9) % (1 << 32), (k[1] + r * 0xBB67AE85) % (1 << 32)
        c = [torch.bitwise_xor(torch.bitwise_xor(h2, c[1]), k0), l2, torch.bitwise_xor(torch.bitwise_xor(h0, c[3]), k1), l0]
    out = c[0]
    for i in (1, 2, 3):
        out = torch.where(word == i, c[i], out)
    return out
