"""Measured cases of the operators that carry a hidden weight matrix through a training step.

* ``quantize``  -- 8-bit floating point blocks of a matrix and of its transpose (``ops.quantize_fp8``);
* ``linear``    -- the product of a linear layer in 8-bit blocks, alone (``ops.linear_fp8`` without gradients);
* ``train``     -- the same with its input and weight gradients;
* ``orthogonalize`` -- Newton-Schulz orthogonalisation of a stack of update matrices (``ops.orthogonalize``);
* ``muon``      -- one optimizer step on same-shaped matrices: momentum, orthogonalisation, decay, update and the
  bf16 copy of the new weights (``ops.muon_step_``).

``run`` computes them in their plain form (32-bit torch operations) unless ``own`` is true, in which case it makes the
calls a user makes.  Block format: 128 values along the reduction (or a 128 x 128 tile of a weight) share the smallest
power of two that keeps them within the 8-bit type's range; codes and scales are zero-padded to whole blocks, and the
scale bytes (biased exponents) are stored as ``[rows/128, blocks/4, row % 32, row / 32 % 4, block % 4]``.
"""

import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
E4M3_MAX = 448.0


def listed():
    return [
        # one short prompt's tokens through a small projection: all latency
        {"name": "linear 16x1024x1024", "op": "linear", "tokens": 16, "inner": 1024, "outer": 1024},
        # a ragged evaluation batch through a 4B model's gate projection
        {"name": "linear 777x2560x9728", "op": "linear", "tokens": 777, "inner": 2560, "outer": 9728},
        # one 8192-token pack through an 8B model's fused gate/up projection
        {"name": "linear 8192x4096x24576", "op": "linear", "tokens": 8192, "inner": 4096, "outer": 24576},
        # odd widths: a small head on a short pack, forward and backward
        {"name": "train 301x1000x1501", "op": "train", "tokens": 301, "inner": 1000, "outer": 1501},
        # an 8B model's attention output projection on one pack, forward and backward
        {"name": "train 8192x4096x4096", "op": "train", "tokens": 8192, "inner": 4096, "outer": 4096},
        # an 8B model's down projection on one pack, forward and backward
        {"name": "train 8192x12288x4096", "op": "train", "tokens": 8192, "inner": 12288, "outer": 4096},
        # a pack's activations, row blocks for the product and column blocks for the weight gradient
        {"name": "quantize 8192x4096", "op": "quantize", "rows": 8192, "cols": 4096, "tile": False},
        # a ragged weight in 128 x 128 tiles, both orientations
        {"name": "quantize tile 1501x1000", "op": "quantize", "rows": 1501, "cols": 1000, "tile": True},
        # a small model's matrix: sixteen short launches
        {"name": "orthogonalize 1x256x512", "op": "orthogonalize", "count": 1, "rows": 256, "cols": 512},
        # the key (or value) projections of 12 layers of an 8B model, in one call
        {"name": "orthogonalize 12x1024x4096", "op": "orthogonalize", "count": 12, "rows": 1024, "cols": 4096},
        # a few odd-sized tall matrices through the whole update
        {"name": "muon 3x1001x777", "op": "muon", "count": 3, "rows": 1001, "cols": 777},
        # the query and output projections of two layers of an 8B model through the whole update
        {"name": "muon 4x4096x4096", "op": "muon", "count": 4, "rows": 4096, "cols": 4096},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "train", "orthogonalize", "muon"])
    if op in ("linear", "train"):
        tokens = _log_uniform(rng, 1 if op == "linear" else 16, 8192)
        inner, outer = _log_uniform(rng, 256, 12288), _log_uniform(rng, 256, 12288)
        if rng.random() < 0.5:  # widths of real layers are mostly multiples of 128
            inner, outer = max(256, inner // 128 * 128), max(256, outer // 128 * 128)
        while tokens * inner * outer > 8192 * 12288 * 4096:
            tokens = max(1, tokens // 2)
        return {"op": op, "tokens": tokens, "inner": inner, "outer": outer}
    if op == "quantize":
        rows, cols = _log_uniform(rng, 1, 16384), _log_uniform(rng, 8, 8192)
        while rows * cols > 8192 * 4096:
            rows = max(1, rows // 2)
        return {"op": op, "rows": rows, "cols": cols, "tile": rng.random() < 0.5}
    rows, cols = _log_uniform(rng, 8, 6144), _log_uniform(rng, 8, 6144)
    count = _log_uniform(rng, 1, 12)
    while count * rows * cols * min(rows, cols) > 4 * 4096**3:
        count, rows = max(1, count - 1), max(8, rows * 3 // 4)
    return {"op": op, "count": count, "rows": rows, "cols": cols}


def _activations(g, rows, cols):
    """Hidden states: normal values with a few channels an order of magnitude larger and rows of differing size."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    channel = torch.randn(cols, generator=g, device="cuda").mul_(0.5).exp_()
    channel = channel * (1 + 15 * (torch.rand(cols, generator=g, device="cuda") < 0.004))
    row = torch.randn(rows, 1, generator=g, device="cuda").mul_(0.3).exp_()
    return (x * channel * row).to(torch.bfloat16)


def _update(g, rows, cols):
    """A gradient: a decaying spectrum of outer products over noise, rows of differing size."""
    rank = max(1, min(rows, cols, 256) // 2)
    decay = torch.arange(1, rank + 1, device="cuda", dtype=torch.float32).pow_(-0.7)
    low = (torch.randn(rows, rank, generator=g, device="cuda") * decay) @ torch.randn(rank, cols, generator=g, device="cuda")
    noise = torch.randn(rows, cols, generator=g, device="cuda")
    row = torch.randn(rows, 1, generator=g, device="cuda").mul_(0.5).exp_()
    return (low + 0.5 * noise) * row * 1e-3


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    op = case["op"]
    s = {"op": op}
    if op == "quantize":
        x = _activations(g, case["rows"], case["cols"])
        s |= {"x": x, "tile": case["tile"]}
    elif op in ("linear", "train"):
        s["x"] = _activations(g, case["tokens"], case["inner"])
        s["w"] = torch.randn(case["outer"], case["inner"], generator=g, device="cuda").mul_(0.02).to(torch.bfloat16)
        if op == "train":
            scale = torch.randn(case["tokens"], 1, generator=g, device="cuda").exp_() * 1e-4
            dy = torch.randn(case["tokens"], case["outer"], generator=g, device="cuda") * scale
            s["dy"] = dy.to(torch.bfloat16)
            s["x"].requires_grad_(True)
            s["w"].requires_grad_(True)
    elif op == "orthogonalize":
        s["u"] = torch.stack([_update(g, case["rows"], case["cols"]) for _ in range(case["count"])])
    else:
        shape = (case["rows"], case["cols"])
        s["g"] = [_update(g, *shape) for _ in range(case["count"])]
        s["m"] = [_update(g, *shape) for _ in range(case["count"])]
        s["p"] = [torch.randn(shape, generator=g, device="cuda").mul_(0.02) for _ in range(case["count"])]
        s["p_bf16"] = [p.to(torch.bfloat16) for p in s["p"]]
        s["kw"] = {"lr": 2e-4, "momentum": 0.95, "nesterov": True, "weight_decay": 0.1, "steps": STEPS, "eps": EPS,
                   "coefficients": COEFFICIENTS, "adjust_lr": "match_rms_adamw"}
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _power(e):
    """2 ** e of integers in [-126, 127], exactly."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _codes(blocks, dims):
    """Codes (as fp32 values) and exponents of blocks reduced over ``dims``."""
    amax = blocks.abs().amax(dim=dims, keepdim=True)
    f, k = torch.frexp(amax)  # amax = f * 2^k, f in [0.5, 1); 448 = 0.875 * 2^9
    e = (k - 9 + (f > 0.875).to(k.dtype)).clamp(min=-127)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    q = (blocks * _power(-e)).to(torch.float8_e4m3fn)
    return q, e


def _pad(x, rows, cols):
    out = x.new_zeros(rows, cols)
    out[: x.shape[0], : x.shape[1]] = x
    return out


def _up(n, m):
    return -(-n // m) * m


def _quantize(x, tile=False):
    """``(codes [R, C up to 128], exponents [R, blocks])`` of a matrix in row blocks or 128 x 128 tiles."""
    rows, cols = x.shape
    pc = _up(cols, 128)
    if tile:
        pr = _up(rows, 128)
        q, e = _codes(_pad(x.float(), pr, pc).view(pr // 128, 128, pc // 128, 128), (1, 3))
        return q.view(pr, pc)[:rows], e.view(pr // 128, 1, pc // 128).expand(-1, 128, -1).reshape(pr, -1)[:rows]
    q, e = _codes(_pad(x.float(), rows, pc).view(rows, pc // 128, 128), (2,))
    return q.view(rows, pc), e.view(rows, pc // 128)


def _pack(e):
    """Scale bytes in the stored order."""
    rows, blocks = e.shape
    b = _pad((e + 127).to(torch.uint8), _up(rows, 128), _up(blocks, 4))
    b = b.view(b.shape[0] // 128, 4, 32, b.shape[1] // 4, 4)
    return b.permute(0, 3, 2, 1, 4).contiguous()


def _values(x, tile=False):
    q, e = _quantize(x, tile)
    scale = torch.where(e > -127, _power(e.clamp(min=-126)), torch.full_like(e, 0, dtype=torch.float32))
    return (q.float().view(x.shape[0], -1, 128) * scale[..., None]).view(x.shape[0], -1)[:, : x.shape[1]]


def _newton_schulz(u):
    """The quintic iteration on a stack of matrices, in 32 bits."""
    norm = u.double().square().sum(dim=(-2, -1), keepdim=True).sqrt().float()
    x = u / norm.clamp(min=EPS)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if tall else x


def _plain(s):
    op = s["op"]
    if op == "quantize":
        (q, e), (qt, et) = _quantize(s["x"], s["tile"]), _quantize(s["x"].t(), s["tile"])
        return {"data": q, "scale": _pack(e), "data_t": qt, "scale_t": _pack(et)}
    if op in ("linear", "train"):
        x, w = s["x"].detach(), s["w"].detach()
        wv = _values(w, tile=True)
        y = (_values(x) @ wv.t()).to(x.dtype)
        if op == "linear":
            return {"y": y}
        dy = s["dy"]
        dx = (_values(dy) @ wv).to(x.dtype)
        dw = (_values(dy.t()) @ _values(x.t()).t()).to(w.dtype)
        return {"y": y, "dx": dx, "dw": dw}
    if op == "orthogonalize":
        return {"o": _newton_schulz(s["u"]).to(torch.bfloat16)}
    kw = s["kw"]
    rows, cols = s["p"][0].shape
    u = []
    for g, m in zip(s["g"], s["m"]):
        m.lerp_(g, 1 - kw["momentum"])
        u.append(g.lerp(m, kw["momentum"]))
    o = _newton_schulz(torch.stack(u))
    ratio = 0.2 * math.sqrt(max(rows, cols))
    for i, p in enumerate(s["p"]):
        p.mul_(1 - kw["lr"] * kw["weight_decay"]).add_(o[i], alpha=-kw["lr"] * ratio)
        s["p_bf16"][i].copy_(p)
    return {"p": s["p"], "m": s["m"], "p_bf16": s["p_bf16"]}


def run(state):
    if not own:
        with torch.no_grad():
            return _plain(state)
    from mvp_engine import ops

    s, op = state, state["op"]
    if op == "quantize":
        q, qt = ops.quantize_fp8(s["x"], block="tile" if s["tile"] else "row", rows=True, columns=True)
        return {"data": q.data, "scale": q.scale, "data_t": qt.data, "scale_t": qt.scale}
    if op == "linear":
        with torch.no_grad():
            return {"y": ops.linear_fp8(s["x"], s["w"])}
    if op == "train":
        y = ops.linear_fp8(s["x"], s["w"])
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    if op == "orthogonalize":
        return {"o": ops.orthogonalize(s["u"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)}
    ops.muon_step_(s["p"], s["g"], s["m"], p_bf16=s["p_bf16"], **s["kw"])
    return {"p": s["p"], "m": s["m"], "p_bf16": s["p_bf16"]}


def work(case):
    op = case["op"]
    if op == "quantize":
        rows, cols = case["rows"], case["cols"]
        per = 1 if case["tile"] else 128  # rows that share a scale's block
        scales = _up(rows, 128) // 128 * -(-cols // 128) * (2 if per == 1 else 256)
        return {"bytes": 4 * rows * cols + scales, "flops": 0}
    if op in ("linear", "train"):
        t, k, n = case["tokens"], case["inner"], case["outer"]
        if op == "linear":
            return {"bytes": 2 * (t * k + n * k + t * n), "flops": 2 * t * k * n}
        return {"bytes": 2 * (2 * t * k + 2 * n * k + 2 * t * n), "flops": 6 * t * k * n}
    short, long = sorted((case["rows"], case["cols"]))
    size = case["count"] * short * long
    # a symmetric product costs half: X X^T and A A by halves, B X whole
    flops = case["count"] * STEPS * (3 * short * short * long + short**3)
    if op == "orthogonalize":
        return {"bytes": 6 * size, "flops": flops}
    return {"bytes": (4 + 8 + 8 + 2) * size, "flops": flops}


# ------------------------------------------------------------------------------------------- 64-bit definition
def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_blocks(x, tile, transpose):
    """Codes and exponents from the definition: the least e with amax <= 448 * 2^e, then nearest-even 8-bit values."""
    x = x.detach().double()
    x = x.t() if transpose else x
    rows, cols = x.shape
    nb, nr = -(-cols // 128), -(-rows // 128)
    amax = torch.zeros(rows, nb, dtype=torch.float64, device=x.device)
    for j in range(nb):
        amax[:, j] = x[:, j * 128 : (j + 1) * 128].abs().max(dim=1).values
    if tile:
        for i in range(nr):
            amax[i * 128 : (i + 1) * 128] = amax[i * 128 : (i + 1) * 128].max(dim=0).values
    log = torch.log2(amax / E4M3_MAX)  # whole where amax is 448 times a power of two, else at least 8e-8 away from whole
    near = torch.round(log)
    e = torch.where((log - near).abs() < 1e-9, near, torch.ceil(log)).clamp(min=-127)
    per_value = e.repeat_interleave(128, dim=1)[:, :cols]
    v = x * _power64(-per_value)
    binade = torch.floor(torch.log2(v.abs().clamp(min=2.0**-20))).clamp(min=-6)
    quantum = _power64(binade - 3)
    return torch.round(v / quantum) * quantum, e, per_value


def _exact_values(x, tile=False, transpose=False):
    q, _, per_value = _exact_blocks(x, tile, transpose)
    return q * _power64(per_value)


def _exact_orthogonal(u):
    a, b, c = COEFFICIENTS
    x = u / torch.linalg.matrix_norm(u, keepdim=True).clamp(min=EPS)
    for _ in range(STEPS):
        if x.shape[-2] <= x.shape[-1]:
            s = torch.matmul(x, x.transpose(-1, -2))
            x = a * x + b * torch.matmul(s, x) + c * torch.matmul(s, torch.matmul(s, x))
        else:
            s = torch.matmul(x.transpose(-1, -2), x)
            x = a * x + b * torch.matmul(x, s) + c * torch.matmul(torch.matmul(x, s), s)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "quantize":
        found = {}
        for name, transpose in (("", False), ("_t", True)):
            q, e, _ = _exact_blocks(s["x"], s["tile"], transpose)
            data = torch.zeros(q.shape[0], e.shape[1] * 128, dtype=torch.float64, device=q.device)
            data[:, : q.shape[1]] = q
            scale = torch.zeros(_up(e.shape[0], 128), _up(e.shape[1], 4), dtype=torch.uint8, device=q.device)
            scale[: e.shape[0], : e.shape[1]] = (e + 127).to(torch.uint8)
            r = torch.arange(scale.shape[0], device=q.device).view(-1, 4, 32).transpose(1, 2)  # [row group, r % 32, r / 32]
            j = torch.arange(scale.shape[1], device=q.device).view(-1, 4)
            found |= {"data" + name: data, "scale" + name: scale[r[:, None, :, :, None], j[None, :, None, None, :]]}
        return found
    if op in ("linear", "train"):
        w = _exact_values(s["w"], tile=True)
        found = {"y": _exact_values(s["x"]) @ w.t()}
        if op == "train":
            found["dx"] = _exact_values(s["dy"]) @ w
            found["dw"] = _exact_values(s["dy"], transpose=True) @ _exact_values(s["x"], transpose=True).t()
        return found
    if op == "orthogonalize":
        return {"o": _exact_orthogonal(s["u"].double())}
    kw, found = s["kw"], {"p": [], "m": [], "p_bf16": []}
    for p, g, m in zip(s["p"], s["g"], s["m"]):
        p, g, m = p.double(), g.double(), m.double()
        m = kw["momentum"] * m + (1 - kw["momentum"]) * g
        u = (1 - kw["momentum"]) * g + kw["momentum"] * m
        step = kw["lr"] * 0.2 * max(p.shape) ** 0.5
        p = p - kw["lr"] * kw["weight_decay"] * p - step * _exact_orthogonal(u)
        found["m"].append(m)
        found["p"].append(p)
        found["p_bf16"].append(p)
    return found
