"""The framework's operators of a model's training step, as cases that can be timed
and compared: the linear layer on an 8-bit floating-point weight with block scales
(``qweight.FP8QWeight``), the codec of that weight, and the cross entropy of a linear
head that never holds its logits (``linear_cross_entropy``).

``run`` computes a case in plain form (32-bit torch operations) or, where ``own`` is
true, through the framework's public entry points.
"""

import math

import torch

own = False

BLOCK = 128
FP8_MAX = 448.0


# ------------------------------------------------------------------------ cases


def _linear(name, tokens, inputs, outputs, dtype="bf16", backward=True, bias=False):
    return dict(name=name, op="linear", tokens=tokens, inputs=inputs, outputs=outputs,
                dtype=dtype, backward=backward, bias=bias)


def _loss(name, tokens, hidden, vocab, dtype="bf16", backward=True, reduction="mean"):
    return dict(name=name, op="loss", tokens=tokens, hidden=hidden, vocab=vocab, dtype=dtype,
                backward=backward, reduction=reduction)


def listed():
    return [
        # generating one token: the up projection of the 8B model, weight-read bound
        _linear("linear 1 token", 1, 4096, 14336, backward=False),
        # a small serving batch through the down projection
        _linear("linear 24 tokens", 24, 14336, 4096, dtype="fp16", backward=False),
        # a toy model's layer (test sizes): everything is launch latency, nothing is a
        # multiple of a block
        _linear("linear step tiny", 100, 688, 250, dtype="fp16", bias=True),
        # one micro-batch of the 1.1B model through its up projection
        _linear("linear step 1b", 4096, 2048, 5632),
        # one micro-batch of the 8B model through its up projection
        _linear("linear step 8b", 4096, 4096, 14336),
        # a long batch through the 8B model's down projection
        _linear("linear step 16k", 16384, 14336, 4096),
        # the optimizer's new fp32 master into the payload, and the payload read back
        dict(name="requantise 8b", op="requantise", outputs=14336, inputs=4096, dtype="bf16"),
        # a toy model's loss: launch latency
        _loss("loss step tiny", 64, 256, 1024),
        # per-token losses and their gradients, no size a multiple of a tile
        _loss("loss step ragged", 333, 1000, 32003, dtype="fp16", reduction="none"),
        # evaluation of the 1.1B model: no gradient wanted
        _loss("loss evaluation 1b", 2048, 2048, 32000, backward=False),
        # one micro-batch of the 1.1B model
        _loss("loss step 1b", 4096, 2048, 32000),
        # one micro-batch of the 8B model
        _loss("loss step 8b", 4096, 4096, 128256),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "fp16"])
    op = rng.choice(["linear", "linear", "loss", "loss", "requantise"])
    if op == "linear":
        limit = 16384 * 14336 * 4096
        while True:
            tokens = _log_uniform(rng, 1, 16384)
            inputs = 16 * _log_uniform(rng, 4, 896)
            outputs = _log_uniform(rng, 64, 14336)
            if tokens * inputs * outputs <= limit:
                break
        return dict(op=op, tokens=tokens, inputs=inputs, outputs=outputs, dtype=dtype,
                    backward=rng.random() < 0.7, bias=rng.random() < 0.3)
    if op == "requantise":
        return dict(op=op, outputs=_log_uniform(rng, 64, 14336),
                    inputs=16 * _log_uniform(rng, 4, 256), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    limit = 4096 * 4096 * 128256
    while True:
        tokens = _log_uniform(rng, 1, 8192)
        hidden = 8 * _log_uniform(rng, 8, 512)
        vocab = _log_uniform(rng, 257, 131072)
        if tokens * hidden * vocab <= limit:
            break
    return dict(op=op, tokens=tokens, hidden=hidden, vocab=vocab, dtype=dtype,
                backward=rng.random() < 0.7, reduction=rng.choice(["mean", "sum", "none"]))


_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _size(case):
    return {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]


def work(case):
    e = _size(case)
    if case["op"] == "linear":
        t, k, n = case["tokens"], case["inputs"], case["outputs"]
        scales = -(-k // BLOCK) * -(-n // BLOCK)
        nbytes = e * t * k + n * k + scales + e * t * n + (e * n if case["bias"] else 0)
        flops = 2 * t * k * n
        if case["backward"]:  # reads the output's gradient, writes dx, dw (and db)
            nbytes += e * t * n + e * t * k + e * n * k + (e * n if case["bias"] else 0)
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "requantise":
        n, k = case["outputs"], case["inputs"]
        # master read, payload written and read, decoded weight written
        return {"bytes": n * k * (4 + 2 + e), "flops": 4 * n * k}
    t, h, v = case["tokens"], case["hidden"], case["vocab"]
    nbytes = e * t * h + e * v * h + 8 * t + 4 * (t if case["reduction"] == "none" else 1)
    flops = 2 * t * h * v
    if case["backward"]:
        nbytes += e * t * h + e * v * h
        flops *= 3
    return {"bytes": nbytes, "flops": flops}


# ----------------------------------------------------------------------- inputs


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=dev) * std

    if case["op"] == "requantise":
        # weights of mixed magnitude: every row has its own scale, one element in a
        # hundred is an outlier
        n, k = case["outputs"], case["inputs"]
        master = normal(n, k, std=0.02) * torch.exp2(normal(n, 1))
        master = torch.where(torch.rand(n, k, generator=g, device=dev) < 0.01, master * 10, master)
        s = dict(case=case, master=master.contiguous(), dtype=dt)
        if own:
            s["weight"] = _own_weight(torch.zeros_like(master, dtype=dt))
        return s
    if case["op"] == "linear":
        t, k, n = case["tokens"], case["inputs"], case["outputs"]
        x = normal(t, k) * torch.exp(0.5 * normal(k))  # features of unequal size, as a norm leaves them
        codes, scale = _encode(normal(n, k, std=0.02), BLOCK, BLOCK)
        s = dict(case=case, x=x.to(dt), codes=codes, scale=scale, dtype=dt, bias=None)
        if case["bias"]:
            s["bias"] = normal(n, std=0.02).to(dt)
        if case["backward"]:
            # a few tokens carry most of a gradient
            s["gy"] = (normal(t, n, std=1e-3) * torch.exp(normal(t, 1))).to(dt)
            s["x"].requires_grad_(True)
            if s["bias"] is not None:
                s["bias"].requires_grad_(True)
        if own:
            s["weight"] = _own_weight_from(codes, scale, dt, case["backward"])
        return s
    t, h, v = case["tokens"], case["hidden"], case["vocab"]
    w = normal(v, h, std=0.02)
    target = torch.randint(v, (t,), generator=g, device=dev)
    # half-trained: the hidden state leans towards its target's row, more or less far
    x = normal(t, h) + 20.0 * torch.rand(t, 1, generator=g, device=dev) * w[target]
    if t > 4:  # padding and prompt tokens take no part
        target = torch.where(torch.rand(t, generator=g, device=dev) < 0.1, -100, target)
    s = dict(case=case, x=x.to(dt), w=w.to(dt), target=target)
    if case["backward"]:
        s["x"].requires_grad_(True)
        s["w"].requires_grad_(True)
        shape = (t,) if case["reduction"] == "none" else ()
        s["g"] = 0.5 + torch.rand(shape, generator=g, device=dev)
    return s


def _own_weight(w):
    from offload_adam_amd.qweight import FP8QWeight

    return FP8QWeight.from_float(w)


def _own_weight_from(codes, scale, dtype, train):
    from offload_adam_amd.qweight import FP8QWeight

    w = FP8QWeight(codes, scale.to(torch.float8_e8m0fnu), dtype)
    return torch.nn.Parameter(w, requires_grad=train)


# ------------------------------------------------------------------- plain form


def _blocks(x, rows, cols):
    """(R, C) -> (ceil(R/rows), rows, ceil(C/cols), cols), padded with zeros."""
    r, c = x.shape
    x = torch.nn.functional.pad(x, (0, -c % cols, 0, -r % rows))
    return x.reshape(-(-r // rows), rows, -(-c // cols), cols)


def _encode(x, rows, cols):
    """e4m3 codes of ``x`` (R, C) and one power-of-two scale per ``rows`` x ``cols``
    block (R/rows, C/cols): the smallest that brings the block's largest magnitude to
    448 or less."""
    r, c = x.shape
    b = _blocks(x.float(), rows, cols)
    mant, exp = torch.frexp(b.abs().amax(dim=(1, 3)))
    e = torch.where(mant > 0.875, exp - 8, exp - 9)
    e = torch.where(mant == 0, 0, e).clamp(-126, 127)
    # powers of two by their bits: exp2 and ldexp may be an ulp off, which moves ties
    down = ((127 - e) << 23).to(torch.int32).view(torch.float32)
    codes = (b * down[:, None, :, None]).to(torch.float8_e4m3fn)
    codes = codes.reshape(b.shape[0] * rows, -1)[:r, :c].contiguous()
    return codes, ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _decode(codes, scale, rows, cols):
    r, c = codes.shape
    b = _blocks(codes.float(), rows, cols) * scale[:, None, :, None]
    return b.reshape(b.shape[0] * rows, -1)[:r, :c]


def _rounded(x, rows, cols):
    """The values that 8-bit codes of ``x`` with ``rows`` x ``cols`` scale blocks hold."""
    return _decode(*_encode(x, rows, cols), rows, cols)


def _plain_linear(s):
    x, dt = s["x"].detach(), s["dtype"]
    w = _decode(s["codes"], s["scale"], BLOCK, BLOCK)
    y = _rounded(x, 1, BLOCK) @ w.T
    if s["bias"] is not None:
        y = y + s["bias"].detach().float()
    out = {"y": y.to(dt)}
    if s["case"]["backward"]:
        gy = s["gy"]
        out["dx"] = (_rounded(gy, 1, BLOCK) @ w).to(dt)
        out["dw"] = (_rounded(gy, BLOCK, 1).T @ _rounded(x, BLOCK, 1)).to(dt)
        if s["bias"] is not None:
            out["db"] = gy.float().sum(0).to(dt)
    return out


def _plain_loss(s):
    case, x, w, target = s["case"], s["x"].detach().float(), s["w"].detach().float(), s["target"]
    z = x @ w.T
    top = z.amax(dim=1, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(dim=1, keepdim=True)
    used = target != -100
    at = torch.where(used, target, 0)[:, None]
    each = (torch.log(total) + top - z.gather(1, at))[:, 0] * used
    count = used.sum().float()
    loss = {"none": each, "sum": each.sum(), "mean": each.sum() / count}[case["reduction"]]
    out = {"loss": loss}
    if case["backward"]:
        dz = p / total
        dz.scatter_add_(1, at, torch.full_like(dz[:, :1], -1.0))
        up = s["g"] / count if case["reduction"] == "mean" else s["g"]
        dz = dz * (up * used)[:, None]
        out["dx"] = (dz @ w).to(s["x"].dtype)
        out["dw"] = (dz.T @ x).to(s["w"].dtype)
    return out


def run(state):
    case = state["case"]
    if own:
        return _own_run(state)
    if case["op"] == "linear":
        return _plain_linear(state)
    if case["op"] == "requantise":
        return _rounded(state["master"], BLOCK, BLOCK).to(state["dtype"])
    return _plain_loss(state)


def _own_run(s):
    case = s["case"]
    if case["op"] == "requantise":
        s["weight"].copy_(s["master"])
        return s["weight"].dequantize()
    if case["op"] == "linear":
        y = torch.nn.functional.linear(s["x"], s["weight"], s["bias"])
        out = {"y": y.detach()}
        if case["backward"]:
            wanted = [s["x"], s["weight"]] + ([s["bias"]] if s["bias"] is not None else [])
            out.update(zip(("dx", "dw", "db"), torch.autograd.grad(y, wanted, s["gy"])))
        return out
    from offload_adam_amd import linear_cross_entropy

    loss = linear_cross_entropy(s["x"], s["w"], s["target"], reduction=case["reduction"])
    out = {"loss": loss.detach()}
    if case["backward"]:
        out["dx"], out["dw"] = torch.autograd.grad(loss, (s["x"], s["w"]), s["g"])
    return out


# --------------------------------------------------------- 64-bit from the definition


def _power(e):
    """2^e in 64 bits, by its exponent bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _held(x, dim):
    """What 8-bit codes hold of ``x`` in 64 bits, blocks of 128 along ``dim``; ``dim``
    None: blocks of 128 x 128.  Rounds each element to the nearest multiple of its
    binade's step (2^-3 of the binade, at least 2^-9), ties to even."""
    x = x.double()
    m = x.abs()
    for d in (0, 1) if dim is None else (dim,):
        n = m.shape[d]
        pad = [0, 0, 0, 0]
        pad[3 if d == 0 else 1] = -n % BLOCK
        m = torch.nn.functional.pad(m, pad).unflatten(d, (-1, BLOCK)).amax(dim=d + 1)
    e = torch.ceil(torch.log2((m / FP8_MAX).clamp_min(2.0**-200)))
    e = e + (m > FP8_MAX * _power(e)).double()
    e = e - (m <= FP8_MAX * _power(e - 1)).double()
    scale = _power(torch.where(m == 0, 0.0, e.clamp(-126, 127)))
    for d in (0, 1) if dim is None else (dim,):
        scale = scale.repeat_interleave(BLOCK, dim=d).narrow(d, 0, x.shape[d])
    v = x / scale
    _, binade = torch.frexp(v.abs().clamp_min(2.0**-6))  # v = f * 2^binade, 1/2 <= f < 1
    step = _power(binade - 4)
    return torch.round(v / step) * step * scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "requantise":
        return _held(s["master"], None)
    if case["op"] == "linear":
        n, k = s["codes"].shape
        spread = s["scale"].double().repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)
        w = s["codes"].float().double() * spread[:n, :k]
        x = s["x"].detach()
        y = torch.mm(_held(x, 1), w.t().contiguous())
        if s["bias"] is not None:
            y += s["bias"].detach().double()
        out = {"y": y}
        if case["backward"]:
            out["dx"] = torch.mm(_held(s["gy"], 1), w)
            out["dw"] = torch.mm(_held(s["gy"], 0).t().contiguous(), _held(x, 0))
            if s["bias"] is not None:
                out["db"] = s["gy"].double().sum(0)
        return out
    x, w, target = s["x"].detach().double(), s["w"].detach().double(), s["target"]
    t, v = x.shape[0], w.shape[0]
    keep = (target >= 0).double()
    count = keep.sum()
    each = torch.zeros(t, dtype=torch.float64, device=x.device)
    dx = torch.zeros_like(x)
    dw = torch.zeros_like(w)
    for lo in range(0, t, 1024):  # tokens are independent of each other
        hi = min(t, lo + 1024)
        z = torch.mm(x[lo:hi], w.t().contiguous())
        lse = torch.logsumexp(z, dim=1)
        hot = (target[lo:hi, None] == torch.arange(v, device=x.device)[None]).double()
        each[lo:hi] = (lse - (z * hot).sum(1)) * keep[lo:hi]
        if case["backward"]:
            up = s["g"].double().expand(t)[lo:hi] * keep[lo:hi]
            if case["reduction"] == "mean":
                up = up / count
            dz = (torch.exp(z - lse[:, None]) - hot) * up[:, None]
            dx[lo:hi] = torch.mm(dz, w)
            dw += torch.mm(dz.t().contiguous(), x[lo:hi])
    total = each.sum()
    loss = {"none": each, "sum": total, "mean": total / count}[case["reduction"]]
    return {"loss": loss, "dx": dx, "dw": dw} if case["backward"] else {"loss": loss}
