"""Cases of the 8-bit linear layer (block quantisation, block-scaled product, the layer's forward and backward) and of
sliding-window attention with sink tokens (forward, forward + backward), with their plain forms in elementary torch
operations and their definitions in 64 bits.

``own = False`` computes the plain forms; ``own = True`` makes the calls a training program makes of the framework.

Quantisation. A block of 128 neighbouring values (along a row, along a column, or a 128 x 128 tile) shares the scale
2^e, e the smallest integer with max|x| <= 448 * 2^e, at least -127 (also for a block of zeros); it is held as the byte
e + 127. A value is x / 2^e rounded to the nearest e4m3 number, ties to even. The blocks at the end are partial.
``rows``: blocks along a row of x [R, C]. ``columns``: blocks along a column, laid out transposed, [C, R]. ``tiles``:
one scale for a tile, laid out as x and transposed. Rows of 8-bit values are padded with zeros to a multiple of 128,
rows of scales to a multiple of 4.

Attention. Query t sees key s when s <= t and (t - s < window or s < sinks).
"""
import math

import torch

own = False

BLOCK = 128


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a single sentence's activations in front of a linear layer of GPT-2 Large: latency
        {"name": "quantize rows 64x1280", "op": "quantize", "rows": 64, "cols": 1280, "blocks": "rows", "dtype": "bf16"},
        # the MLP activations of the benchmark's 64 x 1024 tokens, quantised for both products that read them
        {"name": "quantize both 65536x5120", "op": "quantize", "rows": 65536, "cols": 5120, "blocks": "both", "dtype": "bf16"},
        # an fp32 weight of GPT-2 XL's MLP, both layouts
        {"name": "quantize tiles 6400x1600", "op": "quantize", "rows": 6400, "cols": 1600, "blocks": "tiles", "dtype": "fp32"},
        # few tokens through the QKV projection of GPT-2 Large, weight quantised beforehand
        {"name": "product 16x3840x1280", "op": "product", "m": 16, "n": 3840, "k": 1280, "bias": True, "out": "bf16"},
        # a micro-batch of 8 x 1024 tokens through the MLP's second product of GPT-2 Large
        {"name": "product 8192x1280x5120", "op": "product", "m": 8192, "n": 1280, "k": 5120, "bias": True, "out": "bf16"},
        # off every tile: token count, width and contraction odd
        {"name": "product 1003x1601x777", "op": "product", "m": 1003, "n": 1601, "k": 777, "bias": False, "out": "fp32"},
        # a training step through one linear layer, small model, ragged tokens, fp32 storage
        {"name": "linear 999x256x512", "op": "linear", "m": 999, "n": 512, "k": 256, "bias": True, "dtype": "fp32"},
        # the first MLP product of GPT-2 Large at the reference's micro-batch of 8 x 1024 tokens
        {"name": "linear 8192x1280x5120", "op": "linear", "m": 8192, "n": 5120, "k": 1280, "bias": True, "dtype": "bf16"},
        # the widest product of Llama-7B, 4 x 2048 tokens
        {"name": "linear 8192x4096x22016", "op": "linear", "m": 8192, "n": 22016, "k": 4096, "bias": False, "dtype": "bf16"},
        # forward only (evaluation) over GPT-2 Large's heads, window of a quarter of the context
        {"name": "window 8x1024 h20 d64", "op": "window", "b": 8, "t": 1024, "h": 20, "d": 64, "window": 256, "sinks": 4, "grad": False},
        # a short ragged batch, forward and backward, window and sinks off the tiles
        {"name": "window 3x333 h5 d64 grad", "op": "window", "b": 3, "t": 333, "h": 5, "d": 64, "window": 100, "sinks": 5, "grad": True},
        # a long sequence through Llama-7B's heads, forward and backward
        {"name": "window 1x8192 h32 d128 grad", "op": "window", "b": 1, "t": 8192, "h": 32, "d": 128, "window": 1024, "sinks": 4, "grad": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "linear", "window"])
    if op == "quantize":
        while True:
            rows, cols = _log_int(rng, 1, 65536), _log_int(rng, 64, 11008)
            if rows * cols <= 65536 * 5120 // 2:
                break
        return {"op": op, "rows": rows, "cols": cols, "blocks": rng.choice(["rows", "columns", "both", "tiles"]),
                "dtype": rng.choice(["bf16", "fp32"])}
    if op == "product":
        while True:
            m, n, k = _log_int(rng, 1, 16384), _log_int(rng, 32, 22016), _log_int(rng, 64, 11008)
            if m * n * k <= 8192 * 4096 * 22016:
                break
        return {"op": op, "m": m, "n": n, "k": k, "bias": rng.random() < 0.5, "out": rng.choice(["bf16", "fp32"])}
    if op == "linear":
        while True:
            m, n, k = _log_int(rng, 8, 16384), _log_int(rng, 64, 22016), _log_int(rng, 64, 11008)
            if m * n * k <= 8192 * 4096 * 22016:
                break
        return {"op": op, "m": m, "n": n, "k": k, "bias": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp32"])}
    while True:
        b, t, h = rng.randint(1, 8), _log_int(rng, 1, 8192), rng.choice([1, 2, 5, 12, 16, 20, 25, 32])
        if b * h * t * t <= 32 * 8192 * 8192:
            break
    return {"op": op, "b": b, "t": t, "h": h, "d": rng.choice([64, 128]), "window": _log_int(rng, 1, max(1, t)),
            "sinks": rng.choice([0, 1, 4, 16, 64, 100]), "grad": rng.random() < 0.6}


DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def visible_pairs(t, window, sinks):
    """(query, key) pairs of one head that are not masked."""
    total = 0
    near = min(t, window)
    total += near * (near + 1) // 2 + (t - near) * window  # the window
    far = max(0, t - window)  # query window + i (i < far) sees sinks among its i + 1 keys before the window
    s = min(sinks, far)
    total += s * (s + 1) // 2 + (far - s) * s
    return total


def work(case):
    op = case["op"]
    if op == "quantize":
        n, size = case["rows"] * case["cols"], 2 if case["dtype"] == "bf16" else 4
        copies = 2 if case["blocks"] in ("both", "tiles") else 1
        per = BLOCK * BLOCK if case["blocks"] == "tiles" else BLOCK
        return {"bytes": n * size + copies * (n + n // per), "flops": 2 * n}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        size = 2 if case["out"] == "bf16" else 4
        return {"bytes": (m + n) * k + m * k // BLOCK + m * n * size, "flops": 2 * m * n * k}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": 2 * (m * k + n * k + m * n) * size, "flops": 6 * m * n * k}
    b, t, h, d = case["b"], case["t"], case["h"], case["d"]
    pairs = b * h * visible_pairs(t, case["window"], case["sinks"])
    token = b * t * h * d * 2
    if case["grad"]:
        return {"bytes": 3 * token + token + token + 3 * token, "flops": 14 * d * pairs}
    return {"bytes": 3 * token + token, "flops": 4 * d * pairs}


# ----------------------------------------------------------------------------------------------------------- inputs
def _pad(x, rows, cols):
    r, c = -x.shape[0] % rows, -x.shape[1] % cols
    return torch.nn.functional.pad(x, (0, c, 0, r)) if r or c else x


def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


def _randn(shape, seed, k, dtype=torch.float32):
    g = torch.Generator(device=_device()).manual_seed(seed * 16 + k)
    return torch.randn(shape, generator=g, device=_device(), dtype=dtype)


def _activations(rows, cols, seed, k, dtype):
    """Rows of different sizes and a few wide columns, as in the activations of a trained network."""
    x = _randn((rows, cols), seed, k)
    x *= torch.exp2(2.0 * _randn((rows, 1), seed, k + 1))
    x *= 1.0 + 20.0 * (_randn((1, cols), seed, k + 2) > 2.5)
    return x.to(dtype)


def prepare(case, seed):
    op = case["op"]
    if op == "quantize":
        return {"case": case, "x": _activations(case["rows"], case["cols"], seed, 0, DTYPES[case["dtype"]])}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a_q, a_e = _quantize_rows(_activations(m, k, seed, 0, torch.float32))
        b_q, b_e, _, _ = _quantize_tiles(0.02 * _randn((n, k), seed, 3))
        bias = 0.1 * _randn((n,), seed, 4) if case["bias"] else None
        return {"case": case, "a_q": a_q, "a_e": a_e, "b_q": b_q, "b_e": b_e,
                "bias": bias if bias is None else bias.to(DTYPES[case["out"]])}
    if op == "linear":
        m, n, k, dtype = case["m"], case["n"], case["k"], DTYPES[case["dtype"]]
        x = _activations(m, k, seed, 0, dtype).requires_grad_()
        w = (0.02 * _randn((n, k), seed, 3)).to(dtype).requires_grad_()
        bias = (0.1 * _randn((n,), seed, 4)).to(dtype).requires_grad_() if case["bias"] else None
        return {"case": case, "x": x, "w": w, "bias": bias, "dy": _activations(m, n, seed, 5, dtype)}
    b, t, h, d = case["b"], case["t"], case["h"], case["d"]
    qkv = _randn((b, t, 3 * h * d), seed, 0).to(torch.bfloat16)
    dout = _randn((b, t, h * d), seed, 1).to(torch.bfloat16) if case["grad"] else None
    return {"case": case, "qkv": qkv.requires_grad_() if case["grad"] else qkv, "dout": dout}


# ------------------------------------------------------------------------------------------------------ plain forms
def _exponent(amax):
    m, k = torch.frexp(amax)  # amax = m 2^k, 0.5 <= m < 1, and 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, k - 9, k - 8)
    return torch.where(amax > 0, e, -127).clamp_(min=-127)


def _scale_bytes(e):
    return torch.nn.functional.pad((e + 127).to(torch.uint8), (0, -e.shape[1] % 4))


def _quantize_rows(x):
    v = _pad(x.float(), 1, BLOCK)
    v = v.view(v.shape[0], -1, BLOCK)
    e = _exponent(v.abs().amax(2))
    q = torch.ldexp(v, -e.unsqueeze(2)).to(torch.float8_e4m3fn)
    return q.view(q.shape[0], -1), _scale_bytes(e)


def _quantize_tiles(x):
    r, c = x.shape
    v = _pad(x.float(), BLOCK, BLOCK)
    v = v.view(v.shape[0] // BLOCK, BLOCK, -1, BLOCK)
    e = _exponent(v.abs().amax((1, 3)))
    q = torch.ldexp(v, -e[:, None, :, None]).flatten(2).flatten(0, 1)
    return (q[:r].to(torch.float8_e4m3fn), _scale_bytes(e),
            q[:, :c].t().contiguous().to(torch.float8_e4m3fn), _scale_bytes(e.t().contiguous()))


def _values(q, bytes_, tiles=False):
    """What a quantised matrix stands for, with the padding of its rows."""
    e = bytes_[:, : q.shape[1] // BLOCK].to(torch.int32) - 127
    if tiles:
        e = e.repeat_interleave(BLOCK, 0)[: q.shape[0]]
    v = q.float().view(q.shape[0], -1, BLOCK)
    return torch.ldexp(v, e.unsqueeze(2)).view(q.shape[0], -1)


def _plain_quantize(x, blocks):
    if blocks == "tiles":
        return _quantize_tiles(x)
    rows = _quantize_rows(x) if blocks in ("rows", "both") else ()
    columns = _quantize_rows(x.t()) if blocks in ("columns", "both") else ()
    return rows + columns


def _plain_linear(x, w, bias, dy):
    k, dtype = x.shape[1], x.dtype
    w_q, w_e, wt_q, wt_e = _quantize_tiles(w)
    y = _values(*_quantize_rows(x)) @ _values(w_q, w_e, True).t()
    if bias is not None:
        y = y + bias.float()
    dx = _values(*_quantize_rows(dy)) @ _values(wt_q, wt_e, True).t()
    dw = _values(*_quantize_rows(dy.t())) @ _values(*_quantize_rows(x.t())).t()
    out = [y.to(dtype), dx[:, :k].to(dtype), dw.to(dtype)]
    return out + [dy.float().sum(0).to(dtype)] if bias is not None else out


def _visible(t, window, sinks, device):
    i = torch.arange(t, device=device)
    q, k = i[:, None], i[None, :]
    return (k <= q) & ((q - k < window) | (k < sinks))


def _plain_window(case, qkv, dout):
    b, t, h, d = case["b"], case["t"], case["h"], case["d"]
    scale = 1.0 / math.sqrt(d)
    q, k, v = qkv.float().view(b, t, 3, h, d).permute(2, 0, 3, 1, 4).reshape(3, b * h, t, d)
    s = torch.bmm(q, k.transpose(1, 2)).mul_(scale)
    s.masked_fill_(~_visible(t, case["window"], case["sinks"], s.device), float("-inf"))
    p = s.sub_(s.amax(2, keepdim=True)).exp_()
    p.div_(p.sum(2, keepdim=True))
    o = torch.bmm(p, v)
    out = o.view(b, h, t, d).transpose(1, 2).reshape(b, t, h * d).to(qkv.dtype)
    if dout is None:
        return out
    do = dout.float().view(b, t, h, d).transpose(1, 2).reshape(b * h, t, d)
    ds = torch.bmm(do, v.transpose(1, 2))
    ds.sub_((do * o).sum(2, keepdim=True)).mul_(p)
    dq = torch.bmm(ds, k).mul_(scale)
    dk = torch.bmm(ds.transpose(1, 2), q).mul_(scale)
    dv = torch.bmm(p.transpose(1, 2), do)
    dqkv = torch.stack([dq, dk, dv]).view(3, b, h, t, d).permute(1, 3, 0, 2, 4).reshape(b, t, 3 * h * d)
    return [out, dqkv.to(qkv.dtype)]


# -------------------------------------------------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from pytorch_distributed_amd import ops

        if op == "quantize":
            got = ops.quantize_fp8(state["x"], case["blocks"])
            return [t for m in (got if isinstance(got, tuple) else (got,)) for t in (m.q, m.scale)]
        if op == "product":
            a = ops.Fp8Matrix(state["a_q"], state["a_e"], case["k"])
            b = ops.Fp8Matrix(state["b_q"], state["b_e"], case["k"], tiles=True)
            return ops.fp8_matmul(a, b, bias=state["bias"], out_dtype=DTYPES[case["out"]])
        if op == "linear":
            leaves = [t for t in (state["x"], state["w"], state["bias"]) if t is not None]
            y = ops.fp8_linear(state["x"], state["w"], state["bias"])
            return [y, *torch.autograd.grad(y, leaves, state["dy"])]
        out = ops.window_attention(state["qkv"], case["h"], case["window"], case["sinks"])
        return [out, *torch.autograd.grad(out, [state["qkv"]], state["dout"])] if case["grad"] else out
    with torch.no_grad():
        if op == "quantize":
            return list(_plain_quantize(state["x"], case["blocks"]))
        if op == "product":
            y = _values(state["a_q"], state["a_e"]) @ _values(state["b_q"], state["b_e"], True).t()
            if state["bias"] is not None:
                y = y + state["bias"].float()
            return y.to(DTYPES[case["out"]])
        if op == "linear":
            return _plain_linear(state["x"], state["w"], state["bias"], state["dy"])
        return _plain_window(case, state["qkv"], state["dout"])


# ------------------------------------------------------------------------------------------- definitions in 64 bits
def _exact_blocks(x, tile):
    """x [R, C] in 64 bits -> the e4m3 values and the exponents of 1 x 128 (or 128 x 128) blocks, by search and rounding."""
    r, c = x.shape
    x = _pad(x, BLOCK if tile else 1, BLOCK)
    v = x.view(x.shape[0] // BLOCK, BLOCK, -1, BLOCK) if tile else x.view(x.shape[0], 1, -1, BLOCK)
    amax = v.abs().amax((1, 3), keepdim=True)
    guess = torch.floor(torch.log2(amax.clamp(min=1e-300) / 448.0)) - 1.0
    e = guess
    for _ in range(3):
        e = torch.where(amax > 448.0 * torch.exp2(e), e + 1.0, e)
    e = torch.where(amax > 0, e, torch.full_like(e, -127.0)).clamp(min=-127.0)
    y = v / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)
    y = torch.round(y / step) * step
    return y.reshape(x.shape)[:r], (y * torch.exp2(e)).reshape(x.shape)[:r, :c]


def _exact_values(q, bytes_, rows_per_scale):
    scale = torch.exp2(bytes_.double() - 127.0).repeat_interleave(BLOCK, 1)[:, : q.shape[1]]
    return q.double() * scale.repeat_interleave(rows_per_scale, 0)[: q.shape[0]]


def exact(case, seed):
    state, op = prepare(case, seed), case["op"]
    with torch.no_grad():
        if op == "quantize":
            x, blocks = state["x"].double(), case["blocks"]
            got = []
            if blocks in ("rows", "both"):
                got += [_exact_blocks(x, False)[0], None]
            if blocks in ("columns", "both"):
                got += [_exact_blocks(x.t().contiguous(), False)[0], None]
            if blocks == "tiles":
                got += [_exact_blocks(x, True)[0], None, _exact_blocks(x.t().contiguous(), True)[0], None]
            return got
        if op == "product":
            y = torch.mm(_exact_values(state["a_q"], state["a_e"], 1), _exact_values(state["b_q"], state["b_e"], BLOCK).t())
            return y if state["bias"] is None else y + state["bias"].double()
        if op == "linear":
            x, w, dy = state["x"].double(), state["w"].double(), state["dy"].double()
            wq = _exact_blocks(w, True)[1]
            y = torch.mm(_exact_blocks(x, False)[1], wq.t())
            y = y if state["bias"] is None else y + state["bias"].double()
            dx = torch.mm(_exact_blocks(dy, False)[1], wq)
            dw = torch.mm(_exact_blocks(dy.t().contiguous(), False)[1], _exact_blocks(x.t().contiguous(), False)[1].t())
            return [y, dx, dw] + ([dy.sum(0)] if state["bias"] is not None else [])
        return _exact_window(case, state)


def _exact_window(case, state):
    b, t, h, d = case["b"], case["t"], case["h"], case["d"]
    qkv = state["qkv"].detach().view(b, t, 3, h, d)
    out = torch.empty(b, t, h, d, dtype=torch.float64, device=qkv.device)
    dqkv = torch.empty(b, t, 3, h, d, dtype=torch.float64, device=qkv.device)
    i = torch.arange(t, device=qkv.device)
    age = i.view(-1, 1) - i.view(1, -1)
    seen = (age >= 0) & ((age < case["window"]) | (i.view(1, -1) < case["sinks"]))
    for n in range(b):
        for j in range(h):
            q, k, v = (qkv[n, :, a, j].double().contiguous() for a in range(3))
            logit = (q @ k.t()) / math.sqrt(d)
            p = torch.softmax(torch.where(seen, logit, torch.full_like(logit, -math.inf)), dim=1)
            out[n, :, j] = p @ v
            if case["grad"]:
                g = state["dout"].view(b, t, h, d)[n, :, j].double().contiguous()
                dp = g @ v.t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(d)
                dqkv[n, :, 0, j], dqkv[n, :, 1, j], dqkv[n, :, 2, j] = ds @ k, ds.t() @ q, p.t() @ g
    out = out.view(b, t, h * d)
    return [out, dqkv.view(b, t, 3 * h * d)] if case["grad"] else out
