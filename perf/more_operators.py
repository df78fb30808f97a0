"""Timed cases of what stands in front of the attention: the residual's addition and root-mean-square
norm of the hidden rows, their 8-bit codes, the 8-bit projection with its gradients, and the rotation
of Q and K by positions of several axes.

An 8-bit matrix is codes float8_e4m3fn [rows, width rounded up to 16, zeros behind the width] with one
scale byte b, 2^(b - 127), for 128 values of a row, scales uint8 [rows, blocks], or for 128 x 128
values, [row blocks, blocks]; the exponent is the smallest one with which the group's largest magnitude
is at most 448.

`own` False computes each operator from elementary torch operations in 32 bits; True calls the
library."""

import math

import torch

own = False

BLOCK = 128
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPSILON = 1e-6


def listed():
    return [
        # the hidden row of one new token on its way to a projection: the latency of one call
        dict(name="norm one token, 8 bits", op="norm", rows=1, width=5120, dtype="bf16", stream="bf16", fp8=True),
        # all tokens of the Wan-shaped layer (21 frames of 30 x 52 patches, 40 heads of 128)
        dict(name="norm video, 8 bits", op="norm", rows=32760, width=5120, dtype="bf16", stream="bf16", fp8=True),
        # a training step's norm on a residual stream in 32 bits, backward, an odd number of rows
        dict(name="norm backward", op="norm_backward", rows=8191, width=2560, dtype="bf16", stream="fp32"),
        # one token's Q, K and V of that layer: the weights are read once
        dict(name="project one token", op="project", rows=1, width=5120, outs=15360, dtype="bf16", bias=False),
        # a prompt's rows, sizes that end inside a block and a tile, fp16 with a bias
        dict(name="project prompt", op="project", rows=333, width=4112, outs=5000, dtype="fp16", bias=True),
        # one projection of the Wan-shaped layer
        dict(name="project video", op="project", rows=32760, width=5120, outs=5120, dtype="bf16", bias=True),
        # both gradients of a projection, from rows in 16 bits
        dict(name="projection gradients", op="gradients", rows=4095, width=2560, outs=2560, dtype="bf16"),
        # a text encoder's rows on their way to K and V
        dict(name="quantise prompt", op="quantise", rows=512, width=4096, dtype="fp16", square=False, transpose=False),
        # a feed-forward weight, laid out for the gradient of its input
        dict(name="quantise weight", op="quantise", rows=13824, width=5120, dtype="bf16", square=True, transpose=True),
        # the next token of a sequence, grouped heads
        dict(name="rotate one token", op="rope", batch=1, tokens=1, heads=40, kv_heads=8, dim=128, rotated=128,
             axes=3, pairs="halves", dtype="bf16", whole=True, backward=False),
        # Q and K of the Wan-shaped layer, as the projection leaves them
        dict(name="rotate video", op="rope", batch=1, tokens=32760, heads=40, kv_heads=40, dim=128, rotated=128,
             axes=3, pairs="interleaved", dtype="bf16", whole=True, backward=False),
        # gradients of image tokens at fractional places, two axes, a head dim that is no power of two
        dict(name="rotate images, backward", op="rope", batch=3, tokens=2311, heads=16, kv_heads=16, dim=80,
             rotated=64, axes=2, pairs="halves", dtype="fp32", whole=False, backward=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_backward", "project", "project", "project", "gradients", "quantise", "rope",
                     "rope", "rope"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("norm", "norm_backward"):
        while True:
            rows, width = _log_int(rng, 1, 130000), rng.choice([64, 128, 512, 5120, _log_int(rng, 16, 16000)])
            if rows * width <= 1.6e8:
                break
        stream = rng.choice([dtype, dtype, "fp32"])
        if op == "norm_backward":
            return dict(op=op, rows=rows, width=width, dtype=dtype, stream=stream)
        return dict(op=op, rows=rows, width=width, dtype=dtype, stream=stream, fp8=rng.random() < 0.6)
    if op in ("project", "gradients"):
        while True:
            rows = _log_int(rng, 1 if op == "project" else 100, 33000)
            width, outs = (rng.choice([64, 128]) * _log_int(rng, 1, 100) if rng.random() < 0.5 else
                           _log_int(rng, 30, 14000) for _ in range(2))
            if rows * width * outs * (1 if op == "project" else 4) <= 8.5e11 and width * outs <= 1.0e8:
                break
        case = dict(op=op, rows=rows, width=width, outs=outs, dtype=dtype)
        return case if op == "gradients" else dict(case, bias=rng.random() < 0.5)
    if op == "quantise":
        while True:
            rows, width = _log_int(rng, 1, 60000), _log_int(rng, 16, 16000)
            if rows * width <= 7e7:
                break
        return dict(op=op, rows=rows, width=width, dtype=dtype, square=rng.random() < 0.5,
                    transpose=rng.random() < 0.5)
    while True:
        batch, tokens = _log_int(rng, 1, 8), rng.choice([1, _log_int(rng, 1, 120000)])
        kv_heads = rng.choice([1, 2, 4, 8, 12, 24, 40])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        if heads <= 64 and batch * tokens * (heads + kv_heads) * dim <= 3.3e8:
            break
    return dict(op=op, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                rotated=rng.choice([dim, dim, dim // 2]), axes=rng.choice([1, 2, 3, 3, 3]),
                pairs=rng.choice(["interleaved", "halves"]), dtype=dtype, whole=rng.random() < 0.6,
                backward=rng.random() < 0.4)


# ------------------------------------------------------------------ 8-bit matrices, plain


def _pad(x, width):
    return torch.nn.functional.pad(x, (0, width - x.shape[-1]))


def _groups(x, square):
    """x [rows, width] in 32 bits -> [rows or row blocks, 128 or 1, blocks, 128], zeros behind the edges."""
    rows, width = x.shape
    wide = -(-width // BLOCK) * BLOCK
    if square:
        tall = -(-rows // BLOCK) * BLOCK
        return torch.nn.functional.pad(x, (0, wide - width, 0, tall - rows)).view(tall // BLOCK, BLOCK, -1, BLOCK)
    return _pad(x, wide).view(rows, 1, -1, BLOCK)


def _quantise(x, square=False):
    rows, width = x.shape
    g = _groups(x.float(), square)
    top = g.abs().amax((1, 3), keepdim=True).contiguous()
    byte = (((top.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp(1, 254)
    codes = (g * torch.exp2((127 - byte).float())).flatten(2).flatten(0, 1)[:rows, : -(-width // 16) * 16]
    return codes.to(torch.float8_e4m3fn), byte.view(g.shape[0], g.shape[2]).to(torch.uint8)


def _values(codes, scales):
    """The 32-bit values that an 8-bit matrix stands for."""
    rows, width = codes.shape
    s = torch.exp2(scales.float() - 127)
    if scales.shape[0] != rows:
        s = s.repeat_interleave(BLOCK, 0)[:rows]
    return codes.float() * s.repeat_interleave(BLOCK, 1)[:, :width]


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _hidden(gen, rows, width, dtype, tail=0.7):
    """Rows as a model has them: channels of unlike size, rows of unlike size."""
    by_channel = torch.exp(tail * torch.randn(width, generator=gen, device="cuda"))
    by_row = torch.exp(0.3 * torch.randn((rows, 1), generator=gen, device="cuda"))
    return (torch.randn((rows, width), generator=gen, device="cuda") * by_channel * by_row).to(dtype)


def _positions(case, gen):
    """Places of a video (time, height, width), of images or of text: whole numbers behind those of
    earlier tokens, or fractions where a rate or a size is scaled."""
    b, s, axes = case["batch"], case["tokens"], case["axes"]
    at = torch.arange(s, device="cuda")
    side = max(1, int(math.sqrt(min(s, 52 * 30))))
    grid = torch.stack([at // (side * side), at // side % side, at % side][3 - axes:], -1)
    first = torch.randint(0, 100000, (b, 1, axes), generator=gen, device="cuda")
    if case["whole"]:
        return (grid + first).int()
    return (grid * (0.25 + torch.rand((b, 1, axes), generator=gen, device="cuda"))).float()


def _axis_dims(case):
    """The rotated dims of each axis: even parts, what is left over with the first."""
    part = case["rotated"] // case["axes"] // 2 * 2
    return [case["rotated"] - part * (case["axes"] - 1)] + [part] * (case["axes"] - 1)


def prepare(case, seed):
    op, gen, dtype = case["op"], _gen(seed), TYPES[case["dtype"]]
    state = dict(case=case)
    if op == "norm":
        rows, width = case["rows"], case["width"]
        weight = 1 + 0.2 * torch.randn(width, generator=gen, device="cuda")
        return state | dict(x=_hidden(gen, rows, width, dtype), residual=_hidden(gen, rows, width, TYPES[case["stream"]]),
                            weight=weight.to(dtype))
    if op == "norm_backward":
        rows, width, stream = case["rows"], case["width"], TYPES[case["stream"]]
        weight = 1 + 0.2 * torch.randn(width, generator=gen, device="cuda")
        return state | dict(dy=_hidden(gen, rows, width, dtype, 0.2), s=_hidden(gen, rows, width, stream),
                            dsum=_hidden(gen, rows, width, stream, 0.2), weight=weight)
    if op in ("project", "gradients"):
        rows, width, outs = case["rows"], case["width"], case["outs"]
        x = _hidden(gen, rows, width, dtype)
        w = (torch.randn((outs, width), generator=gen, device="cuda") / math.sqrt(width)).to(torch.bfloat16)
        if op == "project":
            bias = torch.randn(outs, generator=gen, device="cuda").to(dtype) if case["bias"] else None
            return state | dict(a=_quantise(x), b=_quantise(w, square=True), bias=bias)
        # a training program keeps the weight transposed for the gradient of its input
        return state | dict(x=x, dy=_hidden(gen, rows, outs, dtype, 0.2), wt=_quantise(w.t().contiguous(), square=True))
    if op == "quantise":
        return state | dict(x=_hidden(gen, case["rows"], case["width"], dtype))
    b, s, d = case["batch"], case["tokens"], case["dim"]
    # [B, S, H, D], as a projection leaves them, seen as [B, H, S, D]
    q, k = (torch.randn((b, s, h, d), generator=gen, device="cuda").to(dtype).transpose(1, 2)
            for h in (case["heads"], case["kv_heads"]))
    dims = _axis_dims(case)
    freqs = torch.cat([10000.0 ** (-torch.arange(0, n, 2, dtype=torch.float64) / n) for n in dims if n])
    axis = torch.cat([torch.full((n // 2,), i, dtype=torch.int32) for i, n in enumerate(dims)])
    return state | dict(q=q, k=k, positions=_positions(case, gen), freqs=freqs.cuda(), axis=axis.cuda())


# ------------------------------------------------------------------ the operators, plain


def _norm(state):
    x, residual, case = state["x"], state["residual"], state["case"]
    s = (x.float() + residual.float()).to(residual.dtype)
    f = s.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPSILON) * state["weight"].float()
    if case["fp8"]:
        return _values(*_quantise(y)).to(torch.bfloat16), s
    return y.to(x.dtype), s


def _norm_backward(state):
    dy, s = state["dy"].float(), state["s"].float()
    r = torch.rsqrt(s.square().mean(-1, keepdim=True) + EPSILON)
    g = dy * state["weight"]
    dx = r * (g - s * (r * r * (g * s).mean(-1, keepdim=True))) + state["dsum"].float()
    return dx.to(state["s"].dtype), (dy * s * r).sum(0)


def _project(state):
    y = _values(*state["a"]) @ _values(*state["b"]).t()
    if state["bias"] is not None:
        y += state["bias"].float()
    return y.to(TYPES[state["case"]["dtype"]])


def _gradients(state):
    dy, x, dtype = state["dy"], state["x"], TYPES[state["case"]["dtype"]]
    dx = _values(*_quantise(dy)) @ _values(*state["wt"]).t()
    dw = _values(*_quantise(dy.t())) @ _values(*_quantise(x.t())).t()
    return dx.to(dtype), dw


def _rotate(state):
    case = state["case"]
    positions, half = state["positions"].double(), case["rotated"] // 2
    angle = positions[..., state["axis"].long()] * state["freqs"]  # [B, S, R / 2]
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if case["backward"]:
        s = -s
    got = []
    for x in (state["q"], state["k"]):
        y = x.float().contiguous()
        turned = y[..., : case["rotated"]]
        if case["pairs"] == "interleaved":
            a, b = turned.unflatten(-1, (half, 2)).unbind(-1)
            turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
        else:
            a, b = turned[..., :half], turned[..., half:]
            turned = torch.cat([a * c - b * s, b * c + a * s], -1)
        got.append(torch.cat([turned, y[..., case["rotated"]:]], -1).to(x.dtype))
    return got


def run(state):
    case = state["case"]
    op = case["op"]
    if op == "norm":
        if own:
            from sparsepr_amd.kernels.fp8 import fp8_dequantize
            from sparsepr_amd.kernels.rms_norm import rms_norm, rms_norm_fp8

            x, weight, residual = state["x"], state["weight"], state["residual"]
            if case["fp8"]:
                codes, scales, s = rms_norm_fp8(x, weight, residual=residual, epsilon=EPSILON)
                return fp8_dequantize(codes, scales, dtype=torch.bfloat16), s
            return rms_norm(x, weight, residual=residual, epsilon=EPSILON)
        return _norm(state)
    if op == "norm_backward":
        if own:
            from sparsepr_amd.kernels.rms_norm import rms_norm_backward

            return rms_norm_backward(state["dy"], state["s"], state["weight"], dsum=state["dsum"], epsilon=EPSILON)
        return _norm_backward(state)
    if op == "project":
        if own:
            from sparsepr_amd.kernels.fp8 import fp8_matmul

            return fp8_matmul(*state["a"], *state["b"], bias=state["bias"], out_dtype=TYPES[case["dtype"]])
        return _project(state)
    if op == "gradients":
        if own:
            from sparsepr_amd.kernels.fp8 import fp8_matmul, fp8_quantize

            dy, dtype = state["dy"], TYPES[case["dtype"]]
            dx = fp8_matmul(*fp8_quantize(dy), *state["wt"], out_dtype=dtype)
            dw = fp8_matmul(*fp8_quantize(dy, transpose=True), *fp8_quantize(state["x"], transpose=True),
                            out_dtype=torch.float32)
            return dx, dw
        return _gradients(state)
    if op == "quantise":
        if own:
            from sparsepr_amd.kernels.fp8 import fp8_dequantize, fp8_quantize

            codes, scales = fp8_quantize(state["x"], square=case["square"], transpose=case["transpose"])
            return fp8_dequantize(codes, scales, dtype=torch.bfloat16)
        x = state["x"].t() if case["transpose"] else state["x"]
        return _values(*_quantise(x, case["square"])).to(torch.bfloat16)
    if own:
        from sparsepr_amd.kernels.axial_rope import axial_rope

        return axial_rope(state["q"], state["k"], state["positions"], state["freqs"], state["axis"],
                          pairs=case["pairs"], inverse=case["backward"])
    return _rotate(state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    op, wide = case["op"], TYPES[case["dtype"]].itemsize
    if op in ("norm", "norm_backward"):
        n, stream = case["rows"] * case["width"], TYPES[case["stream"]].itemsize
        out = wide if op == "norm_backward" or not case["fp8"] else 2
        per = wide + 2 * stream + out if op == "norm" else wide + 3 * stream
        return {"bytes": n * per + 4 * case["width"], "flops": 0}
    if op == "project":
        m, k, n = case["rows"], case["width"], case["outs"]
        return {"bytes": (m + n) * k + m * n * wide, "flops": 2 * m * n * k}
    if op == "gradients":
        m, k, n = case["rows"], case["width"], case["outs"]
        return {"bytes": wide * (m * n + 2 * m * k) + n * k * 5, "flops": 4 * m * n * k}
    if op == "quantise":
        return {"bytes": case["rows"] * case["width"] * (wide + 2), "flops": 0}
    rows = case["batch"] * case["tokens"]
    return {"bytes": rows * ((case["heads"] + case["kv_heads"]) * case["dim"] * 2 * wide + 4 * case["axes"]), "flops": 0}


# ------------------------------------------------------------------ the same from the definitions, in 64 bits


def _exact_e4m3(v):
    """The nearest 4-bit-significand float of each value, ties to the even one: steps of 2^(e - 3), 2^-9 at least."""
    _, e = torch.frexp(v)
    step = torch.exp2(((e - 1).clamp(min=-6) - 3).double())
    return torch.round(v / step) * step


def _exact_quantised(x, square):
    """The values of x [rows, width] after rounding to 8 bits, in 64 bits, group by group."""
    rows, width = x.shape
    tall, wide = -(-rows // BLOCK) * BLOCK if square else rows, -(-width // BLOCK) * BLOCK
    full = torch.zeros((tall, wide), dtype=torch.float64, device=x.device)
    full[:rows, :width] = x
    g = full.reshape(tall // BLOCK, BLOCK, wide // BLOCK, BLOCK) if square else full.reshape(rows, 1, wide // BLOCK, BLOCK)
    part, e = torch.frexp(g.abs().amax((1, 3), keepdim=True))  # part in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(part == 0, -126, (e - 9 + (part > 0.875).to(e.dtype)).clamp(min=-126))
    scale = torch.exp2(e.double())
    return (_exact_e4m3(g / scale) * scale).reshape(tall, wide)[:rows, : -(-width // 16) * 16]


def _exact_values(codes, scales):
    """codes as bits: sign, four of exponent, three of fraction; scales by index."""
    bits = codes.view(torch.uint8).long()
    e, f = bits // 8 % 16, (bits % 8).double()
    v = torch.where(e == 0, f * 2.0 ** -9, (8 + f) * torch.exp2((e - 10).double()))
    v = torch.where(bits >= 128, -v, v)
    rows, width = codes.shape
    at = torch.arange(rows, device=codes.device)
    at = at if scales.shape[0] == rows else at // BLOCK
    return v * torch.exp2(scales.double() - 127)[at][:, torch.arange(width, device=codes.device) // BLOCK]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        s = (state["x"].double() + state["residual"].double())
        kept = s.to(state["residual"].dtype).double()
        y = kept / torch.sqrt((kept * kept).sum(-1, keepdim=True) / case["width"] + EPSILON) * state["weight"].double()
        return (_exact_quantised(y, False) if case["fp8"] else y), s
    if op == "norm_backward":
        dy, s, w = state["dy"].double(), state["s"].double(), state["weight"].double()
        n = case["width"]
        power = (s * s).sum(-1, keepdim=True) / n + EPSILON
        along = (dy * w * s).sum(-1, keepdim=True) / n
        dx = dy * w / power.sqrt() - s * along / power ** 1.5 + state["dsum"].double()
        return dx, (dy * s / power.sqrt()).sum(0)
    if op == "project":
        a, b = _exact_values(*state["a"]), _exact_values(*state["b"])
        y = torch.cat([rows @ b.T for rows in a.split(4096)])
        return y if state["bias"] is None else y + state["bias"].double()
    if op == "gradients":
        dy, x = state["dy"].double(), state["x"].double()
        dx = _exact_quantised(dy, False) @ _exact_values(*state["wt"]).T
        dw = _exact_quantised(dy.T, False) @ _exact_quantised(x.T, False).T
        return dx, dw
    if op == "quantise":
        x = state["x"].double()
        return _exact_quantised(x.T if case["transpose"] else x, case["square"])
    half, got = case["rotated"] // 2, []
    angle = state["positions"].double()[:, None, :, :].index_select(-1, state["axis"].long()) * state["freqs"]
    turn = torch.polar(torch.ones_like(angle), -angle if case["backward"] else angle)
    for x in (state["q"], state["k"]):
        y = x.double().clone(memory_format=torch.contiguous_format)
        i = torch.arange(half, device=y.device)
        first, second = (2 * i, 2 * i + 1) if case["pairs"] == "interleaved" else (i, i + half)
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        got.append(y)
    return got
