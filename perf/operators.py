"""The 8-bit inference operators as a user calls them: the residual step's norm with an 8-bit output, the quantizers of
rows and of weights, the block-scaled product and the MLP's first projection with its gate.

An 8-bit tensor is float8_e4m3fn with a power-of-two scale (float8_e8m0fnu) for each block of 128 values along a row
(activations) or of 128 x 128 (weights).  The scale of a block is the smallest 2^e, e in [-126, 120], that brings its
largest magnitude to 448 or less."""

import math

import torch

own = False   # True: the framework's operators; False: their plain form in elementary torch operations

BLOCK = 128
TOP = 448.0   # the largest finite float8_e4m3fn
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    """The served model's own sizes (hidden 1,024, MLP 4,096, vocabulary 50,304; a dense prefill of 32 x 2,048 tokens, a
    decode step of up to 32 sequences) and generic ones around them."""
    return [
        # a decode step of 8 sequences: the attention's output arrives as partial sums with its bias
        dict(name="norm decode 8", op="norm", rows=8, dim=1024, parts=4, dtype="bf16"),
        # ragged prompts of a twice wider model in fp16
        dict(name="norm ragged 2999", op="norm", rows=2999, dim=2048, parts=0, dtype="fp16"),
        # the dense prefill's stream
        dict(name="norm prefill 65536", op="norm", rows=65536, dim=1024, parts=0, dtype="bf16"),
        # activations that no norm produced, a wide layer's input
        dict(name="quantize rows 65536", op="quantize", rows=65536, dim=4096, form="rows", dtype="bf16"),
        # a checkpoint's fp32 matrix as it is loaded
        dict(name="quantize weight 8192", op="quantize", rows=8192, dim=1024, form="weight", dtype="fp32"),
        # one token through the MLP's second projection
        dict(name="linear 1 token", op="linear", rows=1, dim=4096, out=1024, bias=True, dtype="bf16"),
        # the head over a full decode step
        dict(name="linear head 32", op="linear", rows=32, dim=1024, out=50304, bias=True, dtype="bf16"),
        # a prompt's chunk into an odd width
        dict(name="linear ragged 777", op="linear", rows=777, dim=2048, out=1001, bias=False, dtype="fp16"),
        # the dense prefill's second projection
        dict(name="linear prefill 65536", op="linear", rows=65536, dim=4096, out=1024, bias=True, dtype="bf16"),
        # the MLP's first projection in a decode step, over ragged prompts and over the dense prefill
        dict(name="gated decode 16", op="gated", rows=16, dim=1024, out=4096, bias=True, dtype="bf16"),
        dict(name="gated ragged 2999", op="gated", rows=2999, dim=1024, out=4096, bias=True, dtype="bf16"),
        dict(name="gated prefill 65536", op="gated", rows=65536, dim=1024, out=4096, bias=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _of16(n):
    return max(16, n // 16 * 16)


def draw(rng):
    op = rng.choice(["norm", "quantize", "linear", "linear", "gated"])
    rows = _log(rng, 1, 65536)
    if op == "norm":
        parts = rng.choice([0, 0, rng.randint(1, 8)]) if rows <= 256 else 0   # partial sums come from decode steps
        return dict(op=op, rows=rows, dim=_of16(_log(rng, 256, 4096)), parts=parts, dtype=rng.choice(["bf16", "fp16"]))
    if op == "quantize":
        form = rng.choice(["rows", "weight"])
        rows = rows if form == "rows" else _log(rng, 128, 16384)
        return dict(op=op, rows=rows, dim=_of16(_log(rng, 128, 4096)), form=form, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    dim = _of16(_log(rng, 128, 4096))
    if op == "linear":
        out = _log(rng, 64, 16384)
        most = (1 << 38) // (dim * out)
        return dict(op=op, rows=max(1, min(rows, most)), dim=dim, out=out, bias=rng.random() < 0.5,
                    dtype=rng.choice(["bf16", "fp16"]))
    out = 128 * _log(rng, 2, 64)
    most = (1 << 37) // (dim * out)
    return dict(op=op, rows=max(1, min(rows, most)), dim=dim, out=out, bias=rng.random() < 0.5,
                dtype=rng.choice(["bf16", "fp16"]))


def _blocks(n):
    return -(-n // BLOCK)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _activations(g, rows, dim):
    """Rows of different size with a few channels that stand out, as a residual stream has them."""
    gain = 1.0 + 7.0 * (torch.rand(dim, generator=g, device="cuda") < 0.01)
    return _randn(g, rows, dim) * torch.exp(0.5 * _randn(g, rows, 1)) * gain


# ------------------------------------------------------------------------------------------------ the plain form
def _spread(scale, rows, dim):
    """Scales of blocks as one factor a value, fp32; ``rows`` None: scales of rows."""
    s = scale.view(torch.uint8).to(torch.int32)
    s = (s << 23).view(torch.float32)   # 2^(code - 127): codes 1 to 254 are the exponent's bits
    s = s.repeat_interleave(BLOCK, 1)[:, :dim]
    return s if rows is None else s.repeat_interleave(BLOCK, 0)[:rows]


def _codes(amax):
    m, e = torch.frexp(amax)            # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    code = e - 9 + (m > 0.875) + 127
    return torch.where(amax > 0, code, torch.ones_like(code)).clamp(1, 247)


def _padded(x, rows, cols):
    return torch.nn.functional.pad(x, (0, cols - x.shape[1], 0, rows - x.shape[0]))


def _quantize(x, tall):
    """x (rows, dim) fp32 -> (data, scale); blocks of ``tall`` x 128."""
    rows, dim = x.shape
    nr, nc = -(-rows // tall), _blocks(dim)
    t = _padded(x, nr * tall, nc * BLOCK).view(nr, tall, nc, BLOCK)
    code = _codes(t.abs().amax(dim=(1, 3)))
    inv = ((254 - code).to(torch.int32) << 23).view(torch.float32)   # 2^(127 - code)
    q = (t * inv[:, None, :, None]).reshape(nr * tall, nc * BLOCK)[:rows, :dim]
    return q.to(torch.float8_e4m3fn), code.to(torch.uint8).view(torch.float8_e8m0fnu)


def _rows_scale(scale):
    """Scales of rows as the operators hand them out: the rows' pitch a multiple of 4 bytes."""
    rows, n = scale.shape
    held = torch.zeros((rows, -(-n // 4) * 4), dtype=torch.uint8, device=scale.device)
    held[:, :n] = scale.view(torch.uint8)
    return held.view(torch.float8_e8m0fnu)[:, :n]


def _plain_linear(s):
    x = s["x"].to(torch.float32) * _spread(s["x_scale"], None, s["x"].shape[1])
    w = s["w"].to(torch.float32) * _spread(s["w_scale"], s["w"].shape[0], s["w"].shape[1])
    y = x @ w.t()
    return y if s["bias"] is None else y + s["bias"].to(torch.float32)


# ------------------------------------------------------------------------------------------------ what is measured
def prepare(case, seed):
    g = _generator(seed)
    rows, dim, dt = case["rows"], case["dim"], DT[case["dtype"]]
    s = dict(op=case["op"], dtype=dt)
    if case["op"] == "norm":
        s["residual"] = _activations(g, rows, dim).to(dt)
        s["weight"] = (1 + 0.1 * _randn(g, dim)).to(dt)
        n = case["parts"]
        s["branch"] = _randn(g, n, rows, dim) / math.sqrt(n) if n else _randn(g, rows, dim).to(dt)
        s["bias"] = (0.1 * _randn(g, dim)).to(dt) if n else None
    elif case["op"] == "quantize":
        s["form"] = case["form"]
        s["x"] = (_activations(g, rows, dim) if case["form"] == "rows" else 0.02 * _randn(g, rows, dim)).to(dt)
    else:
        out = case["out"] * (2 if case["op"] == "gated" else 1)
        s["x"], scale = _quantize(_activations(g, rows, dim), 1)
        s["x_scale"] = _rows_scale(scale)
        s["w"], s["w_scale"] = _quantize(_randn(g, out, dim) / math.sqrt(dim), BLOCK)
        s["bias"] = (0.1 * _randn(g, out)).to(dt) if case["bias"] else None
    return s


def run(state):
    s = state
    if own:
        from atma_amd.kernel import (linear_fp8, linear_gated_fp8, quantize_fp8, quantize_weight_fp8,
                                     residual_rms_norm_fp8)
        from atma_amd.kernel.decode_fusions import PartialSums
        if s["op"] == "norm":
            branch = s["branch"] if s["bias"] is None else PartialSums(s["branch"], [s["bias"]], dtype=s["dtype"])
            data, scale, stream = residual_rms_norm_fp8(branch, s["residual"], s["weight"], EPS)
            return dict(data=data, scale=scale, stream=stream)
        if s["op"] == "quantize":
            data, scale = quantize_fp8(s["x"]) if s["form"] == "rows" else quantize_weight_fp8(s["x"])
            return dict(data=data, scale=scale)
        if s["op"] == "linear":
            return linear_fp8(s["x"], s["x_scale"], s["w"], s["w_scale"], s["bias"], out_dtype=s["dtype"])
        data, scale = linear_gated_fp8(s["x"], s["x_scale"], s["w"], s["w_scale"], s["bias"])
        return dict(data=data, scale=scale)
    if s["op"] == "norm":
        branch = s["branch"]
        if s["bias"] is not None:
            branch = (branch.sum(0) + s["bias"].to(torch.float32)).to(s["dtype"])
        stream = (s["residual"].to(torch.float32) + branch.to(torch.float32)).to(s["dtype"])
        f = stream.to(torch.float32)
        h = f * torch.rsqrt((f * f).mean(1, keepdim=True) + EPS) * s["weight"].to(torch.float32)
        data, scale = _quantize(h, 1)
        return dict(data=data, scale=scale, stream=stream)
    if s["op"] == "quantize":
        data, scale = _quantize(s["x"].to(torch.float32), 1 if s["form"] == "rows" else BLOCK)
        return dict(data=data, scale=scale)
    y = _plain_linear(s)
    if s["op"] == "linear":
        return y.to(s["dtype"])
    a, gate = y.chunk(2, 1)
    data, scale = _quantize(gate * a.clamp_min(0).square(), 1)
    return dict(data=data, scale=scale)


def work(case):
    rows, dim, size = case["rows"], case["dim"], 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n = case["parts"]
        branch = 4 * n * rows * dim + size * dim if n else size * rows * dim
        held = rows * dim + rows * _blocks(dim)
        return {"bytes": branch + 2 * size * rows * dim + size * dim + held, "flops": (6 + n) * rows * dim}
    if case["op"] == "quantize":
        scales = (rows if case["form"] == "rows" else _blocks(rows)) * _blocks(dim)
        return {"bytes": (size + 1) * rows * dim + scales, "flops": 2 * rows * dim}
    gated = case["op"] == "gated"
    out = case["out"] * (2 if gated else 1)
    read = rows * (dim + _blocks(dim)) + out * dim + _blocks(out) * _blocks(dim) + (size * out if case["bias"] else 0)
    made = rows * (case["out"] + _blocks(case["out"])) if gated else size * rows * out
    return {"bytes": read + made, "flops": 2 * rows * dim * out}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_exponent(a):
    """The smallest e in [-126, 120] with a <= 448 * 2^e, from its definition."""
    e = torch.ceil(torch.log2(a / TOP)).clamp(-126, 120)
    e = torch.where(a > TOP * torch.exp2(e), e + 1, e)
    return torch.where((e > -126) & (a <= TOP * torch.exp2(e - 1)), e - 1, e)


def _exact_quantize(x, tall):
    """What the 8-bit values stand for before their rounding: x / scale; and the scales."""
    rows, dim = x.shape
    row = torch.arange(rows, device=x.device) // tall
    col = torch.arange(dim, device=x.device) // BLOCK
    top = x.new_zeros((rows, _blocks(dim))).scatter_reduce(1, col.expand(rows, dim), x.abs(), "amax")
    if tall > 1:
        top = x.new_zeros((-(-rows // tall), top.shape[1])).index_reduce(0, row, top, "amax")
    scale = torch.exp2(_exact_exponent(top))
    return dict(data=x / scale[row][:, col], scale=scale)


def _exact_values(data, scale, tall):
    row = torch.arange(data.shape[0], device=data.device) // tall
    col = torch.arange(data.shape[1], device=data.device) // BLOCK
    return data.double() * torch.exp2(scale.view(torch.uint8).double() - 127)[row][:, col]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        b = s["branch"].double()
        if s["bias"] is not None:
            b = b.sum(0) + s["bias"].double()
        # the stream is held in its own type, and the norm is that of the held stream
        stream = s["residual"].double() + b.to(s["dtype"]).double()
        f = stream.to(s["dtype"]).double()
        h = f / torch.sqrt(f.square().sum(1, keepdim=True) / f.shape[1] + EPS) * s["weight"].double()
        return dict(_exact_quantize(h, 1), stream=stream)
    if case["op"] == "quantize":
        return _exact_quantize(s["x"].double(), 1 if case["form"] == "rows" else BLOCK)
    y = torch.matmul(_exact_values(s["x"], s["x_scale"], 1), _exact_values(s["w"], s["w_scale"], BLOCK).t().contiguous())
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["op"] == "linear":
        return y
    n = case["out"]
    return _exact_quantize(y[:, n:] * torch.relu(y[:, :n]) ** 2, 1)
