"""What a decode step answers with, as a user calls it: products with 4-bit weights (a projection, the MLP's first projection
with its gate, the head), the weights' quantizer, and the sampler that picks the next tokens from the logits.

A 4-bit weight is a pair: bytes of two float4 e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives; the even k in the
low half) and a power-of-two scale (float8_e8m0fnu) for each 32 values along a row.  The scale of a group is the smallest
2^e, e in [-125, 125], that brings its largest magnitude to 7 or less; values round to nearest even, above 6 to 6.

The sampler divides a row's logits by its temperature (0: the largest logit is the answer) and keeps, in order of falling
value, lower indices first, the first ``top_k`` tokens (0: all), of these the shortest beginning that holds ``top_p`` of
their probability, and of these the tokens that have at least ``min_p`` times the most probable one's probability.  Among
the kept tokens, in index order, the answer is the first whose cumulated probability exceeds ``uniform`` times the kept sum."""

import math

import torch

own = False   # True: the framework's operators; False: their plain form in elementary torch operations

GROUP = 32
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    """The served model's own sizes (hidden 1,024, MLP 4,096, vocabulary 50,304; a dense prefill of 32 x 2,048 tokens, a
    decode step of up to 32 sequences, an engine of up to 2,048) and generic ones around them."""
    return [
        # the head as it is loaded
        dict(name="quantize head 50304", op="quantize", rows=50304, dim=1024, dtype="bf16"),
        # a checkpoint's fp32 matrix
        dict(name="quantize first projection 8192", op="quantize", rows=8192, dim=1024, dtype="fp32"),
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
        dict(name="gated ragged 2999", op="gated", rows=2999, dim=1024, out=4096, bias=True, dtype="fp16"),
        dict(name="gated prefill 65536", op="gated", rows=65536, dim=1024, out=4096, bias=True, dtype="bf16"),
        # one request served in fp32 with a nucleus
        dict(name="sample 1", op="sample", rows=1, vocab=50304, top_k=False, top_p=True, min_p=False, greedy=False,
             dtype="fp32"),
        # a full decode step whose requests ask for different things
        dict(name="sample decode 32", op="sample", rows=32, vocab=50304, top_k=True, top_p=True, min_p=True, greedy=True,
             dtype="bf16"),
        # every request that an engine holds by default, at once
        dict(name="sample 2048", op="sample", rows=2048, vocab=50304, top_k=True, top_p=True, min_p=True, greedy=True,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _of_group(n):
    return max(GROUP, n // GROUP * GROUP)


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "gated", "sample", "sample"])
    if op == "quantize":
        dim = _of_group(_log(rng, 128, 4096))
        return dict(op=op, rows=min(_log(rng, 64, 65536), (1 << 27) // dim), dim=dim, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    if op == "sample":
        vocab = _log(rng, 500, 131072)
        yes = lambda: rng.random() < 0.6   # noqa: E731
        return dict(op=op, rows=max(1, min(_log(rng, 1, 2048), 2048 * 50304 // vocab)), vocab=vocab, top_k=yes(), top_p=yes(),
                    min_p=yes(), greedy=yes(), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    rows, dim = _log(rng, 1, 65536), _of_group(_log(rng, 128, 4096))
    out = _log(rng, 64, 16384) if op == "linear" else _log(rng, 128, 8192)
    most = (1 << 38 if op == "linear" else 1 << 37) // (dim * out)
    return dict(op=op, rows=max(1, min(rows, most)), dim=dim, out=out, bias=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16"]))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _activations(g, rows, dim):
    """Normed rows with a few channels that stand out."""
    return _randn(g, rows, dim) * (1.0 + 7.0 * (_rand(g, dim) < 0.01))


# ------------------------------------------------------------------------------------------------ the plain form
def _quantize(w):
    """w (rows, dim) fp32 -> the e2m1 values (rows, dim) fp32 before their scale, and the scales' codes (rows, dim / 32)."""
    t = w.view(w.shape[0], -1, GROUP)
    top = t.abs().amax(2)
    m, e = torch.frexp(top)              # top = m 2^e, m in [0.5, 1); 7 = 0.875 * 2^3
    e = torch.where(top > 0, e - 3 + (m > 0.875), torch.full_like(e, -125)).clamp(-125, 125)
    v = torch.ldexp(t, -e[:, :, None])
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = ((a / step).round() * step).clamp_max(6)
    return torch.copysign(a, v).view(w.shape), (e + 127).to(torch.uint8)


def _packed(v):
    """e2m1 values as bytes: the sign, and the position among 0, 0.5, 1, 1.5, 2, 3, 4, 6."""
    a = v.abs()
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) + 8 * torch.signbit(v).to(torch.uint8)
    return code[:, ::2] + 16 * code[:, 1::2]


def _values(data, scale):
    code = torch.stack((data % 16, data // 16), 2).flatten(1).to(torch.int32)
    a = (code % 8).to(torch.float32)
    a = torch.where(a < 4, a / 2, torch.where(a < 6, a - 2, 2 * a - 8))
    v = torch.where(code < 8, a, -a)
    s = (scale.view(torch.uint8).to(torch.int32) << 23).view(torch.float32)   # 2^(code - 127)
    return v * s.repeat_interleave(GROUP, 1)


def _plain_linear(s):
    y = s["x"].to(torch.float32) @ _values(s["w"], s["w_scale"]).t()
    return y if s["bias"] is None else y + s["bias"].to(torch.float32)


def _plain_sample(s):
    """In 64 bits: which token a cumulated probability reaches lies next to a border."""
    value, index = torch.sort(s["logits"].to(torch.float64), dim=1, descending=True, stable=True)
    t = s["temperature"].to(torch.float64)[:, None]
    w = ((value - value[:, :1]) / torch.where(t > 0, t, 1.0)).exp()
    rank = torch.arange(w.shape[1], device=w.device)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        w = torch.where((k <= 0) | (rank < k), w, 0.0)
    held = w
    if s["top_p"] is not None:
        p = s["top_p"].to(torch.float64)[:, None]
        total = w.cumsum(1)
        before = torch.nn.functional.pad(total[:, :-1], (1, 0))
        held = torch.where((p >= 1) | (before < p * total[:, -1:]), held, 0.0)
    if s["min_p"] is not None:
        held = torch.where(w >= s["min_p"].to(torch.float64)[:, None], held, 0.0)
    total = torch.zeros_like(held).scatter_(1, index, held).cumsum(1)
    found = (total <= s["uniform"].to(torch.float64)[:, None] * total[:, -1:]).sum(1)
    return torch.where(s["temperature"] > 0, found, index[:, 0])


# ------------------------------------------------------------------------------------------------ what is measured
def prepare(case, seed):
    g = _generator(seed)
    rows, dt = case["rows"], DT[case["dtype"]]
    s = dict(op=case["op"])
    if case["op"] == "quantize":
        s["w"] = (0.02 * _randn(g, rows, case["dim"]) * torch.exp(0.3 * _randn(g, rows, 1))).to(dt)
    elif case["op"] == "sample":
        z = 3.0 * _randn(g, rows, case["vocab"]) * torch.exp(0.4 * _randn(g, rows, 1)) - 2.0
        z = z + (_rand(g, rows, case["vocab"]) < 8 / case["vocab"]) * (4.0 + 8.0 * _rand(g, rows, 1))   # a few likely tokens
        s["logits"] = (15.0 * z * torch.rsqrt(z * z + 225.0)).to(dt)   # the model's soft cap
        s["uniform"] = _rand(g, rows)
        t = 0.5 + _rand(g, rows)
        s["temperature"] = torch.where(_rand(g, rows) < 0.2, 0.0, t) if case["greedy"] else t
        off = lambda: _rand(g, rows) < 0.3   # noqa: E731  (requests that leave a filter out)
        k = torch.exp(math.log(200) * _rand(g, rows)).to(torch.int32)
        s["top_k"] = torch.where(off(), 0, k) if case["top_k"] else None
        s["top_p"] = torch.where(off(), 1.0, 0.7 + 0.29 * _rand(g, rows)) if case["top_p"] else None
        s["min_p"] = torch.where(off(), 0.0, 0.2 * _rand(g, rows)) if case["min_p"] else None
    else:
        dim, out = case["dim"], case["out"] * (2 if case["op"] == "gated" else 1)
        s["x"] = _activations(g, rows, dim).to(dt)
        values, scale = _quantize(_randn(g, out, dim) / math.sqrt(dim))
        s["w"], s["w_scale"] = _packed(values), scale.view(torch.float8_e8m0fnu)
        s["bias"] = (0.1 * _randn(g, out)).to(dt) if case["bias"] else None
    return s


def run(state):
    s = state
    if own:
        from atma_amd.kernel import (dequantize_weight_fp4, linear_fp4, linear_gated_fp4, quantize_weight_fp4,
                                     sample_tokens)
        if s["op"] == "quantize":
            data, scale = quantize_weight_fp4(s["w"])
            return dict(values=dequantize_weight_fp4(data, scale, s["w"].dtype), scale=scale)
        if s["op"] == "linear":
            return linear_fp4(s["x"], s["w"], s["w_scale"], s["bias"])
        if s["op"] == "gated":
            return linear_gated_fp4(s["x"], s["w"], s["w_scale"], s["bias"])
        return sample_tokens(s["logits"], s["uniform"], s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                             min_p=s["min_p"])
    if s["op"] == "quantize":
        values, scale = _quantize(s["w"].to(torch.float32))
        scale = scale.view(torch.float8_e8m0fnu)
        return dict(values=_values(_packed(values), scale).to(s["w"].dtype), scale=scale)
    if s["op"] == "sample":
        return _plain_sample(s)
    y = _plain_linear(s)
    if s["op"] == "gated":
        a, gate = y.chunk(2, 1)
        y = gate * a.clamp_min(0).square()
    return y.to(s["x"].dtype)


def work(case):
    rows, size = case["rows"], 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "sample":
        params = 8 + sum(4 * case[name] for name in ("top_k", "top_p", "min_p"))
        return {"bytes": rows * (size * case["vocab"] + params + 8), "flops": 4 * rows * case["vocab"]}
    dim = case["dim"]
    if case["op"] == "quantize":
        return {"bytes": 2 * size * rows * dim + rows * dim // GROUP, "flops": 4 * rows * dim}
    out = case["out"] * (2 if case["op"] == "gated" else 1)
    read = size * rows * dim + out * dim // 2 + out * dim // GROUP + (size * out if case["bias"] else 0)
    return {"bytes": read + size * rows * case["out"], "flops": 2 * rows * dim * out}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_weight(data, scale):
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=data.device)
    grid = torch.cat((grid, -grid))
    v = grid[torch.stack((data & 15, data >> 4), 2).long()].flatten(1)
    col = torch.arange(v.shape[1], device=v.device) // GROUP
    return v * torch.exp2(scale.view(torch.uint8).double() - 127)[:, col]


def exact(case, seed):
    if case["op"] == "sample":
        return None   # whole numbers, which the plain form finds in 64 bits
    s = prepare(case, seed)
    if case["op"] == "quantize":
        w = s["w"].double()
        top = w.abs().view(w.shape[0], -1, GROUP).max(2).values
        e = torch.ceil(torch.log2(top / 7)).clamp(-125, 125)
        e = torch.where(top > 7 * torch.exp2(e), e + 1, e)
        e = torch.where((e > -125) & (top <= 7 * torch.exp2(e - 1)), e - 1, e)
        scale = torch.exp2(e)
        spread = scale[:, torch.arange(w.shape[1], device=w.device) // GROUP]
        a = w.abs() / spread
        # between neighbours half way goes to the one with the even last bit: 0, 1, 2 and 4
        v = 0.5 * ((a > 0.25).double() + (a >= 0.75).double() + (a > 1.25).double() + (a >= 1.75).double())
        v = v + (a > 2.5).double() + (a >= 3.5).double() + 2 * (a > 5).double()
        return dict(values=torch.sign(w) * v * spread, scale=scale)
    y = torch.matmul(s["x"].double(), _exact_weight(s["w"], s["w_scale"]).t().contiguous())
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["op"] == "gated":
        n = case["out"]
        y = y[:, n:] * torch.relu(y[:, :n]) ** 2
    return y
