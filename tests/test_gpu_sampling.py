"""The sampler on the GPU against the oracle, one row at a time in float64: the ids are equal.

A row whose answer the oracle itself does not know for certain is left out: one where a filter's or the draw's border lies within
1e-9 of the sum that it cuts (both sides round in 64 bits, 2^-52 a term, and the kernel holds weights to 2^-44: together below
V 2^-43, 1e-8 for 2^16 terms of one sign, 1e-10 as they fall).  Such rows are counted and few."""

import math

import pytest
import torch

from oracle import sampling as O

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _certain(x, u, t, k, p, m):
    """Whether no border of the oracle's lies within 1e-9 of what it is compared with."""
    if not t > 0 or any(v != v for v in x):
        return True
    full = O.kept(x, t, k)
    total = math.fsum(full.values())
    if p < 1:
        c = 0.0
        for v in full.values():
            if c and abs(c - p * total) < 1e-9 * total:
                return False
            c += v
    if 0 < m < 1 and any(v != 1.0 and abs(v - m) < 1e-9 * m for v in full.values()):
        return False
    w = O.kept(x, t, k, p, m)
    total, c, u = math.fsum(w.values()), 0.0, min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    for i in sorted(w):
        c += w[i]
        if w[i] and abs(c - u * total) < 1e-9 * total:   # (a token of no weight moves no border)
            return False
    return True


def _check(dev, logits, u, t, k=None, p=None, m=None, doubtful=0, **scalars):
    from atma_amd.kernel import sample_tokens
    rows = logits.shape[0]
    held = [None if v is None else torch.tensor(v, dtype=d).to(dev) for v, d in
            ((t, F32), (k, torch.int32), (p, F32), (m, F32))]
    ids = sample_tokens(logits.to(dev), torch.tensor(u, dtype=F32).to(dev), 1.0 if t is None else held[0], top_k=held[1],
                        top_p=held[2], min_p=held[3])
    assert ids.shape == (rows,) and ids.dtype == torch.int64
    f32 = lambda v: torch.tensor(v, dtype=F32).tolist()   # noqa: E731
    u, t = f32(u), f32(t) if t is not None else [1.0] * rows
    k, p, m = k or [0] * rows, f32(p) if p else [1.0] * rows, f32(m) if m else [0.0] * rows
    left = 0
    for r, (x, got) in enumerate(zip(logits.double().tolist(), ids.tolist())):
        args = (x, u[r], t[r], k[r], p[r], m[r])
        if not _certain(*args):
            left += 1
            continue
        assert got == O.draw(*args), (r, u[r], t[r], k[r], p[r], m[r])
    assert left <= doubtful, left
    return ids


def _logits(g, rows, V, spread=3.0):
    return spread * torch.randn(rows, V, generator=g)


@pytest.mark.parametrize("V", [1, 2, 7, 8, 63, 500, 511, 512, 513, 2047, 4097, 8193, 50304, 65535, 65536])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_all_filters(dev, V, dtype):
    g = torch.Generator().manual_seed(V)
    rows = 24 if V < 10000 else 10 if V < 60000 else 4
    rnd = lambda: torch.rand(rows, generator=g)   # noqa: E731
    logits = _logits(g, rows, V).to(dtype)
    u, t = rnd().tolist(), (0.3 + 1.2 * rnd()).tolist()
    t[1] = 0.0
    k = [0 if r % 3 == 0 else int(1 + v * min(V, 300)) for r, v in enumerate(rnd().tolist())]
    p = [1.0 if r % 4 == 1 else 0.2 + 0.79 * v for r, v in enumerate(rnd().tolist())]
    m = [0.0 if r % 2 else 0.3 * v for r, v in enumerate(rnd().tolist())]
    for sel in ((None, None, None), (k, None, None), (None, p, None), (None, None, m), (k, p, None), (k, p, m)):
        _check(dev, logits, u, t, *sel, doubtful=1)


@pytest.mark.parametrize("V", [3000, 20000, 70000])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_many_equal_logits(dev, dtype, V):
    """Borders inside runs of equal logits: the lowest indices are kept."""
    g = torch.Generator().manual_seed(1)
    rows = 16 if V < 50000 else 4
    logits = torch.randint(-3, 3, (rows, V), generator=g).to(dtype)
    logits[3] = 1.5
    u = [(r + 0.5) / rows for r in range(rows)]
    k = [1 + 37 * r for r in range(rows)]
    _check(dev, logits, u, [1.0] * rows, k, doubtful=1)
    p = [(r + 0.37) / rows for r in range(rows)]
    _check(dev, logits, u, [0.8] * rows, None, p, doubtful=1)
    _check(dev, logits, u, [0.8] * rows, k, p, doubtful=1)


@pytest.mark.parametrize("V", [2000, 30000])
def test_logits_close_together_and_far_apart(dev, V):
    """Ranges of logits from far below a temperature to far above it, and rows of which a few tokens have all the weight."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn(12, V, generator=g) * torch.tensor([1e-6, 1e-4, 1e-2, 0.1, 1.0, 10.0, 100.0, 1e4, 1e20, 3.0, 3.0, 3.0])[:, None]
    x[9, 10:] = -math.inf
    x[10, 5:] -= 200
    x[11, 2000 // 2:] = x[11, 0]
    u = [(r + 0.4) / 12 for r in range(12)]
    for k, p in ((None, None), ([40] * 12, None), (None, [0.9] * 12), ([300] * 12, [0.8] * 12)):
        _check(dev, x, u, [1.0] * 12, k, p, doubtful=1)
        _check(dev, x.to(BF), u, [1.0] * 12, k, p, doubtful=1)
        _check(dev, x.to(HF), u, [0.7] * 12, k, p, doubtful=1)
        _check(dev, x.to(HF), u, [0.7] * 12, k, p, [0.05] * 12, doubtful=1)
        _check(dev, x.to(BF), u, [1e-4, 1e-3, 1e3, 1e-2, 30.0, 1e20, 0.7, 1e-2, 3.0, 1e6, 0.1, 50.0], k, p, doubtful=1)


@pytest.mark.parametrize("V", [3000, 5000, 16384, 16385, 50304, 70001])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_many_rows_and_few_agree(dev, V, dtype):
    """The kernels for many rows and for few, and any number of rows a call, answer the same."""
    from atma_amd.kernel import sample_tokens
    g = torch.Generator().manual_seed(9)
    rows = 600 if V < 20000 else 300
    x = _logits(g, rows, V).to(dtype).to(dev)
    u, t = torch.rand(rows, generator=g).to(dev), (torch.rand(rows, generator=g) * 1.5).to(dev)
    k = torch.randint(0, 400, (rows,), generator=g, dtype=torch.int32).to(dev)
    p, m = (0.5 + torch.rand(rows, generator=g)).to(dev), (0.2 * torch.rand(rows, generator=g) - 0.1).to(dev)
    t[3], k[4:8], x[9, 5] = 0, 0, float("nan")
    for sel in ((None, None, None), (k, None, None), (None, p, None), (k, p, m)):
        want = sample_tokens(x, u, t, *sel)
        cut = lambda v, a, b: None if v is None else v[a:b]   # noqa: E731
        got = torch.cat([sample_tokens(x[a:a + 50], u[a:a + 50], t[a:a + 50], *(cut(v, a, a + 50) for v in sel))
                         for a in range(0, rows, 50)])
        assert torch.equal(got, want)


def test_exact_borders(dev):
    """Equal weights: sums are exact on both sides, so borders that meet exactly are decided by the rule."""
    from atma_amd.kernel import sample_tokens
    logits = torch.zeros(9, 8, dtype=BF, device=dev)
    u = torch.arange(9, dtype=F32, device=dev) / 8
    assert sample_tokens(logits, u).tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 7]
    p = torch.tensor([0.0, 0.125, 0.25, 0.26, 0.5, 0.75, 0.875, 0.9, 1.0], device=dev)
    assert sample_tokens(logits, torch.ones(9, device=dev), top_p=p).tolist() == [0, 0, 1, 2, 3, 5, 6, 7, 7]
    assert sample_tokens(logits, torch.ones(9, device=dev), top_k=torch.arange(9, dtype=torch.int32, device=dev)).tolist() == \
        [7, 0, 1, 2, 3, 4, 5, 6, 7]


def test_values_that_are_not_finite(dev):
    inf, nan = math.inf, math.nan
    rows = [[0.0, -inf, 1.0, -inf], [-inf] * 4, [0.0, inf, -inf, inf], [0.0, nan, inf, nan], [-inf, -inf, -3.0, -inf],
            [-0.0, 0.0, -0.0, 0.0], [3e38, -3e38, 1.0, 3e38]]
    for dtype in (BF, F32):
        logits = torch.tensor(rows).to(dtype)
        n = len(rows)
        for u in (0.0, 0.3, 0.6, 0.999):
            for sel in ((None, None, None), ([2] * n, None, None), (None, [0.7] * n, None), ([3] * n, [0.9] * n, [0.1] * n)):
                _check(dev, logits, [u] * n, [1.0] * n, *sel)
        _check(dev, logits, [0.9] * n, [0.0] * n)
    low = torch.full((3, 700), torch.finfo(BF).min, dtype=BF)   # masks of the type's lowest value
    low[1, 650] = 0.5
    _check(dev, low, [0.5] * 3, [1.0] * 3, [5] * 3, [0.9] * 3)


def test_parameters_out_of_range(dev):
    """Every value of a parameter has a meaning."""
    g = torch.Generator().manual_seed(2)
    inf, nan = math.inf, math.nan
    logits = _logits(g, 8, 300).to(BF)
    u = [0.0, -1.0, 1.0, 5.0, nan, inf, -inf, 0.5]
    _check(dev, logits, u, [1.0] * 8)
    t = [0.0, -1.0, nan, -inf, 1e-30, 1e-45, 1e30, inf]
    _check(dev, logits, [0.37] * 8, t)
    _check(dev, logits, [0.37] * 8, [1.0] * 8, [0, -5, 299, 300, 301, 2 ** 31 - 1, -2 ** 31, 1])
    _check(dev, logits, [0.37] * 8, [1.0] * 8, None, [0.0, -1.0, nan, 1.0, 2.0, inf, -inf, 1e-30])
    _check(dev, logits, [0.37] * 8, [1.0] * 8, None, None, [0.0, -1.0, nan, 1.0, 2.0, inf, -inf, 1e-30])


def test_numbers_for_every_row(dev):
    from atma_amd.kernel import sample_tokens
    g = torch.Generator().manual_seed(3)
    logits, u = _logits(g, 20, 1000).to(dev), torch.rand(20, generator=g).to(dev)
    full = lambda v, d=F32: torch.full((20,), v, dtype=d, device=dev)   # noqa: E731
    want = sample_tokens(logits, u, full(0.7), top_k=full(40, torch.int32), top_p=full(0.9), min_p=full(0.02))
    assert torch.equal(sample_tokens(logits, u, 0.7, top_k=40, top_p=0.9, min_p=0.02), want)
    assert torch.equal(sample_tokens(logits, u, full(0.7), 40, 0.9, full(0.02)), want)
    assert torch.equal(sample_tokens(logits, u, 0), logits.argmax(1))


def test_strides_rows_and_outputs(dev):
    from atma_amd.kernel import sample_tokens
    g = torch.Generator().manual_seed(4)
    for dtype in (BF, F32):
        logits = _logits(g, 6, 777).to(dtype).to(dev)
        u = torch.rand(6, generator=g).to(dev)
        k = torch.tensor([5, 0, 30, 2, 1, 9], dtype=torch.int32, device=dev)
        want = sample_tokens(logits, u, 0.9, top_k=k, top_p=0.8)
        wide = torch.full((6, 801), float("inf"), dtype=dtype, device=dev)
        for at in (0, 1, 5, 24):
            wide[:] = float("inf")
            wide[:, at:at + 777] = logits
            assert torch.equal(sample_tokens(wide[:, at:at + 777], u, 0.9, top_k=k, top_p=0.8), want)
        assert torch.equal(sample_tokens(logits.t().contiguous().t(), u, 0.9, top_k=k, top_p=0.8), want)
        same = sample_tokens(logits[:1].expand(6, 777), u, 0.9, top_k=5, top_p=0.8)
        assert torch.equal(same, sample_tokens(logits[:1].repeat(6, 1), u, 0.9, top_k=5, top_p=0.8))
        two = torch.stack((u, u), 1)
        k2 = torch.stack((k, k), 1)
        assert torch.equal(sample_tokens(logits, two[:, 0], 0.9, top_k=k2[:, 1], top_p=0.8), want)
        held = torch.full((8,), -7, dtype=torch.int64, device=dev)
        out = sample_tokens(logits, u, 0.9, top_k=k, top_p=0.8, ids_out=held[1:7])
        assert out.data_ptr() == held[1:].data_ptr() and held.tolist() == [-7, *want.tolist(), -7]
    assert sample_tokens(torch.zeros(0, 9, device=dev), torch.zeros(0, device=dev)).shape == (0,)
    with pytest.raises(ValueError, match="ids_out"):
        sample_tokens(logits, u, ids_out=held)
    with pytest.raises(RuntimeError, match="GPU only"):
        sample_tokens(logits, u.cpu())


def test_a_million_logits(dev):
    """The longest rows: the sums of all weights, equal ones and others, at both ends."""
    from atma_amd.kernel import sample_tokens
    V = 1 << 20
    logits = torch.zeros(4, V, dtype=BF, device=dev)
    u = torch.tensor([0.0, 0.25, 0.5 + 2.0 ** -20, 1 - 2.0 ** -24], device=dev)
    assert sample_tokens(logits, u).tolist() == [0, V // 4, V // 2 + 1, V - 1]
    assert sample_tokens(logits, u, top_p=0.5).tolist() == [0, V // 8, V // 4, V // 2 - 1]
    assert sample_tokens(logits, u, top_k=V // 2).tolist() == [0, V // 8, V // 4, V // 2 - 1]
    g = torch.Generator().manual_seed(5)
    x = _logits(g, 2, V).float()
    _check(dev, x, [0.3, 0.9], [1.0, 0.7], [0, 5000], [0.9, 0.95], doubtful=2)


def test_frequencies(dev):
    """Draws of one row follow its weights: chi-square of 40 cells, 99.99% of right samplers below 85."""
    from atma_amd.kernel import sample_tokens
    g = torch.Generator().manual_seed(6)
    x = _logits(g, 1, 40, 1.0)
    n = 20000
    ids = sample_tokens(x.to(dev).expand(n, 40).contiguous(), torch.rand(n, generator=g).to(dev), 0.8).cpu()
    want = torch.softmax(x[0].double() / 0.8, 0) * n
    seen = torch.bincount(ids, minlength=40).double()
    assert ((seen - want).square() / want).sum() < 85


def test_streams_graphs_and_compile(dev):
    from atma_amd.kernel import sample_tokens
    g = torch.Generator().manual_seed(7)
    logits = [_logits(g, 5, 2000).to(BF).to(dev) for _ in range(3)]
    u = [torch.rand(5, generator=g).to(dev) for _ in range(3)]
    t = torch.tensor([0.0, 0.5, 1.0, 1.5, 0.8], device=dev)

    def f(x, v):
        return sample_tokens(x, v, t, top_k=50, top_p=0.9, min_p=0.01)

    want = [f(x, v) for x, v in zip(logits, u)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f(logits[0], u[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0])
    x, v, ids = logits[0].clone(), u[0].clone(), torch.empty(5, dtype=torch.int64, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sample_tokens(x, v, t, top_k=50, top_p=0.9, min_p=0.01, ids_out=ids)
    for i in (1, 2, 0, 1):
        x.copy_(logits[i])
        v.copy_(u[i])
        graph.replay()
        assert torch.equal(ids, want[i])
    compiled = torch.compile(f, backend="aot_eager")
    assert torch.equal(compiled(logits[2], u[2]), want[2])
