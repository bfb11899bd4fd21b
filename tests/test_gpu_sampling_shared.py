"""Few long rows, which many workgroups share (``atma_sample_tokens_in`` with a workspace), against one workgroup a row
(``atma_sample_tokens``): weights are whole numbers and their sums exact, so the ids are equal, whatever the logits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")


def _both(dev, logits, u, t, k=None, p=None, m=None, shared=True):
    """ids of both; parameters are tensors, numbers or None."""
    from atma_amd import _lib
    lib = _lib.load()
    rows, V = logits.shape
    code = _lib.DTYPE_CODE[logits.dtype]
    held = [v.to(dev).contiguous() if torch.is_tensor(v) else v for v in (t, k, p, m)]
    args = []
    for v, off in zip(held, (1.0, 0, 1.0, 0.0)):
        args += [v.data_ptr(), off] if torch.is_tensor(v) else [None, off if v is None else v]
    u = u.to(dev)
    need = lib.atma_sample_tokens_workspace(rows, V, code)
    assert (need > 0) == shared
    work = torch.full((need + 8,), 0xff, dtype=torch.uint8, device=dev)
    out = []
    for f, more in ((lib.atma_sample_tokens, ()), (lib.atma_sample_tokens_in, (work.data_ptr(), need))):
        ids = torch.full((rows,), -1, dtype=torch.int64, device=dev)
        _lib.check(f(logits.data_ptr(), logits.stride(0), u.data_ptr(), *args, ids.data_ptr(), rows, V, code, *more,
                     _lib.stream_handle(dev)), "sample_tokens")
        out.append(ids.cpu())
    assert (work[need:] == 0xff).all()
    assert torch.equal(out[0], out[1]), (out, u, held)
    assert ((out[0] >= 0) & (out[0] < V)).all()
    return out[1]


def _params(g, rows, V):
    pick = lambda *v: torch.tensor(v, dtype=torch.float64)[torch.randint(0, len(v), (rows,), generator=g)]   # noqa: E731
    rnd = lambda: torch.rand(rows, generator=g, dtype=torch.float64)   # noqa: E731
    t = torch.where(rnd() < 0.7, 0.2 + 1.5 * rnd(), pick(0.0, -1.0, NAN, 1e-3, 1e-30, 60.0, 1e30))
    k = torch.where(rnd() < 0.5, torch.exp(rnd() * 10).floor(), pick(0, -5, 1, 2, V - 1, V, V + 7, 2 ** 31 - 1))
    p = torch.where(rnd() < 0.6, rnd(), pick(1.0, 2.0, 0.0, -1.0, 1e-9, 0.9999999, NAN))
    m = torch.where(rnd() < 0.4, 0.3 * rnd(), pick(0.0, -1.0, 1.0, 2.0, 1e-6, 1e-30, NAN))
    u = torch.where(rnd() < 0.7, rnd(), pick(0.0, 1.0, 1 - 2.0 ** -24, -3.0, 5.0, NAN))
    return u.to(F32), t.to(F32), k.clamp(-9, 2 ** 31 - 1).to(torch.int32), p.to(F32), m.to(F32)


def _rows(g, kind, rows, V):
    x = 3 * torch.randn(rows, V, generator=g)
    if kind == "quarters":          # hundreds and thousands of equal logits
        return (x * 4).round() / 4
    if kind == "whole":             # bins that hold more than the list
        return x.round()
    if kind == "constant":
        return torch.full((rows, V), -1.5)
    if kind == "few":               # whole parts of a row without a weight
        x[torch.rand(rows, V, generator=g) < 0.999] = -INF
        x[0] = -INF
        x[-1, : V // 2] = -INF
    if kind == "infinite":
        x[:, torch.randint(0, V, (3,), generator=g)] = INF
        x[0] = INF
        x[-1, V // 3:] = -INF
    if kind == "nan":
        for r in range(0, rows, 2):
            x[r, torch.randint(0, V, (4,), generator=g)] = NAN
        x[-1, -1] = NAN
    if kind == "close":
        x = 7 + 1e-4 * x
    if kind == "far":
        x = 1e37 * x
    if kind == "zeros":
        x = torch.where(torch.rand(rows, V, generator=g) < 0.5, 0.0, -0.0)
    return x


@pytest.mark.parametrize("kind", ["plain", "quarters", "whole", "constant", "few", "infinite", "nan", "close", "far", "zeros"])
@pytest.mark.parametrize("V,dtype", [(32769, F32), (50304, F32), (65536, BF), (70001, HF), (100003, F32)])
def test_shared_rows(dev, V, dtype, kind):
    g = torch.Generator().manual_seed(V + len(kind))
    for rows in (1, 12):
        logits = _rows(g, kind, rows, V).to(dtype).to(dev)
        for turn in range(4):
            u, t, k, p, m = _params(g, rows, V)
            _both(dev, logits, u, t, k, p, m)
            _both(dev, logits, u, t, None, p, None)
            _both(dev, logits, u, t, k, None, m)
            _both(dev, logits, u, t, None, None, m)
            _both(dev, logits, u, 0.8, int(k[0]), float(p[0]), float(m[0]))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_the_longest_rows(dev, dtype):
    g = torch.Generator().manual_seed(1)
    V = 1 << 20
    for rows in (1, 3):
        logits = _rows(g, "plain", rows, V).to(dtype).to(dev)
        for turn in range(3):
            u, t, k, p, m = _params(g, rows, V)
            _both(dev, logits, u, t, k, p, m)
            _both(dev, logits, u, t, None, p, None)


def test_the_most_rows(dev):
    """The border of the rule, and rows apart and in any order."""
    from atma_amd import _lib
    lib = _lib.load()
    g = torch.Generator().manual_seed(2)
    V = 33333
    most = max(r for r in range(1, 600) if lib.atma_sample_tokens_workspace(r, V, _lib.ATMA_F32))
    wide = _rows(g, "plain", most + 1, V + 5).to(dev)
    for rows in (most, most + 1):
        u, t, k, p, m = _params(g, rows, V)
        _both(dev, wide[:rows, 3:V + 3], u, t, k, p, m, shared=rows == most)


def test_through_the_call(dev):
    """As users have it: eager, on a second stream, captured and replayed with other logits, two at once."""
    from atma_amd.kernel import sample_tokens
    g = torch.Generator().manual_seed(3)
    V, rows = 50304, 4
    rnd = lambda: torch.rand(rows, generator=g).to(dev)   # noqa: E731
    xs = [_rows(g, "plain", rows, V).to(dev) for _ in range(3)]
    u, t, p = rnd(), 0.5 + rnd(), 0.5 + 0.5 * rnd()
    k = torch.tensor([0, 5, 100, 1], dtype=torch.int32, device=dev)
    want = [_both(dev, x, u, t, k, p, None).to(dev) for x in xs]
    call = lambda x: sample_tokens(x, u, t, top_k=k, top_p=p)   # noqa: E731
    for x, w in zip(xs, want):
        assert torch.equal(call(x), w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            a = call(xs[0])
        b = call(xs[1])
        torch.cuda.synchronize()
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    held, ids = xs[0].clone(), torch.empty(rows, dtype=torch.int64, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sample_tokens(held, u, t, top_k=k, top_p=p, ids_out=ids)
    for i in (1, 2, 0, 1):
        held.copy_(xs[i])
        call(xs[2])   # eager work between the replays
        graph.replay()
        assert torch.equal(ids, want[i])
