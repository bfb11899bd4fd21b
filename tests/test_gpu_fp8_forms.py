"""Each kernel of the 8-bit products (``atma_linear_fp8_form``, ``atma_linear_gated_fp8_form``) where it can go wrong: long
chains of K, several tiles a workgroup, special values, layouts, biases, graphs.  Every test names the kernel that its sizes
reach, so that a border that moves shows here.

Tolerances, derived:

* a value: half a step of the output type plus what the matrix instruction drops, as ``test_gpu_fp8``;
* all values of a call together: roundings to nearest are spread over a step, HALF / sqrt(3) rms of a value at most (a step
  is 2 HALF of a value at the bottom of its binade, less of a larger one), 3% more for the finite sample.  The
  instruction loses less than 2^-13 of the largest of eight products from each of them, sqrt(8) 2^-13 / sqrt(3) of their
  largest for eight, and the largest is at most as much as all eight together, whose sum is sqrt(8) smaller than eight times
  one: LOST = sqrt(8) 2^-13 / sqrt(3) of the result;
* an 8-bit activation gate relu(a)^2: LOST of a's and gate's rms moves it by 2 LOST |gate a| and LOST a^2, and a value changes its
  code when that carries it over a border, every 2^-4 of it at the closest: 16 LOST (2 E|1/a| + E|1/gate|), with E|1/a| about 5 for
  normal values cut at 1% of their rms (below, an activation is in the subnormal steps): 16 * 2e-4 * 15 = 5%.  A block
  takes another scale where its largest value is that close to a power of two: 3 LOST / ln 2 of the blocks, 0.1%."""

import pytest
import torch

from oracle import fp8 as O

pytestmark = pytest.mark.gpu

FP8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DROP = 2.0 ** -10
LOST = 8 ** 0.5 * 2.0 ** -13 / 3 ** 0.5
DT = [torch.bfloat16, torch.float16]

FEW16x16, FEW32x16, FEW16x32, FEW32x32, T256x256, T128x128, T64x128, T64x64 = range(8)
GFEW, G256, G128, G64 = range(4)
# form, M, N, K.  The first of each tile has three times more blocks of K than stages or more and two tiles in some
# workgroup at least (256 CUs, one or two workgroups each); the others are the sizes of the special cases
LONG = [(FEW16x16, 7, 1001, 4096), (FEW32x16, 33, 200, 8208), (FEW16x32, 9, 6201, 1040), (FEW32x32, 97, 2500, 1552),
        (T64x64, 40, 36149, 1808), (T64x64, 777, 1001, 2048), (T64x128, 70, 33595, 1200), (T128x128, 265, 34935, 1040),
        (T256x256, 2700, 12301, 912), (T256x256, 4000, 4001, 2064)]
SMALL = [(FEW16x16, 9, 257, 272), (FEW32x32, 129, 1001, 272), (T64x64, 65, 8190, 272), (T64x128, 2000, 1001, 528),
         (T128x128, 2100, 1001, 1040), (T256x256, 4000, 4001, 272)]
# form, M, H, K
GLONG = [(GFEW, 16, 4096, 4608), (G64, 650, 5632, 1200), (G128, 1041, 6784, 1040), (G256, 1553, 7680, 912)]
GSMALL = [(GFEW, 37, 256, 272), (G64, 2001, 1024, 272), (G128, 4201, 2048, 272), (G256, 4090, 2048, 912)]


def _form(form, M, N, K, gated=False):
    from atma_amd import _lib
    lib = _lib.load()
    got = (lib.atma_linear_gated_fp8_form if gated else lib.atma_linear_fp8_form)(M, N, K)
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:   # (another card has other borders)
        assert got == form, f"{M} x {K} -> {N} reaches kernel {got}, not {form}"


def _g(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _rows(dev, rows, dim, seed):
    """Normal rows of different size."""
    g = _g(dev, seed)
    return torch.randn(rows, dim, generator=g, device=dev) * torch.exp(torch.randn(rows, 1, generator=g, device=dev))


def _values(data, scale, tall=1):
    """The float64 values, on their device."""
    s = torch.exp2(scale.contiguous().view(torch.uint8).double() - 127)
    return data.float().double() * O.spread(s, *data.shape, tall)


def _operands(dev, M, N, K, seed=0):
    from atma_amd.kernel import quantize_fp8, quantize_weight_fp8
    x, xs = quantize_fp8(_rows(dev, M, K, seed))
    w, ws = quantize_weight_fp8(torch.randn(N, K, generator=_g(dev, seed + 1), device=dev) / K ** 0.5)
    return x, xs, w, ws


def _exact(x, xs, w, ws, bias=None):
    xv, wt = _values(x, xs), _values(w, ws, 128).t().contiguous()
    y = xv @ wt
    return (y if bias is None else y + bias.double()), xv.abs() @ wt.abs()


def _check(y, exact, size):
    err = (y.double() - exact).abs()
    assert (err <= HALF[y.dtype] * exact.abs() + DROP * size + torch.finfo(y.dtype).smallest_normal).all()
    rms = (err.norm() / exact.norm()).item()
    assert rms <= (1.03 * HALF[y.dtype] ** 2 / 3 + LOST ** 2) ** 0.5, rms


def _scales(h):
    """``oracle.fp8.scales`` of rows, without its loops: the smallest 2^e, e in [-126, 120], with |h| <= 448 2^e."""
    top = torch.nn.functional.pad(h.abs(), (0, -h.shape[1] % 128)).view(h.shape[0], -1, 128).amax(2)
    _, e = torch.frexp(top / 448)               # top / 448 in [2^(e - 1), 2^e); the quotient's rounding is looked at below
    e = torch.where(top <= 448 * torch.exp2((e - 1).double()), e - 1, e)
    e = torch.where(top > 448 * torch.exp2(e.double()), e + 1, e)
    return torch.exp2(torch.where(top > 0, e, torch.full_like(e, -126)).clamp(-126, 120).double())


def test_vectorised_scales(dev):
    h = _rows(dev, 50, 300, 3).double()
    h[1] = 0
    h[2, 5], h[3, 5], h[4, 5], h[5, 299] = 448 * 8, 448 * 8 * (1 + 2.0 ** -40), 1e-300, 1e38
    assert torch.equal(_scales(h).cpu(), O.scales(h.cpu()))


def _check_gated(data, scale, exact, size, codes=True):
    """The activation of the exact sums, rounded once: every value near, few codes and scales other than the exact ones."""
    a, gate = exact.chunk(2, 1)
    da, dg = (DROP * size).chunk(2, 1)
    h, pos = O.gated(exact), a.clamp_min(0)
    dh = dg * (pos + da).square() + gate.abs() * (2 * pos + da) * da
    s = torch.exp2(scale.contiguous().view(torch.uint8).double() - 127)
    full = O.spread(s, *h.shape)
    v = data.float().double() * full
    bound = torch.maximum(2.0 ** -4 * (h.abs() + dh), 2.0 ** -10 * full) * (1 + 2.0 ** -6) + dh
    assert not torch.isnan(v).any() and ((v - h).abs() <= bound).all()
    if codes:
        es = _scales(h)
        same = s == es
        assert (~same).double().mean().item() <= 3 * LOST / 0.69 + 3 / same.numel()
        differ = (data.float().double() != O.round_e4m3(h / O.spread(es, *h.shape))) & (O.spread(same.double(), *h.shape) > 0)
        assert differ.double().mean().item() <= 16 * LOST * 15
        assert ((v - h).norm() / h.norm()).item() <= 1.03 * 2.0 ** -4 / 3 ** 0.5 + 3 * LOST


# ------------------------------------------------------------------------------------------------ values
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("form,M,N,K", LONG + SMALL)
def test_linear(dev, form, M, N, K, dtype):
    from atma_amd.kernel import linear_fp8
    _form(form, M, N, K)
    ops = _operands(dev, M, N, K, M + N + K)
    exact, size = _exact(*ops)
    _check(linear_fp8(*ops, out_dtype=dtype), exact, size)
    for bt in (dtype, torch.float32):
        b = torch.randn(N, generator=_g(dev, 1), device=dev).to(bt)
        _check(linear_fp8(*ops, b, out_dtype=dtype), exact + b.double(), size)


@pytest.mark.parametrize("bias", [None, torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("form,M,H,K", GLONG + GSMALL)
def test_linear_gated(dev, form, M, H, K, bias):
    from atma_amd.kernel import linear_gated_fp8
    _form(form, M, H, K, gated=True)
    ops = _operands(dev, M, 2 * H, K, M + H + K)
    b = None if bias is None else torch.randn(2 * H, generator=_g(dev, 1), device=dev).to(bias)
    data, scale = linear_gated_fp8(*ops, b)
    _check_gated(data, scale, *_exact(*ops, b))


# ------------------------------------------------------------------------------------------------ special values
def _special_rows(dev, M, N, K, seed):
    """Operands with a row of zeros, a NaN, an infinity before quantizing and a NaN scale, the last in the last row."""
    from atma_amd.kernel import quantize_fp8, quantize_weight_fp8
    v = _rows(dev, M, K, seed)
    v[0], v[2, K // 2], v[3, K - 1] = 0, float("nan"), float("-inf")
    x, xs = quantize_fp8(v)
    xs.view(torch.uint8)[M - 1, -1] = 255
    w, ws = quantize_weight_fp8(torch.randn(N, K, generator=_g(dev, seed + 1), device=dev) / K ** 0.5)
    keep = torch.ones(M, dtype=torch.bool, device=dev)
    keep[[2, 3, M - 1]] = False
    return x, xs, w, ws, keep


@pytest.mark.parametrize("form,M,N,K", SMALL)
def test_linear_keeps_rows_and_features_apart(dev, form, M, N, K):
    from atma_amd.kernel import linear_fp8
    _form(form, M, N, K)
    x, xs, w, ws, keep = _special_rows(dev, M, N, K, 8)
    b = torch.randn(N, generator=_g(dev, 2), device=dev).bfloat16()
    y = linear_fp8(x, xs, w, ws, b)
    assert torch.isnan(y[~keep]).all() and torch.equal(y[0], b)
    exact, size = _exact(x[keep], xs[keep], w, ws, b)
    _check(y[keep], exact, size)
    lost = ws.clone()
    lost.view(torch.uint8)[1, 0] = 255   # a NaN scale of the second block of weights
    z = linear_fp8(x, xs, w, lost, b)
    rows = keep.nonzero().view(-1)
    assert torch.isnan(z[:, 128:256]).all()
    assert torch.equal(z[rows, :128], y[rows, :128]) and torch.equal(z[rows, 256:], y[rows, 256:])


@pytest.mark.parametrize("form,M,H,K", GSMALL)
def test_gated_keeps_rows_and_blocks_apart(dev, form, M, H, K):
    from atma_amd.kernel import linear_gated_fp8
    _form(form, M, H, K, gated=True)
    x, xs, w, ws, keep = _special_rows(dev, M, 2 * H, K, 8)
    data, scale = linear_gated_fp8(x, xs, w, ws)
    codes, d = scale.view(torch.uint8), data.float()
    assert torch.isnan(d[~keep]).all() and (codes[~keep] == 1).all()
    assert (d[0] == 0).all() and (codes[0] == 1).all()
    _check_gated(data[keep], scale[keep], *_exact(x[keep], xs[keep], w, ws))
    for block in (1, H // 128):   # of a, of gate
        lost = ws.clone()
        lost.view(torch.uint8)[block, 0] = 255
        z, zs = linear_gated_fp8(x, xs, w, lost)
        hit = torch.zeros(H // 128, dtype=torch.bool, device=dev)
        hit[block % (H // 128)] = True
        cols = hit.repeat_interleave(128)
        rows = keep.nonzero().view(-1)
        assert torch.isnan(z.float()[:, cols]).all() and (zs.view(torch.uint8)[:, hit] == 1).all()
        assert torch.equal(z.view(torch.uint8)[rows][:, ~cols], data.view(torch.uint8)[rows][:, ~cols])
        assert torch.equal(zs.view(torch.uint8)[rows][:, ~hit], codes[rows][:, ~hit])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form,M,N,K", SMALL)
def test_linear_bias_of_special_values(dev, form, M, N, K, dtype):
    """Infinities and NaN in a bias reach their own feature: the first, one inside, the last."""
    from atma_amd.kernel import linear_fp8
    _form(form, M, N, K)
    ops = _operands(dev, M, N, K, 4)
    b = torch.randn(N, generator=_g(dev, 1), device=dev).to(dtype)
    clean = linear_fp8(*ops, b)
    at = [0, N // 2, N - 1]
    special = b.clone()
    special[at] = torch.tensor([float("inf"), float("nan"), float("-inf")], device=dev).to(dtype)
    y = linear_fp8(*ops, special)
    assert (y[:, 0] == float("inf")).all() and torch.isnan(y[:, N // 2]).all() and (y[:, N - 1] == float("-inf")).all()
    y[:, at] = clean[:, at]
    assert torch.equal(y, clean)


@pytest.mark.parametrize("form,M,H,K", GSMALL)
def test_gated_of_special_activations(dev, form, M, H, K):
    """An activation that is not finite (an infinite bias of a or gate, a finite a whose square is past the fp32 range) is
    NaN in its place and does not enter its block's scale; the largest finite ones set it."""
    from atma_amd.kernel import linear_gated_fp8
    _form(form, M, H, K, gated=True)
    ops = _operands(dev, M, 2 * H, K, 4)
    inf, big = float("inf"), 3e19     # big^2 = 9e38
    b = 0.1 * torch.randn(2 * H, generator=_g(dev, 1), device=dev)
    clean = b.clone()
    # feature: (a's bias, gate's bias), spread over the waves and lane halves of the first and the last block
    special = {0: (inf, 1.0), 17: (big, 1.0), 40: (1.0, inf), 77: (inf, -1.0), 127: (float("nan"), 1.0), H - 100: (big, -1.0),
               H - 128 + 55: (1.0, float("nan")), H - 1: (inf, inf)}
    for f, (pa, pg) in special.items():
        b[f], b[H + f] = pa, pg
        clean[f], clean[H + f] = float("-inf"), 0.0      # such a feature is 0: in no block's scale
    data, scale = linear_gated_fp8(*ops, b)
    want, ws = linear_gated_fp8(*ops, clean)
    d, w = data.float(), want.float()
    at = sorted(special)
    # (an a that the rest of its sum takes below zero is 0 and 0 inf or 0 NaN, NaN all the same; big is past every sum here)
    assert torch.isnan(d[:, at]).all() and (w[:, at] == 0).all()
    other = torch.ones(H, dtype=torch.bool, device=dev)
    other[at] = False
    assert torch.equal(d[:, other], w[:, other]) and not torch.isnan(d[:, other]).any()
    assert torch.equal(scale.view(torch.uint8), ws.view(torch.uint8))
    # the largest finite activations: 1e18^2 = 1e36 with a gate of up to some 100
    b, f = clean.clone(), 9
    b[f], b[H + f] = 1e18, 10.0
    data, scale = linear_gated_fp8(*ops, b)
    exact, size = _exact(*ops, torch.where(torch.isinf(b), torch.full_like(b, -1e30), b))
    a, gate = exact[:, f], exact[:, H + f]
    h = a.square() * gate
    v = _values(data, scale)[:, f]
    assert ((v - h).abs() <= (2.0 ** -4 * (1 + 2.0 ** -6)) * h.abs() + 2 * DROP * size[:, H + f] * a.square()).all()


# ------------------------------------------------------------------------------------------------ layouts
def _wide(t, off, value):
    """t as a slice of wider rows at an offset, ``value`` around it."""
    u = t.view(torch.uint8)
    held = torch.full((u.shape[0] + 1, (u.shape[1] + 63) // 16 * 16), value, dtype=torch.uint8, device=t.device)
    held[:u.shape[0], off:off + u.shape[1]] = u
    return held.view(t.dtype)[:u.shape[0], off:off + u.shape[1]]


def _turned(t):
    return t.view(torch.uint8).t().contiguous().t().view(t.dtype)


@pytest.mark.parametrize("gated,form,M,N,K", [(False, *s) for s in SMALL] + [(True, *s) for s in GSMALL])
def test_other_layouts(dev, gated, form, M, N, K):
    """Slices of wider or misaligned tensors, broadcast rows, scales transposed, padded and at odd offsets: the bits of the
    call on fresh tensors."""
    from atma_amd.kernel import linear_fp8, linear_gated_fp8
    _form(form, M, N, K, gated)
    x, xs, w, ws = _operands(dev, M, (2 if gated else 1) * N, K, 6)

    def call(*ops):
        return torch.cat([t.view(torch.uint8).view(M, -1) for t in linear_gated_fp8(*ops)], 1) if gated else linear_fp8(*ops)

    want = call(x, xs, w, ws)
    for ops in ((_wide(x, 0, 127), _wide(xs, 0, 255), _wide(w, 16, 127), _wide(ws, 4, 255)),
                (_wide(x, 5, 127), xs.contiguous(), _wide(w, 3, 127), ws.contiguous()),
                (_turned(x), _turned(xs), _turned(w), _turned(ws)), (x, _wide(xs, 1, 255), w, _wide(ws, 2, 255))):
        assert torch.equal(call(*ops), want)
    one = call(x[:1].expand(M, K), xs[:1].expand(M, xs.shape[1]), w, ws)
    assert torch.equal(one, want[:1].expand_as(one))


@pytest.mark.parametrize("gated,form,M,N,K", [(False, *s) for s in SMALL] + [(True, *s) for s in GSMALL])
def test_a_bias_anywhere(dev, gated, form, M, N, K):
    """A bias at an odd offset, with a stride, expanded, in each type: as a fresh copy of it."""
    from atma_amd.kernel import linear_fp8, linear_gated_fp8
    _form(form, M, N, K, gated)
    n = (2 if gated else 1) * N
    ops = _operands(dev, M, n, K, 4)
    for dtype in (*DT, torch.float32):
        held = torch.randn(2 * n + 3, generator=_g(dev, 1), device=dev).to(dtype)
        for b in (held[1:n + 1], held[3:2 * n + 3:2], held[7].expand(n)):
            if gated:
                for p, q in zip(linear_gated_fp8(*ops, b), linear_gated_fp8(*ops, b.clone())):
                    assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))
            else:
                assert torch.equal(linear_fp8(*ops, b), linear_fp8(*ops, b.clone()))


# ------------------------------------------------------------------------------------------------ streams and graphs
@pytest.mark.parametrize("gated,form,M,N,K", [(False, *s) for s in SMALL] + [(True, *s) for s in GSMALL])
def test_captured_repeated_and_on_another_stream(dev, gated, form, M, N, K):
    from atma_amd.kernel import linear_fp8, linear_gated_fp8, quantize_fp8
    _form(form, M, N, K, gated)
    n = (2 if gated else 1) * N
    w, ws = _operands(dev, 1, n, K, 4)[2:]
    b = torch.randn(n, generator=_g(dev, 1), device=dev).bfloat16()

    def call(x, xs):
        out = linear_gated_fp8(x, xs, w, ws, b) if gated else (linear_fp8(x, xs, w, ws, b),)
        return [t.view(torch.uint8) for t in out]

    inputs = [quantize_fp8(_rows(dev, M, K, s)) for s in range(3)]
    want = [call(*i) for i in inputs]
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(call(*inputs[0]), want[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(*inputs[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want[1]))
    static = [t.clone() for t in inputs[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(*static)
    for i in (1, 2, 0, 1):
        for s, t in zip(static, inputs[i]):
            s.view(torch.uint8).copy_(t.view(torch.uint8))
        graph.replay()
        eager = call(*inputs[i])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[i])) and all(torch.equal(p, q) for p, q in zip(eager, want[i]))


# ------------------------------------------------------------------------------------------------ the C ABI's outputs
@pytest.mark.parametrize("form,M,N,K", SMALL)
def test_linear_stores_rows_anywhere(dev, form, M, N, K):
    """y at any element and any stride from N on, multiples of 8 among them; what lies between its rows stays as it was."""
    from atma_amd import _lib
    from atma_amd.kernel import linear_fp8
    _form(form, M, N, K)
    x, xs, w, ws = _operands(dev, M, N, K, 4)
    want = linear_fp8(x, xs, w, ws)
    for off, ldy in ((1, (N + 7) // 8 * 8), (3, (N + 7) // 8 * 8 + 8), (0, N), (7, N + 1), (4, (N + 15) // 8 * 8)):
        held = torch.full((off + M * ldy + 8,), 7.0, dtype=torch.bfloat16, device=dev)
        y = held[off:off + M * ldy].view(M, ldy)
        rc = _lib.load().atma_linear_fp8(
            x.data_ptr(), x.stride(0), xs.data_ptr(), xs.stride(0), w.data_ptr(), w.stride(0), ws.data_ptr(), ws.stride(0),
            None, 0, y.data_ptr(), ldy, M, N, K, 1, _lib.stream_handle(dev))
        assert rc == 0, _lib.load().atma_last_error()
        assert torch.equal(y[:, :N], want)
        assert (y[:, N:] == 7).all() and (held[:off] == 7).all() and (held[off + M * ldy:] == 7).all()
