"""Which kernel a product with 4-bit weights takes, asked without a launch: sizes that are not served, and that every kernel of the
rule is reached."""

from atma_amd import _lib


def test_forms():
    lib = _lib.load()
    linear, gated = lib.atma_linear_fp4_form, lib.atma_linear_gated_fp4_form
    for f in (linear, gated):
        for bad in ((0, 64, 64), (-1, 64, 64), (1, 0, 64), (1, -1, 64), (1, 64, 0), (1, 64, 40), (1, 64, 1 << 23), ((1 << 30) + 1, 64, 64),
                    (1, (1 << 28) + 1, 64), (1, 1 << 62, 64)):
            assert f(*bad) == -1
    assert gated(1, (1 << 27) + 1, 64) == -1 and linear(1, 1 << 28, 64) >= 0
    sizes = [(m, n, k) for m in (1, 16, 64, 256, 1024, 4096) for n in (64, 1024, 8192, 50304) for k in (64, 1024, 4096)]
    assert {linear(*s) for s in sizes} == set(range(9)) and {gated(*s) for s in sizes} == {0, 5, 6, 8}
    # the kernel that keeps the tokens' K in LDS serves only what fits there, the kernels of few rows no more than 1,024 of them
    assert linear(16, 8192, 2048) == 2 and linear(16, 8192, 2049 // 32 * 32 + 256) != 2
    assert all(f(1 << 30, 1, 1 << 22) >= 3 for f in (linear, gated))
