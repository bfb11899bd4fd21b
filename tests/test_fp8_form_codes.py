"""Which kernel an 8-bit product's sizes take, asked without a launch: sizes that are not served, and both ends of the rule."""

from atma_amd import _lib


def test_forms():
    lib = _lib.load()
    linear, gated = lib.atma_linear_fp8_form, lib.atma_linear_gated_fp8_form
    for bad in ((0, 64, 64), (1, 0, 64), (1, 64, 0), (1, 64, 40), (1, 64, 1 << 23), ((1 << 30) + 1, 64, 64), (1, (1 << 28) + 1, 64)):
        assert linear(*bad) == -1
    for bad in ((0, 128, 64), (1, 64, 64), (1, 192, 64), (1, 128, 40), (1, (1 << 27) + 128, 64)):
        assert gated(*bad) == -1
    assert linear(1, 1, 16) == 0 and 4 <= linear(65536, 4096, 1024) <= 7
    assert gated(1, 128, 16) == 0 and 1 <= gated(65536, 4096, 1024) <= 3
    # any K that LDS does not hold goes to the tiles
    assert gated(1, 128, 128 * 36) == 0 and gated(1, 128, 128 * 36 + 16) != 0
