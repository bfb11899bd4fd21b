"""No byte behind a bias is read by the 8-bit products: of an odd number of 16-bit values the last is read by a load of its
own size, not with the word that holds it.  A read of the whole word gives the same results, so the generated code is
looked at: each kernel that takes odd widths has 2-byte loads (which nothing else in them needs)."""

import re
import subprocess

from atma_amd import _build


def test_16_bit_biases_are_read_by_their_size(tmp_path):
    src, out = _build.CSRC / "fp8_gemm.hip", tmp_path / "out.s"
    proc = subprocess.run([*_build.compile_command(src), "--cuda-device-only", "-S", str(src), "-o", str(out)],
                          stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert proc.returncode == 0, proc.stdout[-2000:]
    bodies = dict(re.findall(r"\n(_Z\w+):.*?\n(.*?)\n\s*\.section", out.read_text(), flags=re.S))
    few = [n for n in bodies if "fp8_few_kernel" in n or "fp8_gated_few_kernel" in n]
    tiles = [n for n in bodies if "fp8_tile_kernel" in n and "Lb0EE" in n]   # (gated ones have an even number of features)
    assert len(few) > 1 and len(tiles) > 1
    for n in few:
        assert bodies[n].count("global_load_ushort") >= 4, n
    for n in tiles:
        assert bodies[n].count("global_load_ushort") >= 1, n
