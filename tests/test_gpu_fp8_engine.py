"""Every 8-bit MLP call that the engine makes, prefills and decode steps, against float64 on the stream that the call had.

(The logits of a whole model say little: a value that noise carries over a rounding border moves the next block's input by more
than the noise, so two right models drift apart by the 8-bit rounding itself.)

Tolerance, relative to the branch: its own rounding, HALF / sqrt(3) rms.  The norm is fp32, 2^-16 off: an input of the first
product is on the other side of a border, a step of 2^-3 of it at most, with a chance of 2^-16 / step, sqrt(2^-16 / 8) =
1.4e-3 rms, which enters gate relu(a)^2 three times (sqrt(5) in quadrature), 3.1e-3.  The first product's sums lose 2e-4 (the
matrix instruction): at most 5% of the activations take a neighbouring code, a step of 2^-3 at most, 2^-3 / sqrt(3) = 0.072
rms over a binade: sqrt(0.05) 0.072 = 1.6e-2; a block in a thousand takes another scale, whose own rounding is 2^-3 / sqrt(3):
sqrt(1e-3) 0.072 = 2.3e-3."""

import pytest
import torch

from oracle import fp8 as O

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _held(t):
    data, scale = O.quantize(t)
    return data * O.spread(scale, *t.shape)


def _weight(m, name):
    return O.values(getattr(m, name + "_weight").view(torch.float8_e4m3fn), getattr(m, name + "_scale").view(torch.float8_e8m0fnu),
                    128)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_mlp_call_of_the_engine(dev, dtype):
    from atma_amd.engine import Config, LLMEngine
    from tests.test_gpu_engine import _drive, _model, _prompts
    hf, model, _ = _model(dtype)
    cfg = Config(kvcache_block_size=16, max_num_seqs=4, max_num_batched_tokens=4096, max_model_len=160, enforce_eager=True,
                 num_kvcache_blocks=64, hf_config=hf, fp8_mlp=True)
    engine = LLMEngine(cfg, model=model)
    calls = []

    def watch(block):
        norm, mlp = block.norm2.add_norm_fp8, block.mlp.forward_fp8

        def add_norm_fp8(branch, residual):
            out = norm(branch, residual)
            calls.append([block, out[2].detach().cpu()])
            return out

        def forward_fp8(*args):
            y = mlp(*args)
            calls[-1].append(y.detach().cpu())
            return y

        block.norm2.add_norm_fp8, block.mlp.forward_fp8 = add_norm_fp8, forward_fp8

    for block in model.blocks:
        watch(block)
    _drive(engine, _prompts([17, 1, 70], 2), new_tokens=3)
    engine.exit()
    # one prefill, two more steps of decoding
    assert [len(c) for c in calls] == [3] * len(calls) and len(calls) == 3 * len(model.blocks)
    assert sorted({c[1].shape[0] for c in calls}) == [3, 88]
    allowed = (HALF[dtype] ** 2 / 3 * 1.03 + 3.1e-3 ** 2 + 1.6e-2 ** 2 + 2.3e-3 ** 2) ** 0.5
    for block, stream, y in calls:
        m = block.mlp
        h, _ = O.residual_norm(stream, None, block.norm2.weight.detach().cpu(), block.norm2.eps, dtype)
        a, _ = O.linear(_held(h), _weight(m, "fc"), m.fc_bias.cpu())
        exact, _ = O.linear(_held(O.gated(a)), _weight(m, "proj"), m.proj_bias.cpu())
        err = ((y.double() - exact).norm() / exact.norm()).item()
        print(f"{tuple(stream.shape)} error {err:.2e} of {allowed:.2e}", flush=True)
        assert err <= allowed
