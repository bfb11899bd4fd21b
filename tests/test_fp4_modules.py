"""The modules with 4-bit weights and the sampling parameters where no GPU is needed: what has no 4-bit form, checkpoints,
the configuration, the random numbers of a request."""

import pytest
import torch
from torch import nn

from atma_amd.engine import Atma, AtmaConfig, Config, SamplingParams, Sequence
from atma_amd.engine.sequence import uniform
from atma_amd.layers import global_attention as G
from atma_amd.layers.loader import load_model, save_checkpoint


class SubMLP(G.MLP):
    def forward(self, x, defer=False):
        return 2 * super().forward(x)


class SubLinear(G.Linear):
    def forward(self, x):
        return super().forward(x) + 1


@pytest.fixture
def quantized(monkeypatch):
    """A stand-in for the quantizer, which needs the GPU."""
    def quantize(w):
        codes = (w.detach() * 1000).to(torch.int64).remainder(16).to(torch.uint8)
        return codes[:, ::2] + 16 * codes[:, 1::2], torch.full((w.shape[0], w.shape[1] // 32), 127, dtype=torch.uint8)
    monkeypatch.setattr(G, "quantize_weight_fp4", quantize)
    hf = AtmaConfig(vocab_size=64, num_hidden_layers=3, hidden_size=64, head_dim=16)
    return lambda seed: Atma(hf).init_weights(0.05, seed)


def _hooked(m):
    m.register_forward_hook(lambda *a: None)
    return m


def _parametrised(m):
    nn.utils.parametrize.register_parametrization(m, "weight", nn.Identity())
    return m


def test_changed_modules_are_refused(quantized):
    def mlp(change):
        m = G.MLP(32)
        change(m)
        return m
    for bad in (SubMLP(32), _hooked(G.MLP(32)), mlp(lambda m: _hooked(m.fc)), mlp(lambda m: _parametrised(m.proj)),
                mlp(lambda m: setattr(m, "fc", SubLinear(32, 256))), G.MLP(48)):
        with pytest.raises(ValueError, match="Fp4MLP"):
            G.Fp4MLP(bad)
    for bad in (SubLinear(32, 8), _hooked(G.Linear(32, 8)), _parametrised(G.Linear(32, 8)), G.Linear(48, 8), nn.Identity()):
        with pytest.raises(ValueError, match="Fp4Linear"):
            G.Fp4Linear(bad)
    held = G.Fp4Linear(nn.Linear(32, 8, bias=False).eval())
    assert held.fp4_bias is None and not held.training
    model = quantized(1)
    _hooked(model.blocks[2].mlp)
    with pytest.raises(ValueError):
        model.quantize_weights_fp4()
    assert not any(isinstance(m, (G.Fp4MLP, G.Fp4Linear)) for m in model.modules())   # none is replaced
    model = quantized(1)
    _hooked(model.proj)
    with pytest.raises(ValueError):
        model.quantize_weights_fp4()
    assert not any(isinstance(m, (G.Fp4MLP, G.Fp4Linear)) for m in model.modules())


@pytest.mark.parametrize("strict", [True, False])
def test_checkpoints(quantized, tmp_path, strict):
    path = tmp_path / "weights.pt"
    save_checkpoint(quantized(1), path)
    model = quantized(2).quantize_weights_fp4()
    assert model.quantize_weights_fp4() is model   # (nothing left to do)
    with pytest.raises(RuntimeError, match="blocks.0.mlp holds its weights in 4 bits"):
        load_model(model, path, strict=strict)
    with pytest.raises(RuntimeError, match="proj holds its weights in 4 bits"):
        load_model(model, {"proj.weight": torch.zeros(64, 64)}, strict=strict)
    want = quantized(1).quantize_weights_fp4()
    save_checkpoint(want, path)
    load_model(model, path, strict=True)
    for (name, a), b in zip(model.state_dict().items(), want.state_dict().values()):
        assert torch.equal(a, b), name
    assert model.half().proj.fp4_weight.dtype == torch.uint8


def test_modules_and_configuration_refuse(monkeypatch):
    with pytest.raises(RuntimeError, match="GPU only"):
        G.Fp4MLP(G.MLP(32))
    with pytest.raises(RuntimeError, match="GPU only"):
        G.Fp4Linear(G.Linear(32, 8))
    assert Config().fp4_weights is False
    from atma_amd.engine import ModelRunner
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    hf = AtmaConfig(vocab_size=64, num_hidden_layers=1, hidden_size=64, head_dim=16)
    with pytest.raises(ValueError, match="exclude"):
        ModelRunner(Config(hf_config=hf, fp8_mlp=True, fp4_weights=True))
    hf.dtype = torch.float32
    with pytest.raises(ValueError, match="16-bit"):
        ModelRunner(Config(hf_config=hf, fp4_weights=True))


def test_sampling_parameters():
    for bad in (dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.1), dict(min_p=-0.1), dict(min_p=1.5)):
        with pytest.raises(ValueError):
            SamplingParams(**bad)
    import numpy as np
    for bad in (dict(seed=0.5), dict(seed="1"), dict(top_k=2.5)):
        with pytest.raises(TypeError):
            SamplingParams(**bad)
    p = SamplingParams(seed=np.int64(3), top_k=np.int32(4))
    assert type(p.seed) is int and type(p.top_k) is int and Sequence([1], p).uniform() == uniform(3, 0)
    assert not SamplingParams().picks and not SamplingParams(temperature=0.0, top_k=5).picks
    for good in (dict(top_k=1), dict(top_p=0.5), dict(min_p=0.1), dict(seed=0)):
        assert SamplingParams(**good).picks


def test_random_numbers_of_a_request():
    # the first outputs of splitmix64 from seed 0 begin with these 24 bits
    assert [round(uniform(0, n) * 2 ** 24) for n in range(3)] == [0xE220A8, 0x6E789E, 0x06C45D]
    assert uniform(-1, 0) == uniform(2 ** 64 - 1, 0)
    u = [uniform(s, n) for s in range(200) for n in range(50)]
    assert all(0 <= v < 1 and v * 2 ** 24 == int(v * 2 ** 24) for v in u) and abs(sum(u) / len(u) - 0.5) < 0.01
    a, b = (Sequence([1, 2, 3], SamplingParams(seed=7)) for _ in range(2))
    first = [a.uniform(n) for n in range(3)]
    assert first == [uniform(7, n) for n in range(3)]
    b.token_ids.append(5)
    assert b.uniform() == first[1] and b.uniform(1) == first[2]
    assert Sequence([1]).uniform() != Sequence([1]).uniform()
