"""Checkpoints and the 8-bit MLP: its own state goes round; that of a 16-bit MLP, which it cannot hold, is refused."""

import pytest
import torch

from atma_amd.layers import global_attention as G
from atma_amd.layers.loader import load_model, save_checkpoint


@pytest.fixture
def quantized(monkeypatch):
    """Models whose MLPs are in 8 bits, with a stand-in for the quantizer, which needs the GPU."""
    from atma_amd.engine import Atma, AtmaConfig
    monkeypatch.setattr(G, "quantize_weight_fp8", lambda w: (w.detach().mul(100).to(torch.float8_e4m3fn),
                                                             torch.full((2, 2), 127, dtype=torch.uint8)))
    hf = AtmaConfig(vocab_size=64, num_hidden_layers=3, hidden_size=64, head_dim=16)
    return lambda seed: Atma(hf).init_weights(0.05, seed)


@pytest.mark.parametrize("strict", [True, False])
def test_a_16_bit_checkpoint_is_refused_after_quantizing(quantized, tmp_path, strict):
    path = tmp_path / "weights.pt"
    save_checkpoint(quantized(1), path)
    model = quantized(2).quantize_mlps()
    with pytest.raises(RuntimeError, match="blocks.0.mlp holds its weights in 8 bits"):
        load_model(model, path, strict=strict)
    other = load_model(quantized(2), path, strict=strict).quantize_mlps()
    want = quantized(1).quantize_mlps()
    for a, b in zip(other.state_dict().values(), want.state_dict().values()):
        assert torch.equal(a, b)


def test_8_bit_state_goes_round(quantized, tmp_path):
    path = tmp_path / "weights.pt"
    first = quantized(1).quantize_mlps()
    save_checkpoint(first, path)
    second = load_model(quantized(2).quantize_mlps(), path, strict=True)
    for (name, a), b in zip(first.state_dict().items(), second.state_dict().values()):
        assert torch.equal(a, b), name


def test_one_mlp_by_itself(quantized):
    mlp = G.MLP(32)
    held = G.Fp8MLP(mlp)
    with pytest.raises(RuntimeError, match="Fp8MLP holds its weights in 8 bits"):
        held.load_state_dict(mlp.state_dict(), strict=False)
    held.load_state_dict(G.Fp8MLP(G.MLP(32)).state_dict())
