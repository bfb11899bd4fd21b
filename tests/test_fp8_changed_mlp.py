"""An MLP that is more than its weights and biases has no 8-bit form: it is refused, and no other one is replaced."""

import pytest
from torch import nn

from atma_amd.layers.global_attention import MLP, Fp8MLP, Linear


class SubMLP(MLP):
    def forward(self, x, defer=False):
        return 2 * super().forward(x)


class SubLinear(Linear):
    def forward(self, x):
        return super().forward(x) + 1


def _own_forward(m):
    m.forward = lambda x, **kw: x


CHANGES = {
    "hook": lambda m: m.register_forward_hook(lambda *a: None),
    "pre-hook": lambda m: m.register_forward_pre_hook(lambda *a: None),
    "forward": _own_forward,
}


def _changed(where, change):
    m = MLP(32)
    CHANGES[change](getattr(m, where) if where else m)
    return m


def _subclass():
    return SubMLP(32)


def _projection(name, cls):
    m = MLP(32)
    old = getattr(m, name)
    setattr(m, name, cls(old.in_features, old.out_features))
    return m


def _parametrised(name):
    m = MLP(32)
    nn.utils.parametrize.register_parametrization(getattr(m, name), "weight", nn.Identity())
    return m


BAD = [_subclass, *(lambda w=w, c=c: _changed(w, c) for w in ("", "fc", "proj") for c in CHANGES),
       *(lambda n=n: _projection(n, SubLinear) for n in ("fc", "proj")), *(lambda n=n: _parametrised(n) for n in ("fc", "proj"))]


@pytest.mark.parametrize("make", BAD)
def test_changed_mlps_are_refused(make):
    m = make()
    # (the sizes are served: nothing but the change is in the way)
    with pytest.raises(ValueError, match="Fp8MLP is made from"):
        Fp8MLP(m)


def test_plain_projections_are_taken():
    with pytest.raises(RuntimeError, match="GPU only"):   # past the checks of the module
        Fp8MLP(_projection("fc", nn.Linear))
    handle = nn.modules.module.register_module_forward_hook(lambda *a: None)   # sees the module that takes its place
    try:
        with pytest.raises(RuntimeError, match="GPU only"):
            Fp8MLP(MLP(32))
    finally:
        handle.remove()


def test_nothing_is_replaced_beside_a_refused_mlp(monkeypatch):
    from atma_amd.engine import AtmaConfig
    from atma_amd.engine import model as M
    made = []

    class Stand(nn.Module):
        check = staticmethod(getattr(Fp8MLP, "check", lambda mlp: None))

        def __init__(self, mlp):
            super().__init__()
            made.append(mlp)
            self.check(mlp)

    monkeypatch.setattr(M, "Fp8MLP", Stand)
    hf = AtmaConfig(vocab_size=64, num_hidden_layers=3, hidden_size=64, head_dim=16)
    model = M.Atma(hf)
    before = [b.mlp for b in model.blocks]
    handle = model.blocks[2].mlp.proj.register_forward_hook(lambda *a: None)
    with pytest.raises(ValueError, match="Fp8MLP is made from"):
        model.quantize_mlps()
    assert [b.mlp for b in model.blocks] == before and made == []
    handle.remove()
    model.quantize_mlps()
    assert made == before and all(type(b.mlp) is Stand for b in model.blocks)


@pytest.mark.parametrize("training", [True, False])
def test_mode_is_kept(monkeypatch, training):
    """A model in ``eval()`` stays in it."""
    from atma_amd.layers import global_attention as G
    monkeypatch.setattr(G, "quantize_weight_fp8", lambda w: (w.detach().byte(), w.detach().byte()))
    assert Fp8MLP(MLP(32).train(training)).training is training
