"""Towers on the operators against the towers' own layers, on the CPU: ``ops.linear`` and ``ops.layer_norm`` are stood in for by their definitions in
eager torch, so what is tested is which layers ``use_kernels`` calls, with what, and when."""
import pytest
import torch

import test_ops as towers
from lsdm_amd import ops
from lsdm_amd.text import use_kernels

ACTS = {"none": lambda z: z, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "quick_gelu": lambda z: z * torch.sigmoid(1.702 * z), "silu": torch.nn.functional.silu,
        "sigmoid": torch.sigmoid, "tanh": torch.tanh}


@pytest.fixture(autouse=True)
def _host_operators(monkeypatch):
    def linear(x, w, b=None, activation="none", residual=None, *, checkpoint8=False):
        y = ACTS[activation](torch.nn.functional.linear(x, w, b))
        return y if residual is None else y + residual

    def layer_norm(x, w=None, b=None, eps=1e-5, *, checkpoint8=False):
        return torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, eps)
    monkeypatch.setattr(ops, "linear", linear)
    monkeypatch.setattr(ops, "layer_norm", layer_norm)
    with torch.enable_grad():
        yield


def ids():
    return torch.randint(1, 40, (3, 7), generator=torch.Generator().manual_seed(2))


def same(a, b):
    assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)       # (the stand-ins add in the same order; a handful of fp32 roundings at most)


def outputs(m, x, seed=5):
    torch.manual_seed(seed)
    return m(x).last_hidden_state


def test_dropout_layers_follow_their_own_mode():
    """Dropout layers put in training mode under an evaluating tower (Monte-Carlo dropout), and the other way round."""
    for tower_trains in (False, True):
        eager, m = towers.bert(dropout=0.5), use_kernels(towers.bert(dropout=0.5))
        for t in (eager, m):
            t.train(tower_trains)
            for layer in t.modules():
                if isinstance(layer, torch.nn.Dropout):
                    layer.train(not tower_trains)
        for seed in (5, 6):
            same(outputs(eager, ids(), seed), outputs(m, ids(), seed))
        assert torch.equal(outputs(m, ids(), 5), outputs(m, ids(), 6)) == tower_trains
