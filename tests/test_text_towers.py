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


def _pairs():
    """(eager, on the operators, the input) of both kinds of tower."""
    x = torch.randn(5, 2, 64, generator=torch.Generator().manual_seed(4))
    return [(towers.bert().eval(), towers.bert().eval(), ids()), (towers.clip_block().eval(), towers.clip_block().eval(), x)]


def _hook_everything(m, into):
    for name, layer in m.named_modules():
        if name:
            layer.register_forward_hook(lambda mod, args, out, name=name: into.append((name, (out[0] if isinstance(out, tuple) else out).detach())) if not hasattr(out, "keys") else None)


@pytest.mark.parametrize("when", ["before", "after"])
@pytest.mark.parametrize("which", [0, 1])
def test_forward_hooks_fire_with_the_layers_own_values(which, when):
    eager, m, x = _pairs()[which]
    seen = [[], []]
    _hook_everything(eager, seen[0])
    if when == "before":
        _hook_everything(m, seen[1])
    use_kernels(m)
    if when == "after":
        _hook_everything(m, seen[1])
    with torch.no_grad():
        eager(x)
        m(x)
    assert [n for n, _ in seen[0]] == [n for n, _ in seen[1]]
    for (_, a), (_, b) in zip(*seen):
        same(a, b)


HOOKED = [(0, "encoder.layer.0.intermediate.dense"), (0, "encoder.layer.0.intermediate.intermediate_act_fn"), (0, "encoder.layer.1.output.dense"),
          (0, "encoder.layer.1.output.dropout"), (0, "encoder.layer.0.attention.output.dense"), (0, "pooler.dense"), (0, "pooler.activation"), (1, "mlp"), (1, "mlp.c_fc"),
          (1, "mlp.gelu"), (1, "mlp.c_proj")]


@pytest.mark.parametrize("kind", ["register_forward_pre_hook", "register_forward_hook", "register_full_backward_pre_hook", "register_full_backward_hook"])
@pytest.mark.parametrize("which,name", HOOKED)
def test_every_kind_of_hook_on_one_layer(which, name, kind):
    """A hook on a single layer of a fused block, and its results once it is removed again."""
    eager, m, x = _pairs()[which]
    use_kernels(m)
    seen = [[], []]
    flat = lambda v: [t.detach() for t in v if isinstance(t, torch.Tensor)] if isinstance(v, tuple) else [v.detach()]
    handles = [getattr(t.get_submodule(name), kind)(lambda mod, *vs, into=into: into.append([flat(v) for v in vs])) for t, into in zip((eager, m), seen)]
    y = [t(x) for t in (eager, m)]
    for v in y:
        (v if which else v.pooler_output).square().sum().backward()
    assert len(seen[0]) == len(seen[1]) == 1
    for a, b in zip(seen[0][0], seen[1][0]):
        assert len(a) == len(b)
        for u, v in zip(a, b):
            assert torch.allclose(u, v, rtol=1e-4, atol=1e-5)
    for h in handles:
        h.remove()
    with torch.no_grad():
        a, b = eager(x), m(x)
        same(a if which else a.pooler_output, b if which else b.pooler_output)
    assert len(seen[1]) == 1


@pytest.mark.parametrize("which", [0, 1])
def test_hooks_on_every_module_of_the_process(which):
    from torch.nn.modules.module import register_module_forward_hook
    eager, m, x = _pairs()[which]
    use_kernels(m)
    names = [{id(v): n for n, v in t.named_modules()} for t in (eager, m)]
    calls = []
    handle = register_module_forward_hook(lambda mod, args, out: calls.append(id(mod)))
    try:
        with torch.no_grad():
            eager(x)
            first = [names[0][i] for i in calls]
            calls.clear()
            m(x)
            assert [names[1][i] for i in calls] == first
    finally:
        handle.remove()


class Adapter(torch.nn.Module):
    """A layer a user puts around a dense one."""
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x):
        return self.inner(x) + 0.5 * x.mean(-1, keepdim=True)


def _adapt(m, name, change):
    block, child = m.get_submodule(name.rpartition(".")[0]) if "." in name else m, name.rpartition(".")[2]
    setattr(block, child, change(getattr(block, child)))


CHANGES = [(0, "encoder.layer.0.intermediate.dense", Adapter), (0, "encoder.layer.1.output.dense", Adapter), (0, "pooler.dense", Adapter),
           (0, "encoder.layer.0.intermediate.intermediate_act_fn", lambda old: torch.nn.ReLU()), (0, "encoder.layer.0.intermediate.intermediate_act_fn", lambda old: torch.nn.Softplus()),
           (0, "pooler.activation", lambda old: torch.nn.GELU(approximate="tanh")), (0, "encoder.layer.1.output.dropout", Adapter),
           (1, "mlp.c_fc", Adapter), (1, "mlp.c_proj", Adapter), (1, "mlp.gelu", lambda old: torch.nn.SiLU()),
           (1, "mlp", lambda old: torch.nn.Sequential(*old, torch.nn.Tanh())), (1, "mlp", Adapter)]


@pytest.mark.parametrize("again", [False, True])
@pytest.mark.parametrize("i", range(len(CHANGES)), ids=["%s-%d" % (c[1], i) for i, c in enumerate(CHANGES)])
def test_layers_exchanged_after_use_kernels(i, again):
    which, name, change = CHANGES[i]
    eager, m, x = _pairs()[which]
    use_kernels(m)
    for t in (eager, m):
        _adapt(t, name, change)
    if again:
        use_kernels(m)
    with torch.no_grad():
        a, b = eager(x), m(x)
    same(a if which else a.last_hidden_state, b if which else b.last_hidden_state)
    if not which:
        same(a.pooler_output, b.pooler_output)


@pytest.mark.parametrize("name", ["encoder.layer.0.intermediate", "encoder.layer.1.output", "pooler"])
def test_a_blocks_own_forward_is_kept(name):
    """Packages that place a module's calls put a function of their own into the module as ``forward``."""
    m, calls = towers.bert().eval(), []
    block = m.get_submodule(name)
    inner = block.forward
    block.forward = lambda *a: calls.append(name) or inner(*a)
    kept = block.forward
    use_kernels(m)
    use_kernels(m)
    assert block.forward is kept
    with torch.no_grad():
        same(m(ids()).pooler_output, towers.bert().eval()(ids()).pooler_output)
    assert calls == [name]


def test_layers_with_a_forward_of_their_own_inside_a_block():
    eager, m, x = _pairs()[1]
    use_kernels(m)
    for t in (eager, m):
        t.mlp.gelu.forward = lambda z: z.clamp(min=0)
    with torch.no_grad():
        same(eager(x), m(x))


@pytest.mark.parametrize("which,name", [(0, "encoder.layer.0.intermediate"), (0, "encoder.layer.1.output"), (0, "pooler"), (1, "")])
def test_replicas_call_their_own_layers(which, name):
    """What torch.nn.parallel.replicate does to a module: a copy of its attributes, whose children and parameters are then exchanged."""
    _, m, x = _pairs()[which]
    use_kernels(m)
    block = m.get_submodule(name)
    torch.manual_seed(9)
    args = [torch.randn(4, 3, 200 if name.endswith("output") else 64 if which else 96)] + [torch.randn(4, 3, 96)] * name.endswith("output")
    with torch.no_grad():
        before = block(*args)
        other = block._replicate_for_data_parallel()._replicate_for_data_parallel()
        for child in ("mlp",) if which else ("dense",):
            old = getattr(other, child)
            new = use_kernels(towers.clip_block()).mlp if which else type(old)(old.in_features, old.out_features)
            for p in new.parameters():
                p.normal_()
            other._modules = dict(other._modules)
            other._modules[child] = new
        after = other(*args)
        assert torch.equal(block(*args), before) and not torch.allclose(after, before, atol=1e-2)
        same(after, type(other).forward(other, *args))


class BertOutput(torch.nn.Module):
    """Not the package's: the same name and layers in another order."""
    def __init__(self):
        super().__init__()
        self.dense, self.LayerNorm, self.dropout = torch.nn.Linear(24, 24), torch.nn.LayerNorm(24), torch.nn.Dropout(0.0)

    def forward(self, hidden_states, input_tensor):
        return self.dropout(self.dense(self.LayerNorm(hidden_states))) + input_tensor


def test_blocks_of_other_packages_keep_their_forward():
    a, b = torch.randn(2, 5, 24)
    torch.manual_seed(3)
    eager = BertOutput()
    torch.manual_seed(3)
    m = use_kernels(BertOutput())
    with torch.no_grad():
        same(eager(a, b), m(a, b))
    # CLIP's block is known by its structure (several packages carry it): one whose forward takes more is not it
    block = towers.clip_block()
    type(block).forward = lambda self, x, mask=None: x + self.mlp(self.ln_2(x))
    x = torch.randn(5, 2, 64)
    with torch.no_grad():
        want = block(x)
        same(use_kernels(block)(x), want)
        same(block(x, mask=None), want)


def test_a_tower_of_a_type_without_kernels_is_refused_as_a_whole():
    m = towers.bert().double()
    kinds = [type(v) for v in m.modules()]
    with pytest.raises(ValueError, match="float64"):
        use_kernels(m)
    assert [type(v) for v in m.modules()] == kinds and not any("forward" in vars(v) for v in m.modules())
    mixed = torch.nn.Sequential(torch.nn.Linear(4, 4), torch.nn.LayerNorm(4, dtype=torch.float64))
    with pytest.raises(ValueError, match="float64"):
        use_kernels(mixed)
    assert type(mixed[0]) is torch.nn.Linear
    assert use_kernels(torch.nn.Sequential(torch.nn.Linear(4, 4), torch.nn.LayerNorm(4, elementwise_affine=False))) is not None
