"""The text towers' layers on the operators of ``lsdm_amd.ops``.

The path's text features come from a third-party tower (model/sdm.py:146-149, 245-285: the ``clip`` package's text transformer or ``transformers``'
BERT), which runs on eager layers.  ``use_kernels(tower)`` puts this library's dense layers and layer norms under such a tower -- or any module built
of ``nn.Linear`` and ``nn.LayerNorm`` -- in place: parameters, names and ``state_dict`` stay as they are, and it can be trained as before.

    tower = transformers.BertModel.from_pretrained("bert-base-uncased").to("cuda")
    use_kernels(tower)                       # inference
    use_kernels(tower, checkpoint8=True)     # fine-tuning with what the backward pass reads kept in 8 bits (bfloat16 / float16 towers)

``SceneDiffusionModel(..., text_kernels=True)`` does it for the tower the model loads itself.  What a block lets be fused is: BERT's
``dense -> activation`` and ``dense -> + input -> LayerNorm``, its pooler, and CLIP's ``x + c_proj(gelu(c_fc(ln_2(x))))``; everything else is replaced
layer by layer, and attention itself stays with the package.  A block whose layers carry hooks or were exchanged since runs its own ``forward``.
Autocast does not reach the operators: give the tower the type instead (a call that mixes types raises ``ValueError``).
bfloat16 towers and short prompt lists gain (BERT of 12 layers: 0.4 to 0.7 of the eager time); a float32 tower over 64 prompts and more takes 4 to 16 %
longer than eager.
"""
import functools
import inspect

import torch.nn as nn
from torch.nn.modules.module import _has_any_global_hook

from . import ops

# activation modules whose function ops.linear has in its epilogue
_ACT_BY_CLASS = {"GELUActivation": "gelu", "GELU": "gelu", "QuickGELU": "quick_gelu", "QuickGELUActivation": "quick_gelu", "SiLU": "silu", "SiLUActivation": "silu",
                 "ReLU": "relu", "Sigmoid": "sigmoid", "Tanh": "tanh"}


# the blocks that are fused, by class and children: BERT's of ``transformers``; CLIP's of any package that carries it, known by its ``forward(x)`` as well
_BLOCKS = {"BertIntermediate": {"dense", "intermediate_act_fn"}, "BertSelfOutput": {"dense", "LayerNorm", "dropout"}, "BertOutput": {"dense", "LayerNorm", "dropout"},
           "BertPooler": {"dense", "activation"}, "ResidualAttentionBlock": {"attn", "ln_1", "mlp", "ln_2"}}
_DENSE = ("dense", "c_fc", "c_proj")


def _activation_name(module):
    if getattr(module, "approximate", "none") != "none":          # nn.GELU(approximate="tanh") is another function
        return None
    return _ACT_BY_CLASS.get(type(module).__name__)


class Linear(nn.Linear):
    """``nn.Linear`` evaluated by ``ops.linear``."""
    checkpoint8 = False

    def forward(self, x, activation="none", residual=None):
        return ops.linear(x, self.weight, self.bias, activation, residual, checkpoint8=self.checkpoint8)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last axis evaluated by ``ops.layer_norm`` (half-precision rows with float32 parameters included)."""
    checkpoint8 = False

    def forward(self, x):
        return ops.layer_norm(x, self.weight, self.bias, self.eps, checkpoint8=self.checkpoint8)


def _plain(*modules):
    """Whether nobody looks at or changes these layers' calls (hooks, a ``forward`` put into the module): a fused block leaves some of them out and gives
    others' results with more in them, so it runs its own ``forward`` where this is false."""
    return not (_has_any_global_hook() or any(m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks or "forward" in vars(m) for m in modules))


# The fused forms ask at every call whether the block still holds what was fused: layers are exchanged (adapters, quantised layers) and hooked at any time.
def _dense_act(self, hidden_states):
    dense, act = self.dense, self.intermediate_act_fn
    if type(dense) is not Linear or _activation_name(act) != self._kernel_activation or not _plain(dense, act):
        return type(self).forward(self, hidden_states)
    return dense(hidden_states, self._kernel_activation)


def _dense_residual_norm(self, hidden_states, input_tensor):
    dense, drop = self.dense, self.dropout                         # the dropout sits between the product and the sum, and its own mode says whether it drops
    if type(dense) is not Linear or type(drop) is not nn.Dropout or (drop.training and drop.p > 0) or not _plain(dense, drop):
        return type(self).forward(self, hidden_states, input_tensor)
    return self.LayerNorm(dense(hidden_states, residual=input_tensor))


def _pooler(self, hidden_states):
    dense, act = self.dense, self.activation
    if type(dense) is not Linear or _activation_name(act) != self._kernel_activation or not _plain(dense, act):
        return type(self).forward(self, hidden_states)
    return dense(hidden_states[:, 0], self._kernel_activation)


_MLP = ["c_fc", "gelu", "c_proj"]


def _clip_block(self, x):
    mlp = self.mlp
    layers = [*mlp._modules.values()]
    if (type(mlp) is not nn.Sequential or [*mlp._modules] != _MLP or type(layers[0]) is not Linear or type(layers[2]) is not Linear
            or _activation_name(layers[1]) != self._kernel_activation or not _plain(mlp, *layers)):
        return type(self).forward(self, x)
    x = x + self.attention(self.ln_1(x))
    return layers[2](layers[0](self.ln_2(x), self._kernel_activation), residual=x)


_FUSED = (_dense_act, _dense_residual_norm, _pooler, _clip_block)


def _put(module, forward):
    module.forward = functools.partial(forward, module)           # (copies and pickles with the module, as a bound method would not)
    module._replicate_for_data_parallel = functools.partial(_replicate, module)


def _replicate(module):
    """A replica's attributes are copied one by one, the module inside ``forward`` would stay the original."""
    replica = type(module)._replicate_for_data_parallel(module)
    _put(replica, module.forward.func)
    return replica


def _fuse(module):
    """Replaces the ``forward`` of a block whose layers form one of the fused patterns: exactly these children, the dense layers among them replaced above (a
    subclass of ``nn.Linear``, a further layer in the block, or a ``forward`` that someone put into the module keeps the block as it is)."""
    name, children, own = type(module).__name__, dict(module.named_children()), vars(module).get("forward")
    if isinstance(own, functools.partial) and own.func in _FUSED:
        for attribute in ("forward", "_replicate_for_data_parallel"):     # an earlier call's: the block may have changed since
            vars(module).pop(attribute, None)
    elif own is not None:
        return
    mlp = dict(children["mlp"].named_children()) if "mlp" in children else {}
    if name == "ResidualAttentionBlock":
        if list(inspect.signature(type(module).forward).parameters) != ["self", "x"]:
            return
    elif type(module).__module__.split(".")[0] != "transformers":
        return
    if set(children) != _BLOCKS.get(name) or any(type(c) is not Linear for n, c in [*children.items(), *mlp.items()] if n in _DENSE):
        return
    if name == "BertIntermediate":
        act = _activation_name(module.intermediate_act_fn)
        forward = _dense_act
    elif name in ("BertSelfOutput", "BertOutput"):
        act, forward = "none", _dense_residual_norm
    elif name == "BertPooler":
        act, forward = _activation_name(module.activation), _pooler
    elif name == "ResidualAttentionBlock" and hasattr(module, "attention") and list(mlp) == _MLP:
        act, forward = _activation_name(module.mlp.gelu), _clip_block
    else:
        return
    if act is not None:
        module._kernel_activation = act
        _put(module, forward)


def _layer_class(module):
    """The class that takes ``module``'s place, or None."""
    kind = type(module)
    if kind in (nn.Linear, Linear):
        return Linear
    if kind in (nn.LayerNorm, LayerNorm) or (isinstance(module, nn.LayerNorm) and kind.__module__.split(".")[0] == "clip"):
        return LayerNorm if len(module.normalized_shape) == 1 and module.normalized_shape[0] <= ops.NORM_MAX_WIDTH else None
    return None


def use_kernels(tower, *, checkpoint8=False):
    """Puts the operators under ``tower``'s layers, in place; returns ``tower``.  Layers of other kinds are left as they are.  Raises ``ValueError``, and
    changes nothing, if there is nothing to replace or a layer's parameters have a type that the operators do not take (float64)."""
    found = [(module, _layer_class(module)) for module in tower.modules() if _layer_class(module)]
    if not found:
        raise ValueError("use_kernels: no Linear or LayerNorm layer in %s" % type(tower).__name__)
    for module, kind in found:
        if module.weight is not None and module.weight.dtype not in ops.DTYPES:
            raise ValueError("use_kernels: a %s layer holds %s parameters; the operators take float32, bfloat16 and float16" % (kind.__name__, module.weight.dtype))
    for module, kind in found:
        module.__class__ = kind
        module.checkpoint8 = checkpoint8
    for module in tower.modules():
        _fuse(module)
    return tower
