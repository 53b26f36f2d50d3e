"""The text towers' layers on the operators of ``lsdm_amd.ops``.

The path's text features come from a third-party tower (model/sdm.py:146-149, 245-285: the ``clip`` package's text transformer or ``transformers``'
BERT), which runs on eager layers.  ``use_kernels(tower)`` puts this library's dense layers and layer norms under such a tower -- or any module built
of ``nn.Linear`` and ``nn.LayerNorm`` -- in place: parameters, names and ``state_dict`` stay as they are, and it can be trained as before.

    tower = transformers.BertModel.from_pretrained("bert-base-uncased").to("cuda")
    use_kernels(tower)                       # inference
    use_kernels(tower, checkpoint8=True)     # fine-tuning with what the backward pass reads kept in 8 bits (bfloat16 / float16 towers)

``SceneDiffusionModel(..., text_kernels=True)`` does it for the tower the model loads itself.  What a block lets be fused is: BERT's
``dense -> activation`` and ``dense -> + input -> LayerNorm``, its pooler, and CLIP's ``x + c_proj(gelu(c_fc(ln_2(x))))``; everything else is replaced
layer by layer, and attention itself stays with the package.  A block whose layers carry hooks runs unfused, so that they see what they always saw.
Autocast does not reach the operators: give the tower the type instead (a call that mixes types raises ``ValueError``).
"""
import functools

import torch.nn as nn
from torch.nn.modules.module import _has_any_global_hook

from . import ops

# activation modules whose function ops.linear has in its epilogue
_ACT_BY_CLASS = {"GELUActivation": "gelu", "GELU": "gelu", "QuickGELU": "quick_gelu", "QuickGELUActivation": "quick_gelu", "SiLU": "silu", "SiLUActivation": "silu",
                 "ReLU": "relu", "Sigmoid": "sigmoid", "Tanh": "tanh"}


# the blocks that are fused, by class and children
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


def _hooked(*modules):
    """Whether someone looks at these layers' calls: a fused block leaves some of them out and gives others' results with more in them, so it runs its own
    ``forward`` then."""
    return _has_any_global_hook() or any(m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks for m in modules)


def _dense_act(self, hidden_states):
    if _hooked(self.dense, self.intermediate_act_fn):
        return type(self).forward(self, hidden_states)
    return self.dense(hidden_states, self._kernel_activation)


def _dense_residual_norm(self, hidden_states, input_tensor):
    drop = self.dropout                                            # it sits between the product and the sum, and its own mode says whether it drops
    if type(drop) is not nn.Dropout or (drop.training and drop.p > 0) or _hooked(self.dense, drop):
        return type(self).forward(self, hidden_states, input_tensor)
    return self.LayerNorm(self.dense(hidden_states, residual=input_tensor))


def _pooler(self, hidden_states):
    if _hooked(self.dense, self.activation):
        return type(self).forward(self, hidden_states)
    return self.dense(hidden_states[:, 0], self._kernel_activation)


def _clip_block(self, x):
    if _hooked(self.mlp, *self.mlp):
        return type(self).forward(self, x)
    x = x + self.attention(self.ln_1(x))
    return self.mlp.c_proj(self.mlp.c_fc(self.ln_2(x), self._kernel_activation), residual=x)


def _fuse(module):
    """Replaces the ``forward`` of a block whose layers form one of the fused patterns: exactly these children, the dense layers among them replaced above (a
    subclass of ``nn.Linear``, or a further layer in the block, keeps the block's own ``forward``)."""
    name, children = type(module).__name__, dict(module.named_children())
    mlp = dict(children["mlp"].named_children()) if "mlp" in children else {}
    if set(children) != _BLOCKS.get(name) or any(type(c) is not Linear for n, c in [*children.items(), *mlp.items()] if n in _DENSE):
        return
    if name == "BertIntermediate":
        act = _activation_name(module.intermediate_act_fn)
        forward = _dense_act
    elif name in ("BertSelfOutput", "BertOutput"):
        act, forward = "none", _dense_residual_norm
    elif name == "BertPooler":
        act, forward = _activation_name(module.activation), _pooler
    elif name == "ResidualAttentionBlock" and hasattr(module, "attention") and list(mlp) == ["c_fc", "gelu", "c_proj"]:
        act, forward = _activation_name(module.mlp.gelu), _clip_block
    else:
        return
    if act is not None:
        module._kernel_activation = act
        module.forward = functools.partial(forward, module)       # (copies and pickles with the module, as a bound method would not)


def use_kernels(tower, *, checkpoint8=False):
    """Puts the operators under ``tower``'s layers, in place; returns ``tower``.  Layers of other kinds are left as they are.  Raises ``ValueError`` if
    there is nothing to replace."""
    found = 0
    for module in tower.modules():
        kind = type(module)
        if kind in (nn.Linear, Linear):
            module.__class__ = Linear
        elif kind in (nn.LayerNorm, LayerNorm) or (isinstance(module, nn.LayerNorm) and kind.__module__.split(".")[0] == "clip"):
            if len(module.normalized_shape) != 1 or module.normalized_shape[0] > ops.NORM_MAX_WIDTH:
                continue
            module.__class__ = LayerNorm
        else:
            continue
        module.checkpoint8 = checkpoint8
        found += 1
    if not found:
        raise ValueError("use_kernels: no Linear or LayerNorm layer in %s" % type(tower).__name__)
    for module in tower.modules():
        _fuse(module)
    return tower
