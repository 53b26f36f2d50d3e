"""Operators of the text towers on the HIP device: dense layer with epilogue, layer norm, 8-bit activation checkpoints.

``linear(x, weight, bias, activation, residual)``   ``a(x @ weight.T + bias) + residual`` in one launch, with its backward pass
``layer_norm(x, weight, bias, eps)``                layer norm over the last axis, with its backward pass
``checkpoint8(x)`` -> ``Checkpoint8``, ``.restore()`` a tensor in 33/32 bytes per value; ``checkpoint8=True`` of the two above keeps what their
                                                    backward passes read in that form

They run in ``liblsdm_hip.so`` (include/lsdm_hip.h: ``lsdm_linear*``, ``lsdm_layer_norm*``, ``lsdm_pack8``, ``lsdm_unpack8``) on the current stream of
the tensors' device (argument checks, allocation and autograd nodes: csrc/torch_ops.cpp); host tensors raise ``LsdmError``.
``lsdm_amd.text.use_kernels`` puts them under a CLIP / BERT tower.

Types: float32, bfloat16, float16, the same for all tensors of a call (``bias`` and the norm's ``weight`` / ``bias`` may also be float32).  Products
accumulate and everything else is evaluated in 32 bits; results are rounded once.  In 16 bits the backward pass of ``linear`` rounds dz = dy a'(z) to the
tensors' type, as the matrix cores take their operands in it (a'(z) itself is kept in 16 bits that round it by 2^-14 of its value near 1,
2^-13 at 1/16 and 2^-8 at 1e-7).
Shapes: any leading axes, any sizes including 0 rows (at most 2^30 rows and columns, 2^25 rows of ``weight``, 2^35 values of a checkpoint); the last axis
should be contiguous (other layouts are copied first).
Gradients are differentiable once; forward-mode derivatives there are none (a dual tensor raises ``LsdmError``).  Results do not depend on timing (no
atomics): the same call gives the same bits.

8-bit checkpoints: groups of 32 consecutive values of a row share a power-of-two step 2^e (e = max(floor(log2 max|x|) - 6, -126)); a value is kept
as the int8 nearest to x / 2^e.  What is restored is exact in x's own type, bfloat16 and float32 (in float16 values of another type may lie outside its
range); a group that holds an infinity or a NaN comes back as NaN, so an overflow is never hidden.  ``linear(..., checkpoint8=True)`` keeps ``x`` in this
form and a'(z) as one byte (step 1/192, exact at 0 and 1); ``layer_norm(..., checkpoint8=True)`` keeps the normalised rows.  This is what is held between
the passes: ``linear``'s backward pass restores one layer's ``x`` in full width as scratch memory while it runs.  Codes taken from computed values flip on
their last bit, which float32 gradients would show: in float32 ``linear`` keeps a'(z) in 32 bits, and ``layer_norm`` refuses ``checkpoint8``.

Tracers (``torch.jit.trace``, ``make_fx``, fake tensors) do not see what the kernels write: such calls raise ``LsdmError``.
HIP graphs: forward and backward passes can be captured.  A leaf whose gradient node is held by a live autograd graph built eagerly on the default
stream cannot take part in a capture (the runtime would have to join the default stream to it), whether it is an input itself or stands behind one: such a
call raises ``LsdmError``.
"""
import torch

from . import _lib

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "quick_gelu": 3, "silu": 4, "sigmoid": 5, "tanh": 6}
NORM_MAX_WIDTH = 16384


class Checkpoint8:
    """A tensor kept in 8 bits: ``codes`` int8 (rows, width), ``exps`` uint8 (rows, ceil(width / 32)), its ``shape`` and ``dtype``."""
    __slots__ = ("codes", "exps", "shape", "dtype")

    def __init__(self, codes, exps, shape, dtype):
        self.codes, self.exps, self.shape, self.dtype = codes, exps, shape, dtype

    def restore(self, dtype=None):
        """-> the values the checkpoint stands for, as a tensor of the original shape (``dtype``: the original's by default)."""
        return _lib.load_torch_ops().unpack8(self.codes, self.exps, self.shape, self.dtype if dtype is None else dtype)


def checkpoint8(x):
    """``x`` (..., width) -> ``Checkpoint8``.  The groups run along the last axis.  Not differentiable: it stores values."""
    codes, exps = _lib.load_torch_ops().pack8(x)
    return Checkpoint8(codes, exps, x.shape, x.dtype)


def linear(x, weight, bias=None, activation="none", residual=None, *, checkpoint8=False):
    """``a(x @ weight.T + bias) + residual``: x (..., K), weight (N, K), bias (N) or None, residual (..., N) or None -> (..., N).

    ``activation``: one of ``ACTIVATIONS`` or None.  ``checkpoint8``: keep ``x`` and a'(z) in 8 bits for the backward pass (the module docstring)."""
    act = 0 if activation is None else ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError("linear: activation must be one of %s, got %r" % (sorted(ACTIVATIONS), activation))
    return _lib.load_torch_ops().linear(x, weight, bias, act, residual, bool(checkpoint8))


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, checkpoint8=False):
    """Layer norm over the last axis: x (..., D), weight / bias (D) or None -> (..., D); D <= 16384.  Rows of any finite values (their squares need not fit
    the type); a row that holds an infinity or a NaN is NaN.

    ``checkpoint8`` (bfloat16 / float16): keep the normalised rows in 8 bits for the backward pass (the module docstring)."""
    return _lib.load_torch_ops().layer_norm(x, weight, bias, eps, bool(checkpoint8))
