"""Operators of the text towers on the HIP device: dense layer with epilogue, layer norm, 8-bit activation checkpoints.

``linear(x, weight, bias, activation, residual)``   ``a(x @ weight.T + bias) + residual`` in one launch, with its backward pass
``layer_norm(x, weight, bias, eps)``                layer norm over the last axis, with its backward pass
``checkpoint8(x)`` -> ``Checkpoint8``, ``.restore()`` a tensor in 33/32 bytes per value; ``checkpoint8=True`` of the two above keeps what their
                                                    backward passes read in that form

They run in ``liblsdm_hip.so`` (include/lsdm_hip.h: ``lsdm_linear*``, ``lsdm_layer_norm*``, ``lsdm_pack8``, ``lsdm_unpack8``) on the current stream of
the tensors' device; host tensors raise ``LsdmError``.  ``lsdm_amd.text.use_kernels`` puts them under a CLIP / BERT tower.

Types: float32, bfloat16, float16, the same for all tensors of a call (``bias`` and the norm's ``weight`` / ``bias`` may also be float32).  Products
accumulate and everything else is evaluated in 32 bits; results are rounded once.  In 16 bits two more roundings are part of the backward pass of
``linear``: a'(z) is kept in the tensors' type, and dz = dy a'(z) is rounded to it, as the matrix cores take their operands in that type.
Shapes: any leading axes, any sizes including 0 rows; the last axis should be contiguous (other layouts are copied first).
Gradients are differentiable once.  Results do not depend on timing (no atomics): the same call gives the same bits.

8-bit checkpoints: groups of 32 consecutive values of a row share a power-of-two step 2^e (e = max(floor(log2 max|x|) - 6, -126)); a value is kept
as the int8 nearest to x / 2^e.  What is restored is exact in every type; a group that holds an infinity or a NaN comes back as NaN, so an overflow
is never hidden.  ``linear(..., checkpoint8=True)`` keeps ``x`` in this form and a'(z) as one byte (step 1/192, exact at 0 and 1);
``layer_norm(..., checkpoint8=True)`` keeps the normalised rows.  Codes taken from computed values flip on their last bit, which float32 gradients
would show: in float32 ``linear`` keeps a'(z) in 32 bits, and ``layer_norm`` refuses ``checkpoint8``.

HIP graphs: forward and backward passes can be captured.  A leaf whose gradient node is held by a live autograd graph built eagerly on the default
stream cannot take part in a capture (the runtime would have to join the default stream to it): such a call raises ``LsdmError``.
"""
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "quick_gelu": 3, "silu": 4, "sigmoid": 5, "tanh": 6}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_PARAM_F32, _DERIV8, _BACKWARD, _DX, _DW, _DB, _DERIV, _CODES, _X_UN, _W_UN, _DY_UN = (1 << i for i in range(11))   # lsdm_hip.h: LSDM_OP_*
NORM_MAX_WIDTH = 16384
_MAX_SIZE = 1 << 30


def _call(name, *args):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    if rc != 0:
        raise _lib.LsdmError("%s failed (%d): %s" % (name, rc, lib.lsdm_last_error(None).decode()))


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _check_tensors(who, x, **others):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise _lib.LsdmError("%s runs in liblsdm_hip.so on HIP device tensors; got %s" % (who, getattr(x, "device", type(x).__name__)))
    if x.dtype not in _DTYPES:
        raise ValueError("%s: dtype must be float32, bfloat16 or float16, got %s" % (who, x.dtype))
    for name, t in others.items():
        if t is not None and t.device != x.device:
            raise _lib.LsdmError("%s: %s is on %s, x on %s" % (who, name, t.device, x.device))


def _rows(t, width):
    """-> (2-D tensor with unit stride along its rows, row stride); copies only what no row stride can describe."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    ld = t.stride(0)
    if t.stride(1) == 1 and ld >= width:
        return t, ld
    t = t.contiguous()
    return t, width


def _unaligned(t, ld, width):
    es = t.element_size()
    return bool((t.data_ptr() | ld * es | width * es) & 15)


@functools.lru_cache(maxsize=4096)
def _linear_bytes(dtype, flags, M, N, K):
    n = _lib.load().lsdm_linear_workspace(dtype, flags, M, N, K)
    if n < 0:
        raise _lib.LsdmError("lsdm_linear_workspace failed (%d): %s" % (n, _lib.load().lsdm_last_error(None).decode()))
    return n


def _scratch(nbytes, like):
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


# ------------------------------------------------------------------------------------------------ 8-bit checkpoints
class Checkpoint8:
    """A tensor kept in 8 bits: ``codes`` int8 (rows, width), ``exps`` uint8 (rows, ceil(width / 32)), its ``shape`` and ``dtype``."""
    __slots__ = ("codes", "exps", "shape", "dtype")

    def __init__(self, codes, exps, shape, dtype):
        self.codes, self.exps, self.shape, self.dtype = codes, exps, shape, dtype

    def restore(self, dtype=None):
        """-> the values the checkpoint stands for, as a tensor of the original shape (``dtype``: the original's by default)."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _DTYPES:
            raise ValueError("Checkpoint8.restore: dtype must be float32, bfloat16 or float16, got %s" % dtype)
        out = torch.empty(self.shape, dtype=dtype, device=self.codes.device)
        if out.numel():
            rows, width = self.codes.shape
            _call("lsdm_unpack8", out.device.index, _DTYPES[dtype], rows, width, self.codes.data_ptr(), self.exps.data_ptr(), out.data_ptr(), _stream(out))
        return out


def _pack8(x2, ld, width):
    rows = x2.shape[0]
    codes = torch.empty((rows, width), dtype=torch.int8, device=x2.device)
    exps = torch.empty((rows, (width + 31) // 32), dtype=torch.uint8, device=x2.device)
    if codes.numel():
        _call("lsdm_pack8", x2.device.index, _DTYPES[x2.dtype], rows, width, x2.data_ptr(), ld, codes.data_ptr(), exps.data_ptr(), _stream(x2))
    return codes, exps


def checkpoint8(x):
    """``x`` (..., width) -> ``Checkpoint8``.  The groups run along the last axis.  Not differentiable: it stores values."""
    _check_tensors("checkpoint8", x)
    if x.dim() < 1:
        raise ValueError("checkpoint8: a tensor of at least one axis is needed")
    if x.shape[-1] > _MAX_SIZE:
        raise ValueError("checkpoint8: the last axis may hold at most 2^30 values")
    if x.numel() == 0:
        width = x.shape[-1]
        rows = x.numel() // width if width else 0
        return Checkpoint8(torch.empty((rows, width), dtype=torch.int8, device=x.device), torch.empty((rows, (width + 31) // 32), dtype=torch.uint8, device=x.device),
                           x.shape, x.dtype)
    with torch.no_grad():
        x2, ld = _rows(x.detach(), x.shape[-1])
        return Checkpoint8(*_pack8(x2, ld, x.shape[-1]), x.shape, x.dtype)


# ------------------------------------------------------------------------------------------------ linear
def _linear_forward(x2, ldx, weight, ldw, bias, act, residual, want_deriv, deriv8):
    M, K = x2.shape
    N = weight.shape[0]
    y = torch.empty((M, N), dtype=x2.dtype, device=x2.device)
    deriv = torch.empty((M, N), dtype=torch.uint8 if deriv8 else x2.dtype, device=x2.device) if want_deriv else None
    if M == 0 or N == 0:
        return y, deriv
    dt = _DTYPES[x2.dtype]
    flags = (_PARAM_F32 if bias is not None and bias.dtype == torch.float32 else 0) | (_DERIV8 if deriv8 else 0)
    ldr = 0
    if residual is not None:
        residual, ldr = _rows(residual, N)
    ws = None
    nbytes = 0
    if M > 64:                      # (lsdm_linear needs no scratch memory for few rows)
        nbytes = _linear_bytes(dt, flags | (_X_UN if _unaligned(x2, ldx, K) else 0) | (_W_UN if _unaligned(weight, ldw, K) else 0), M, N, K)
        ws = _scratch(nbytes, x2)
    _call("lsdm_linear", x2.device.index, dt, act, flags, M, N, K, x2.data_ptr(), ldx, weight.data_ptr(), ldw, _ptr(bias), _ptr(residual), ldr, y.data_ptr(),
          _ptr(deriv), _ptr(ws), nbytes, _stream(x2))
    return y, deriv


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, checkpoint):
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        K, N = weight.shape[1], weight.shape[0]
        x2, ldx = _rows(x, K)
        w2, ldw = _rows(weight, K)
        b = bias.contiguous() if bias is not None else None
        inner = need_x or need_w or need_b
        deriv8 = checkpoint and x.dtype != torch.float32
        y, deriv = _linear_forward(x2, ldx, w2, ldw, b, act, residual, inner and act != 0, deriv8)
        codes = exps = None
        if need_w and checkpoint:
            codes, exps = _pack8(x2, ldx, K)
        ctx.save_for_backward(x if need_w and not checkpoint else None, codes, exps, weight if need_x else None, deriv)
        ctx.shapes = (x.shape, weight.shape, y.shape[0])
        ctx.bias_dtype = bias.dtype if bias is not None else x.dtype
        ctx.deriv8, ctx.inner = deriv8, inner
        return y.view(x.shape[:-1] + (N,))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if ctx.inner:
            x, codes, exps, weight, deriv = ctx.saved_tensors
            xshape, wshape, M = ctx.shapes
            N, K = wshape
            dt, dev = dy.dtype, dy.device
            new = torch.empty if M and N and K else torch.zeros
            dx = new(xshape, dtype=dt, device=dev) if need_x else None
            dw = new(wshape, dtype=dt, device=dev) if need_w else None
            db = (torch.empty if M and N else torch.zeros)(N, dtype=ctx.bias_dtype, device=dev) if need_b else None
            if M and N and K:
                dy2, lddy = _rows(dy, N)
                flags = (_PARAM_F32 if ctx.bias_dtype == torch.float32 else 0) | (_DERIV8 if ctx.deriv8 else 0)
                plan = flags | _BACKWARD | (_DX if need_x else 0) | (_DW if need_w else 0) | (_DB if need_b else 0) | (_DERIV if deriv is not None else 0) \
                    | (_CODES if codes is not None else 0) | (_DY_UN if _unaligned(dy2, lddy, N) else 0)
                x2 = w2 = None
                ldx = ldw = 0
                if x is not None:
                    x2, ldx = _rows(x, K)
                    plan |= _X_UN if _unaligned(x2, ldx, K) else 0
                if weight is not None:
                    w2, ldw = _rows(weight, K)
                    plan |= _W_UN if _unaligned(w2, ldw, K) else 0
                nbytes = _linear_bytes(_DTYPES[dt], plan, M, N, K)
                ws = _scratch(nbytes, dy2)
                _call("lsdm_linear_backward", dev.index, _DTYPES[dt], flags, M, N, K, dy2.data_ptr(), lddy, _ptr(deriv), _ptr(x2), ldx, _ptr(codes), _ptr(exps),
                      _ptr(w2), ldw, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nbytes, _stream(dy2))
        return dx, dw, db, (dy if need_r else None), None, None


def linear(x, weight, bias=None, activation="none", residual=None, *, checkpoint8=False):
    """``a(x @ weight.T + bias) + residual``: x (..., K), weight (N, K), bias (N) or None, residual (..., N) or None -> (..., N).

    ``activation``: one of ``ACTIVATIONS``.  ``checkpoint8``: keep ``x`` and a'(z) in 8 bits for the backward pass (the module docstring)."""
    _check_tensors("linear", x, weight=weight, bias=bias, residual=residual)
    act = ACTIVATIONS.get(activation if activation is not None else "none")
    if act is None:
        raise ValueError("linear: activation must be one of %s, got %r" % (sorted(ACTIVATIONS), activation))
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError("linear: expected x (..., K) and weight (N, K), got %s and %s" % (tuple(x.shape), tuple(weight.shape)))
    N, K = weight.shape
    if K < 1:
        raise ValueError("linear: weight has no columns")
    if weight.dtype != x.dtype or (residual is not None and residual.dtype != x.dtype):
        raise ValueError("linear: weight and residual must have x's dtype %s" % x.dtype)
    if bias is not None and (bias.shape != (N,) or bias.dtype not in (x.dtype, torch.float32)):
        raise ValueError("linear: bias must be (%d,) of dtype %s or float32, got %s %s" % (N, x.dtype, tuple(bias.shape), bias.dtype))
    if residual is not None and (residual.shape[:-1] != x.shape[:-1] or residual.shape[-1] != N):
        raise ValueError("linear: residual must have the result's shape %s, got %s" % (tuple(x.shape[:-1]) + (N,), tuple(residual.shape)))
    if x.numel() // K > _MAX_SIZE or N > _MAX_SIZE or K > _MAX_SIZE:
        raise ValueError("linear: at most 2^30 rows and columns")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, residual, act, bool(checkpoint8))
    x2, ldx = _rows(x, K)
    w2, ldw = _rows(weight, K)
    y, _ = _linear_forward(x2, ldx, w2, ldw, bias.contiguous() if bias is not None else None, act, residual, False, False)
    return y if x.dim() == 2 else y.view(x.shape[:-1] + (N,))


# ------------------------------------------------------------------------------------------------ layer norm
def _norm_forward(x2, ld, D, weight, bias, eps, keep, checkpoint):
    rows = x2.shape[0]
    y = torch.empty((rows, D), dtype=x2.dtype, device=x2.device)
    mean = rstd = codes = exps = None
    if keep:
        mean = torch.empty(rows, dtype=torch.float32, device=x2.device) if not checkpoint else None
        rstd = torch.empty(rows, dtype=torch.float32, device=x2.device)
        if checkpoint:
            codes = torch.empty((rows, D), dtype=torch.int8, device=x2.device)
            exps = torch.empty((rows, (D + 31) // 32), dtype=torch.uint8, device=x2.device)
    if rows:
        f32 = any(p is not None and p.dtype == torch.float32 for p in (weight, bias))
        _call("lsdm_layer_norm", x2.device.index, _DTYPES[x2.dtype], _PARAM_F32 if f32 else 0, rows, D, x2.data_ptr(), ld, _ptr(weight), _ptr(bias), eps,
              y.data_ptr(), _ptr(mean), _ptr(rstd), _ptr(codes), _ptr(exps), _stream(x2))
    return y, mean, rstd, codes, exps


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, checkpoint):
        D = x.shape[-1]
        x2, ld = _rows(x, D)
        w = weight.contiguous() if weight is not None else None
        b = bias.contiguous() if bias is not None else None
        y, mean, rstd, codes, exps = _norm_forward(x2, ld, D, w, b, eps, True, checkpoint)
        ctx.save_for_backward(None if checkpoint else x, mean, rstd, codes, exps, weight)
        ctx.xshape, ctx.rows = x.shape, x2.shape[0]
        ctx.param_dtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        x, mean, rstd, codes, exps, weight = ctx.saved_tensors
        D, rows, dev = ctx.xshape[-1], ctx.rows, dy.device
        dx = torch.empty(ctx.xshape, dtype=dy.dtype, device=dev) if need_x else None
        new = torch.empty if rows else torch.zeros
        dw = new(D, dtype=ctx.param_dtype, device=dev) if need_w else None
        db = new(D, dtype=ctx.param_dtype, device=dev) if need_b else None
        if rows:
            dy2, lddy = _rows(dy, D)
            x2, ld = _rows(x, D) if x is not None else (None, 0)
            w = weight.contiguous() if weight is not None else None
            nbytes = _norm_bytes(rows, D) if need_w or need_b else 0
            ws = _scratch(nbytes, dy2)
            _call("lsdm_layer_norm_backward", dev.index, _DTYPES[dy.dtype], _PARAM_F32 if ctx.param_dtype == torch.float32 else 0, rows, D, dy2.data_ptr(), lddy,
                  _ptr(x2), ld, _ptr(codes), _ptr(exps), _ptr(w), _ptr(mean), _ptr(rstd), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nbytes, _stream(dy2))
        return dx, dw, db, None, None


@functools.lru_cache(maxsize=4096)
def _norm_bytes(rows, D):
    n = _lib.load().lsdm_layer_norm_workspace(rows, D)
    if n < 0:
        raise _lib.LsdmError("lsdm_layer_norm_workspace failed (%d): %s" % (n, _lib.load().lsdm_last_error(None).decode()))
    return n


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, checkpoint8=False):
    """Layer norm over the last axis: x (..., D), weight / bias (D) or None -> (..., D); D <= 16384.

    ``checkpoint8`` (bfloat16 / float16): keep the normalised rows in 8 bits for the backward pass (the module docstring)."""
    _check_tensors("layer_norm", x, weight=weight, bias=bias)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= NORM_MAX_WIDTH:
        raise ValueError("layer_norm: the last axis must hold 1 to %d values, got shape %s" % (NORM_MAX_WIDTH, tuple(x.shape)))
    D = x.shape[-1]
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (p.shape != (D,) or p.dtype not in (x.dtype, torch.float32)):
            raise ValueError("layer_norm: %s must be (%d,) of dtype %s or float32, got %s %s" % (name, D, x.dtype, tuple(p.shape), p.dtype))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("layer_norm: weight and bias must have the same dtype, got %s and %s" % (weight.dtype, bias.dtype))
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError("layer_norm: eps must be >= 0, got %r" % eps)
    if checkpoint8 and x.dtype == torch.float32:
        raise ValueError("layer_norm: checkpoint8 takes bfloat16 or float16 (float32 gradients would show the codes' rounding decisions)")
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps, bool(checkpoint8))
    x2, ld = _rows(x, D)
    y = _norm_forward(x2, ld, D, weight.contiguous() if weight is not None else None, bias.contiguous() if bias is not None else None, eps, False, False)[0]
    return y if x.dim() == 2 else y.view(x.shape)
