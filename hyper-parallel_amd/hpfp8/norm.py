"""Layer norm with the calling convention of torch.nn.functional.layer_norm, the norm before a linear."""
from __future__ import annotations

from typing import Optional, Sequence, Union

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .kept import _TYPES, _as_rows, _check_rows, _check_saved, _groups
from .linear import _hand_off

MAX_WIDTH = 16384
_OF_CODE = {code: dtype for dtype, code in _TYPES.items()}


def _forward(x2, weight, bias, eps, stats: bool, keep: bool, shape=None):
    """(y of that shape, mean, rstd, codes, scale_inv); without ``stats`` the middle two are None, without ``keep`` the last two, with it the mean."""
    rows, cols = x2.shape
    # (not made as rows and returned as a view of them: an autograd function's result that is a view can't be written to)
    y = torch.empty(x2.shape if shape is None else shape, dtype=x2.dtype, device=x2.device)
    mean = rstd = codes = scale_inv = None
    if stats:
        rstd = torch.empty((rows,), dtype=torch.float32, device=x2.device)
        if not keep:
            mean = torch.empty_like(rstd)
    if keep:
        codes = torch.empty((rows, cols), dtype=ops.FP8, device=x2.device)
        scale_inv = torch.empty((rows, _groups(cols)), dtype=torch.float32, device=x2.device)
    vector = weight if weight is not None else bias
    _lib.call("hpfp8_layer_norm_forward", ops._ptr(x2), _TYPES[x2.dtype], rows, cols, x2.stride(0), ops._ptr(weight), ops._ptr(bias),
              0 if vector is None else _TYPES[vector.dtype], eps, ops._ptr(y), ops._ptr(mean), ops._ptr(rstd), ops._ptr(codes),
              ops._ptr(scale_inv), ops._stream())
    return y, mean, rstd, codes, scale_inv


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, cols, eps, keep):
        x2 = _as_rows(x, cols)
        w = None if weight is None else weight.reshape(-1).contiguous()
        b = None if bias is None else bias.reshape(-1).contiguous()
        y, mean, rstd, codes, scale_inv = _forward(x2, w, b, eps, True, keep, x.shape)
        if keep:
            ctx.save_for_backward(codes, scale_inv, rstd, weight)
        else:
            ctx.save_for_backward(x, mean, rstd, weight)
        ctx.keep, ctx.cols, ctx.shape, ctx.dtype = keep, cols, x.shape, x.dtype
        vector = weight if weight is not None else bias
        ctx.vector = None if vector is None else (vector.shape, vector.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        shape, dtype = ctx.vector if ctx.vector is not None else (None, torch.float32)
        return _backward(grad_out, *ctx.saved_tensors, ctx.keep, ctx.cols, ctx.shape, _TYPES[ctx.dtype], shape, _TYPES[dtype],
                         ctx.needs_input_grad[1], ctx.needs_input_grad[2]) + (None, None, None)


def _backward(grad_out, kept, other, rstd, weight, keep, cols, shape, dtype, vector, vector_dtype, need_dw, need_db):
    """(dx, dw, db).  kept, other: x and its mean, or the codes and scales of its normalised values; vector: the shape of weight and bias."""
    go = _as_rows(grad_out, cols)
    rows = go.shape[0]
    f32 = torch.float32
    _check_saved(*(((kept, ops.FP8, rows * cols), (other, f32, rows * _groups(cols))) if keep else ((kept, _OF_CODE[dtype], rows * cols), (other, f32, rows))),
                 (rstd, f32, rows), *(((weight, _OF_CODE[vector_dtype], cols),) if weight is not None else ()))
    # (hooks on saved tensors may have handed them back with other strides)
    kept, other, rstd = kept.contiguous() if keep else kept, other.contiguous(), rstd.contiguous()
    dx = torch.empty(shape, dtype=_OF_CODE[dtype], device=go.device)
    dw, db = (torch.empty(vector, dtype=_OF_CODE[vector_dtype], device=go.device) if need else None for need in (need_dw, need_db))
    partial = torch.empty((_lib.load().hpfp8_layer_norm_partials(rows, cols), 2, cols), dtype=torch.float32, device=go.device)
    w = None if weight is None else weight.reshape(-1).contiguous()
    x2 = None if keep else _as_rows(kept, cols)
    _lib.call("hpfp8_layer_norm_backward", ops._ptr(go), go.stride(0), ops._ptr(x2), 0 if x2 is None else x2.stride(0),
              None if keep else ops._ptr(other), ops._ptr(kept) if keep else None, ops._ptr(other) if keep else None, ops._ptr(rstd), dtype, rows,
              cols, ops._ptr(w), vector_dtype, ops._ptr(dx), ops._ptr(dw), ops._ptr(db), ops._ptr(partial), ops._stream())
    return dx, dw, db


if ops._native is not None:
    ops._native.bind_norm_backward(_backward)


_LAYER_NORM_DEFAULTS = dict(weight=None, bias=None, eps=1e-5, keep_8bit=False)


def layer_norm(input: torch.Tensor, normalized_shape: Union[int, Sequence[int]], weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5, *, keep_8bit: bool = False) -> torch.Tensor:
    """torch.nn.functional.layer_norm on bfloat16, float16 or float32 tensors: statistics and sums in fp32, one rounding of each result,
    the gradients of weight and bias summed over the rows in a fixed order (the same bits every time).

    weight and bias have ``normalized_shape`` and one type, input's or another of the three.  A row (the product of ``normalized_shape``)
    has at most 16384 values.  ``keep_8bit`` keeps the normalised input for the backward as E4M3 codes with one scale for each 128 values
    of a row, 1.03 bytes a value instead of input itself; the gradients are then those of the values that the codes stand for."""
    tensors = tuple(t for t in (input, weight, bias) if t is not None)
    if torch.overrides.has_torch_function(tensors):
        return _hand_off(layer_norm, tensors, (input, normalized_shape), dict(weight=weight, bias=bias, eps=eps, keep_8bit=keep_8bit),
                         _LAYER_NORM_DEFAULTS)
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    if ops._gpu(input):
        device = ops._device()
        y = ops._native.layer_norm(input, shape, weight, bias, eps, keep_8bit, device, ops._raw_stream(device))
        if y is not None:
            return y
    _check_rows(input, "input")
    shape = torch.Size(shape)
    if len(shape) < 1 or input.shape[-len(shape):] != shape:
        raise ValueError(f"input {tuple(input.shape)} does not end with normalized_shape {tuple(shape)}")
    cols = shape.numel()
    if not 0 < cols <= MAX_WIDTH:
        raise ValueError(f"a row must have 1 to {MAX_WIDTH} values, got {cols}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _check_rows(t, name)
            if t.shape != shape:
                raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must be of one type, got {weight.dtype} and {bias.dtype}")
    if ops._in_graph(*tensors):
        return ops._apply(_LayerNorm, 2, input, weight, bias, cols, float(eps), bool(keep_8bit))
    w = None if weight is None else weight.detach().reshape(-1).contiguous()
    b = None if bias is None else bias.detach().reshape(-1).contiguous()
    return _forward(_as_rows(input.detach(), cols), w, b, float(eps), False, False, input.shape)[0]


class LayerNorm(nn.LayerNorm):
    """torch.nn.LayerNorm (its parameters and state dict) computed by `layer_norm`; ``keep_8bit`` as there."""

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, *, keep_8bit: bool = False,
                 device=None, dtype=torch.bfloat16):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device=device, dtype=dtype)
        self.keep_8bit = keep_8bit

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps, keep_8bit=self.keep_8bit)

    def extra_repr(self) -> str:
        return super().extra_repr() + f", keep_8bit={self.keep_8bit}"
