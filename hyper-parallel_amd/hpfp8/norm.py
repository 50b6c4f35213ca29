"""The norm before a linear: layer norm with the calling convention of torch.nn.functional.layer_norm, and the root-mean-square norm with
that of torch.nn.functional.rms_norm, with the residual stream's addition in the same pass and, for inference, its result in the 8 bits that
the linear reads."""
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


def _vector(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.reshape(-1).contiguous()


def _width(input, normalized_shape, **vectors) -> int:
    """The number of values of a row; raises for what does not go together."""
    shape = torch.Size(normalized_shape)
    if len(shape) < 1 or input.shape[-len(shape):] != shape:
        raise ValueError(f"input {tuple(input.shape)} does not end with normalized_shape {tuple(shape)}")
    cols = shape.numel()
    if not 0 < cols <= MAX_WIDTH:
        raise ValueError(f"a row must have 1 to {MAX_WIDTH} values, got {cols}")
    for name, t in vectors.items():
        if t is not None:
            _check_rows(t, name)
            if t.shape != shape:
                raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return cols


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
    cols = _width(input, shape, weight=weight, bias=bias)
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


def _rms_forward(x, residual, weight, cols, eps, stats: bool):
    """(y, x + residual or None, rstd or None)"""
    x2, w = _as_rows(x, cols), _vector(weight)
    r2 = None if residual is None else _as_rows(residual, cols)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    total = None if residual is None else torch.empty_like(y)
    rstd = torch.empty((x2.shape[0],), dtype=torch.float32, device=x.device) if stats else None
    _lib.call("hpfp8_rms_norm_forward", ops._ptr(x2), x2.stride(0), ops._ptr(r2), 0 if r2 is None else r2.stride(0), _TYPES[x.dtype], x2.shape[0], cols,
              ops._ptr(w), 0 if w is None else _TYPES[w.dtype], eps, ops._ptr(total), ops._ptr(y), ops._ptr(rstd), ops._stream())
    return y, total, rstd


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, cols, eps):
        y, total, rstd = _rms_forward(x, residual, weight, cols, eps, True)
        ctx.save_for_backward(x if residual is None else total, rstd, weight)
        ctx.set_materialize_grads(False)
        ctx.cols, ctx.shape, ctx.dtype, ctx.residual = cols, x.shape, x.dtype, residual is not None
        ctx.vector = None if weight is None else (weight.shape, weight.dtype)
        return y if residual is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_sum=None):
        shape, dtype = ctx.vector if ctx.vector is not None else (None, torch.float32)
        ds, dw = _rms_backward(grad_out, grad_sum, *ctx.saved_tensors, ctx.cols, ctx.shape, _TYPES[ctx.dtype], shape, _TYPES[dtype],
                               ctx.needs_input_grad[2])
        return ds, ds if ctx.residual else None, dw, None, None


def _rms_backward(grad_out, grad_sum, kept, rstd, weight, cols, shape, dtype, vector, vector_dtype, need_dw):
    """(the gradient of what was normalised, dw).  kept: that, x or its sum with the residual; vector: the shape of weight.  Where the normalised
    result itself was not used, grad_out is None, and grad_sum is all there is."""
    if grad_out is None:
        return grad_sum, None
    go = _as_rows(grad_out, cols)
    rows = go.shape[0]
    f32 = torch.float32
    _check_saved((kept, _OF_CODE[dtype], rows * cols), (rstd, f32, rows), *(((weight, _OF_CODE[vector_dtype], cols),) if weight is not None else ()))
    s2, rstd, w = _as_rows(kept, cols), rstd.contiguous(), _vector(weight)       # (hooks on saved tensors may have changed their strides)
    gs = None if grad_sum is None else _as_rows(grad_sum, cols)
    ds = torch.empty(shape, dtype=_OF_CODE[dtype], device=go.device)
    dw = torch.empty(vector, dtype=_OF_CODE[vector_dtype], device=go.device) if need_dw else None
    partial = torch.empty((_lib.load().hpfp8_rms_norm_partials(rows, cols), cols), dtype=f32, device=go.device)
    _lib.call("hpfp8_rms_norm_backward", ops._ptr(go), go.stride(0), ops._ptr(s2), s2.stride(0), ops._ptr(gs), 0 if gs is None else gs.stride(0),
              ops._ptr(rstd), dtype, rows, cols, ops._ptr(w), vector_dtype, ops._ptr(ds), ops._ptr(dw), ops._ptr(partial), ops._stream())
    return ds, dw


if ops._native is not None:
    ops._native.bind_rms_norm_backward(_rms_backward)


def _default_eps(eps: Optional[float]) -> float:
    return torch.finfo(torch.float32).eps if eps is None else float(eps)       # (what torch's takes for the 16-bit types too)


def _check_residual(input, residual) -> None:
    if residual is None:
        return
    _check_rows(residual, "residual")
    if residual.dtype != input.dtype:
        raise TypeError(f"input and residual must be of one type, got {input.dtype} and {residual.dtype}")
    if residual.shape != input.shape:
        raise ValueError(f"residual must have input's shape {tuple(input.shape)}, got {tuple(residual.shape)}")


_RMS_NORM_DEFAULTS = dict(weight=None, eps=None, residual=None)


def rms_norm(input: torch.Tensor, normalized_shape: Union[int, Sequence[int]], weight: Optional[torch.Tensor] = None,
             eps: Optional[float] = None, *, residual: Optional[torch.Tensor] = None):
    """torch.nn.functional.rms_norm on bfloat16, float16 or float32 tensors: the sum of squares in fp32, one rounding of each result, the
    weight's gradient summed over the rows in a fixed order (the same bits every time).

    With ``residual`` (input's shape and type) the result is a pair, as a transformer block goes on with both: the norm of
    ``input + residual``, and that sum, rounded to their type ahead of the norm.  Gradients flow through both.

    weight has ``normalized_shape`` and input's type or another of the three.  A row (the product of ``normalized_shape``) has at most 16384
    values."""
    tensors = tuple(t for t in (input, weight, residual) if t is not None)
    if torch.overrides.has_torch_function(tensors):
        return _hand_off(rms_norm, tensors, (input, normalized_shape), dict(weight=weight, eps=eps, residual=residual), _RMS_NORM_DEFAULTS)
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    eps = _default_eps(eps)
    if ops._gpu(input):
        device = ops._device()
        made = ops._native.rms_norm(input, shape, weight, residual, eps, device, ops._raw_stream(device))
        if made is not None:
            return made
    _check_rows(input, "input")
    cols = _width(input, shape, weight=weight)
    _check_residual(input, residual)
    if ops._in_graph(*tensors):
        return ops._apply(_RmsNorm, 2, input, residual, weight, cols, eps)
    y, total, _ = _rms_forward(input.detach(), None if residual is None else residual.detach(), None if weight is None else weight.detach(), cols, eps,
                               False)
    return y if residual is None else (y, total)


_E4M3, _E4M3_POW2, _INT8 = 0, 1, 2


def _rms_quantize(name, form, input, weight, eps, residual):
    eps = _default_eps(eps)
    if ops._gpu(input):
        device = ops._device()
        made = ops._native.rms_norm_quantize(input, weight, residual, eps, form, device, ops._raw_stream(device))
        if made is not None:
            return made
    _check_rows(input, "input")
    if input.dim() < 1:
        raise ValueError("input must have at least one dimension")
    cols = _width(input, input.shape[-1:], weight=weight)
    if cols % ops.BLOCK:
        raise ValueError(f"last dim {cols} is not a multiple of {ops.BLOCK}")
    _check_residual(input, residual)
    if ops._in_graph(input, weight, residual):
        raise RuntimeError(f"{name} is for inference: its results have no gradient and no place in a trace (call it under torch.no_grad())")
    x2, w = _as_rows(input, cols), _vector(weight)
    r2 = None if residual is None else _as_rows(residual, cols)
    rows = x2.shape[0]
    codes = torch.empty(input.shape, dtype=torch.int8 if form == _INT8 else ops.FP8, device=input.device)
    total = None if residual is None else torch.empty(input.shape, dtype=input.dtype, device=input.device)
    shape = (rows,) if form == _INT8 else (cols // ops.BLOCK, rows)
    scale_inv = torch.empty(shape, dtype=torch.float32, device=input.device)
    of = (ops._ptr(x2), x2.stride(0), ops._ptr(r2), 0 if r2 is None else r2.stride(0), _TYPES[input.dtype], rows, cols, ops._ptr(w),
          0 if w is None else _TYPES[w.dtype], eps)
    to = (ops._ptr(total), ops._ptr(codes), ops._ptr(scale_inv), ops._stream())
    if form == _INT8:
        _lib.call("hpfp8_rms_norm_quantize_int8", *of, *to)
        scale_inv = scale_inv.view(input.shape[:-1])
    else:
        _lib.call("hpfp8_rms_norm_quantize_1x128_kmajor", *of, int(form == _E4M3_POW2), *to)
        scale_inv = scale_inv.t()
        if input.dim() != 2:
            scale_inv = scale_inv.reshape(input.shape[:-1] + (cols // ops.BLOCK,))
    return (codes, scale_inv) if residual is None else (codes, scale_inv, total)


def rms_norm_quantize_1x128(input: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: Optional[float] = None, *,
                            residual: Optional[torch.Tensor] = None, pow2: bool = False):
    """`rms_norm` over the last dimension (a multiple of 128), its fp32 result quantized as `quantize_1x128(kmajor=True)` quantizes: (codes,
    scale_inv[..., C/128]), what `gemm_blockwise` takes, and with ``residual`` the sum as a third.  For inference."""
    return _rms_quantize("rms_norm_quantize_1x128", _E4M3_POW2 if pow2 else _E4M3, input, weight, eps, residual)


def rms_norm_quantize_int8(input: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: Optional[float] = None, *,
                           residual: Optional[torch.Tensor] = None):
    """`rms_norm` over the last dimension (a multiple of 128), its fp32 result quantized as `quantize_int8` quantizes: (codes, scale_inv[...]),
    what `gemm_int8` takes, and with ``residual`` the sum as a third.  For inference."""
    return _rms_quantize("rms_norm_quantize_int8", _INT8, input, weight, eps, residual)


class RMSNorm(nn.RMSNorm):
    """torch.nn.RMSNorm (its parameter and state dict) computed by `rms_norm`; called with ``residual`` it returns the pair."""

    def __init__(self, normalized_shape, eps: Optional[float] = None, elementwise_affine: bool = True, device=None, dtype=torch.bfloat16):
        super().__init__(normalized_shape, eps, elementwise_affine, device=device, dtype=dtype)

    def forward(self, input: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm(input, self.normalized_shape, self.weight, self.eps, residual=residual)
