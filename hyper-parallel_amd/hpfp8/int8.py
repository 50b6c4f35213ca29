"""Linear in 8-bit integers: a weight's codes with one scale for each output channel, its input's with one for each token.

`int8_linear(x, quantize_weight_int8(w))` is torch.nn.functional.linear with a frozen weight of 1 byte an element.  Codes are
``rint(v * (127 / amax))`` of a row v with the largest magnitude amax, and stand for code * (amax / 127); the product of codes is summed in 32-bit
integers, exactly, so a result depends on nothing but its own row and channel.  The input's gradient is the same product with the weight's
transposed codes, of the output's gradient times the channels' scales, quantized with one scale for each token.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .kept import _TYPES, _as_rows, _check_rows
from .linear import _hand_off

MAX_FEATURES = 130944       # the sums of so many products of two codes fit 32 bits


class Int8Weight(NamedTuple):
    """A weight [N, K] in 8-bit integers: what `quantize_weight_int8` makes."""
    codes: torch.Tensor                 # int8 [N, K]
    scale_inv: torch.Tensor             # fp32 [N]
    codes_t: Optional[torch.Tensor] = None     # int8 [K, N], for the input's gradient (made in each backward where it is not there)

    def __repr__(self) -> str:          # (shapes, never values: see Fp8Weight)
        def one(t):
            return "None" if t is None else f"{tuple(t.shape)}@{t.data_ptr():#x}"
        return f"Int8Weight(codes={one(self.codes)}, scale_inv={one(self.scale_inv)}, codes_t={one(self.codes_t)})"

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The weight that the codes stand for."""
        return (self.codes.float() * self.scale_inv.unsqueeze(1)).to(dtype)


def quantize_int8(x: torch.Tensor, *, column_scale: Optional[torch.Tensor] = None):
    """x[..., C] (bfloat16, float16 or float32, C a multiple of 128) -> (int8 codes, scale_inv[...]): one scale for each row.  With
    ``column_scale`` (float32 [C]) of x * column_scale, rounded to fp32.  A row with an infinity or a NaN has codes of 0 and that for its scale.

    The largest magnitude that a row's scale is made from is at least 1e-12; with ``column_scale``, as a gradient's rows have, at least 2^-118."""
    return _quantize(x, column_scale, "quantize_int8")


def _quantize(x, column_scale=None, name: Optional[str] = None):
    """name: of the operator that a program calls; None inside another one, which has its place in a trace or refuses it."""
    if ops._gpu(x):
        device = ops._device()
        made = ops._native.quantize_int8(x, column_scale, device, ops._raw_stream(device))
        if made is not None:
            return made
    if name is not None:
        ops._refuse_trace(name, x, column_scale)
    _check_rows(x, "x")
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    cols = x.shape[-1]
    if cols % ops.BLOCK or not 0 < cols <= MAX_FEATURES:
        raise ValueError(f"last dim {cols} is not a multiple of {ops.BLOCK} of at most {MAX_FEATURES}")
    if column_scale is not None:
        column_scale = ops._check_f32(column_scale, "column_scale")
        if column_scale.shape != (cols,):
            raise ValueError(f"column_scale must have shape {(cols,)}, got {tuple(column_scale.shape)}")
        column_scale = column_scale.contiguous()
    x2 = _as_rows(x, cols)
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale_inv = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _lib.call("hpfp8_quantize_int8", ops._ptr(x2), _TYPES[x.dtype], x2.shape[0], cols, x2.stride(0), ops._ptr(column_scale), ops._ptr(codes),
              ops._ptr(scale_inv), ops._stream())
    return codes, scale_inv


def _transposed(codes: torch.Tensor) -> torch.Tensor:
    return ops.transpose_codes(codes.view(torch.uint8)).view(torch.int8)


def quantize_weight_int8(weight: torch.Tensor, with_transpose: bool = False) -> Int8Weight:
    """The 8-bit form of a weight [out_features, in_features], both multiples of 128; with the transposed codes, which the input's gradient
    reads, if asked for."""
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[0] % ops.BLOCK:
        raise ValueError("weight must be [out_features, in_features], both multiples of 128")
    codes, scale_inv = quantize_int8(weight.detach())
    return Int8Weight(codes, scale_inv, _transposed(codes) if with_transpose else None)


def _check_codes(t, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int8:
        raise TypeError(f"{name} must be an int8 tensor")
    ops._check_device(t, name)
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) % 16):
        raise ValueError(f"{name} must be 2-D with unit inner stride and a row stride that is a multiple of 16")
    return t


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if t is None:
        return None
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def gemm_int8(a: torch.Tensor, sa: torch.Tensor, b: torch.Tensor, sb: Optional[torch.Tensor], bias: Optional[torch.Tensor] = None, *,
              out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """c[..., n] = (a[..., :] . b[n, :]) * sa[...] * sb[n] + bias[n] for int8 codes a[..., K] and b[N, K], both multiples of 128, the sum of products
    exact; sa fp32, a scale for each row of a; sb fp32 [N], None for scales of 1; bias of ``out_dtype`` (bfloat16, float16 or float32).  It has no
    gradients: scales or a bias that require one are refused."""
    if out_dtype not in _TYPES:
        raise TypeError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    return _multiply(a, sa, b, sb, bias, out_dtype, "gemm_int8")


def _multiply(a, sa, b, sb, bias, out_dtype, name: Optional[str] = None):
    """name: as in `_quantize`."""
    if ops._gpu(a):
        device = ops._device()
        c = ops._native.gemm_int8(a, sa, b, sb, bias, _TYPES[out_dtype], device, ops._raw_stream(device))
        if c is not None:
            return c
    if name is not None:
        ops._refuse_trace(name, sa, sb, bias)
        for what, t in (("sa", sa), ("sb", sb), ("bias", bias)):
            if torch.is_grad_enabled() and isinstance(t, torch.Tensor) and t.requires_grad:
                raise ValueError(f"gemm_int8 has no gradient for {what}: detach it")
    if not isinstance(a, torch.Tensor) or a.dtype != torch.int8 or a.dim() < 1:
        raise TypeError("a must be an int8 tensor with at least one dimension")
    lead = a.shape[:-1]
    k = a.shape[-1]
    a = _check_codes(a if a.dim() == 2 else a.reshape(a.numel() // k if k else 0, k), "a")
    b = _check_codes(b, "b")
    m, n = a.shape[0], b.shape[0]
    if b.shape[1] != k or k % ops.BLOCK or n % ops.BLOCK or not 0 < k <= MAX_FEATURES:
        raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} must have rows of one length, a multiple of {ops.BLOCK} of at most {MAX_FEATURES}, "
                         f"and b a multiple of {ops.BLOCK} of them")
    sa = ops._check_f32(sa, "sa")
    if sa.numel() != m:
        raise ValueError(f"sa must have a scale for each of {m} rows, got {tuple(sa.shape)}")
    if sb is not None:
        sb = ops._check_f32(sb, "sb")
        if sb.shape != (n,):
            raise ValueError(f"sb must have shape {(n,)}, got {tuple(sb.shape)}")
    _check_bias(bias, n, out_dtype)
    sa, sb, bias = sa.contiguous(), _aligned(sb), _aligned(bias)
    # (not made as rows and returned as a view of them: an autograd function's result that is a view can't be written to)
    c = torch.empty(lead + (n,), dtype=out_dtype, device=a.device)
    _lib.call("hpfp8_gemm_int8", ops._ptr(a), ops._ld(a), ops._ptr(sa), ops._ptr(b), ops._ld(b), ops._ptr(sb), m, n, k, ops._ptr(bias), ops._ptr(c), n,
              _TYPES[out_dtype], ops._stream())
    return c


def _check_bias(bias, n: int, dtype: torch.dtype) -> None:
    if bias is None:
        return
    if not isinstance(bias, torch.Tensor) or bias.dtype != dtype:
        raise TypeError(f"bias must be a tensor of {dtype}")
    ops._check_device(bias, "bias")
    if bias.shape != (n,):
        raise ValueError(f"bias must have shape {(n,)}, got {tuple(bias.shape)}")


class _Int8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, codes, scale_inv, codes_t, bias):
        xq, sx = _quantize(x)
        y = _multiply(xq, sx, codes, scale_inv, bias, x.dtype)
        ctx.save_for_backward(codes if codes_t is None else codes_t, scale_inv)
        ctx.transposed, ctx.shape = codes_t is not None, x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        codes, scale_inv = ctx.saved_tensors
        return _int8_backward(grad_out, codes, scale_inv, ctx.transposed, ctx.shape) + (None, None, None, None)


def _int8_backward(grad_out, codes, scale_inv, transposed: bool, shape):
    """(x's gradient,).  codes: the weight's transposed ones, or as they are (as hooks on saved tensors hand them back)."""
    out, k = grad_out.shape[-1], shape[-1]
    if codes.dtype != torch.int8 or tuple(codes.shape) != ((k, out) if transposed else (out, k)) or scale_inv.dtype != torch.float32 or \
            scale_inv.shape != (out,):
        raise ValueError(f"saved codes and scales came back as {tuple(codes.shape)} of {codes.dtype} and {tuple(scale_inv.shape)} of {scale_inv.dtype}")
    goq, sgo = quantize_int8(grad_out, column_scale=scale_inv)
    wt = codes.contiguous() if transposed and codes.stride(1) != 1 else (codes if transposed else _transposed(codes.contiguous()))
    return gemm_int8(goq, sgo, wt, None, out_dtype=grad_out.dtype).view(shape),


if ops._native is not None:
    ops._native.bind_int8_backward(_int8_backward)


def int8_linear(input: torch.Tensor, weight: Int8Weight, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """torch.nn.functional.linear with a weight in 8-bit integers: input [..., in_features] (bfloat16, float16 or float32), bias [out_features] of
    input's type; the result has that type too.  in_features and out_features are multiples of 128, the number of tokens is any.

    Differentiable in input; the weight is frozen, its codes and its scales, and so is the bias."""
    tensors = (input,) if bias is None else (input, bias)
    if torch.overrides.has_torch_function(tensors):
        return _hand_off(int8_linear, tensors, (input, weight, bias), {}, {})
    if not isinstance(weight, Int8Weight):
        raise TypeError("weight must be an Int8Weight (quantize_weight_int8)")
    codes, scale_inv, codes_t = weight
    if ops._gpu(input):
        device = ops._device()
        y = ops._native.int8_linear(input, codes, scale_inv, codes_t, bias, device, ops._raw_stream(device))
        if y is not None:
            return y
    _check_rows(input, "input")
    _check_codes(codes, "weight.codes")
    n, k = codes.shape
    if input.dim() < 1 or input.shape[-1] != k:
        raise ValueError(f"input {tuple(input.shape)} does not end with the weight's in_features {k}")
    if k % ops.BLOCK or n % ops.BLOCK or not 0 < k <= MAX_FEATURES or not 0 < n <= MAX_FEATURES:
        raise ValueError(f"the weight's shape {(n, k)} must be of multiples of {ops.BLOCK} of at most {MAX_FEATURES}")
    ops._check_f32(scale_inv, "weight.scale_inv")
    if scale_inv.shape != (n,):
        raise ValueError(f"weight.scale_inv must have shape {(n,)}, got {tuple(scale_inv.shape)}")
    if codes_t is not None:
        _check_codes(codes_t, "weight.codes_t")
        if codes_t.shape != codes.shape[::-1]:
            raise ValueError(f"weight.codes_t must be the transpose of weight.codes {tuple(codes.shape)}, got {tuple(codes_t.shape)}")
    _check_bias(bias, n, input.dtype)
    if scale_inv.requires_grad and torch.is_grad_enabled():
        raise ValueError("int8_linear has no gradient for the weight's scales: detach them")
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise ValueError("int8_linear has no gradient for a bias: detach it, or add it to the result")
    if ops._in_graph(input):
        return ops._apply(_Int8Linear, 1, input, codes, scale_inv, codes_t, bias)
    xq, sx = _quantize(input)
    return _multiply(xq, sx, codes, scale_inv, bias, input.dtype)


def _refresh(layer: "Int8Linear", _keys) -> None:           # (a function of the module's, so that a layer can be pickled)
    layer.refresh()


class Int8Linear(nn.Module):
    """A linear whose weight is frozen in 8-bit integers (buffers ``weight_codes``, ``weight_scale_inv`` and, with a bias, ``bias``), computed by
    `int8_linear`.  Made of a trained layer by `from_linear`.

    With ``with_transpose`` it also holds the transposed codes, which the input's gradient reads, as a buffer that is in no state dict; without
    them, and after ``weight_codes`` was written or replaced, each backward makes them anew.  ``load_state_dict`` and `refresh` bring them up to
    date (a write that the version counter does not see, through ``weight_codes.data``, needs the latter)."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, *, with_transpose: bool = False, device=None, dtype=torch.bfloat16):
        super().__init__()
        if in_features % ops.BLOCK or out_features % ops.BLOCK or not 0 < in_features <= MAX_FEATURES or not 0 < out_features <= MAX_FEATURES:
            raise ValueError(f"in_features and out_features must be multiples of 128 of at most {MAX_FEATURES}")
        self.in_features, self.out_features, self.with_transpose = in_features, out_features, with_transpose
        self.register_buffer("weight_codes", torch.zeros((out_features, in_features), dtype=torch.int8, device=device))
        self.register_buffer("weight_scale_inv", torch.ones((out_features,), dtype=torch.float32, device=device))
        self.register_buffer("bias", torch.zeros((out_features,), dtype=dtype, device=device) if bias else None)
        self.register_buffer("weight_codes_t", None, persistent=False)
        self.refresh()
        self.register_load_state_dict_post_hook(_refresh)

    @classmethod
    def from_linear(cls, linear: nn.Module, *, with_transpose: bool = False) -> "Int8Linear":
        """Of a layer with a ``weight`` [out_features, in_features] and a ``bias`` or None: torch.nn.Linear, `Fp8Linear`."""
        weight, bias = linear.weight, linear.bias
        made = cls(weight.shape[1], weight.shape[0], bias is not None, device=weight.device, dtype=weight.dtype)
        made.weight_codes, made.weight_scale_inv, _ = quantize_weight_int8(weight)
        if bias is not None:
            made.bias = bias.detach().clone()
        made.with_transpose = with_transpose
        made.refresh()
        return made

    def _note_codes(self) -> None:
        # (the tensor itself, not its address, which another could have later; one made in inference mode has no version to go by)
        codes = self.weight_codes
        self._transposed_of = None if codes.is_inference() else (codes, codes._version)

    def _up_to_date(self) -> bool:
        of = self._transposed_of
        return of is not None and of[0] is self.weight_codes and of[1] == of[0]._version

    def __getstate__(self):             # (a copy's codes are another tensor, with a version of its own)
        return {**self.__dict__, "_transposed_of": self._up_to_date()}

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        up_to_date, self._transposed_of = self._transposed_of, None
        if up_to_date:
            self._note_codes()

    def refresh(self) -> None:
        """Make the transposed codes, where the layer holds them, of ``weight_codes`` as it is now."""
        codes = self.weight_codes
        self.weight_codes_t = None if not self.with_transpose else (_transposed(codes) if codes.is_cuda else codes.t().contiguous())
        self._note_codes()

    def _apply(self, fn, recurse=True):
        up_to_date = self._up_to_date()
        scale_inv = self.weight_scale_inv
        super()._apply(fn, recurse)
        if self.weight_scale_inv.dtype != torch.float32:            # (.to(torch.bfloat16) is meant for the bias)
            self.weight_scale_inv = scale_inv.to(self.weight_scale_inv.device)
        self._transposed_of = None
        if up_to_date:
            self._note_codes()
        return self

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        codes_t = self.weight_codes_t
        if codes_t is not None and not self._up_to_date():
            codes_t = None
        return int8_linear(input, Int8Weight(self.weight_codes, self.weight_scale_inv, codes_t), self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
