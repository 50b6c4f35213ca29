"""Activations kept in 8 bits between forward and backward.

An activation that is only needed again in the backward can wait there as E4M3 codes with one fp32 scale for each 128 values of its last
dimension: 1.03 bytes a value instead of two or four.  `fp8_linear` keeps its input that way by itself; this module does it for the rest
of a model:

  `quantize_activation(x)`     codes and scales of any floating tensor, `.dequantize()` what they stand for
  `keep_activations_8bit()`    around any torch code: what its backward nodes save is kept so
  `activation(x, kind)`        silu, gelu, gelu_tanh or swiglu, the codes written in the pass that computes the result, and the derivative
                               taken from them in the pass that computes the gradient
"""
from __future__ import annotations

import contextlib
from typing import Callable, NamedTuple, Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .linear import _hand_off

_TYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
KINDS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "swiglu": 3}


def _check_rows(x, name: str) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if x.dtype not in _TYPES:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {x.dtype}")
    ops._check_device(x, name)


def _as_rows(x: torch.Tensor, cols: int) -> torch.Tensor:
    """x as [rows, cols] with unit stride along a row: a view where x's strides allow it."""
    x = x.reshape(x.numel() // cols if cols else 0, cols)
    return x if cols == 1 or x.stride(1) == 1 else x.contiguous()


def _check_saved(*saved) -> None:
    """(tensor, dtype, number of elements) of what a backward is about to give to its kernels.  It is what the forward saved unless a hook on
    saved tensors handed back something else; that is refused, as the kernels would read beyond it, or memory that is not the GPU's."""
    for t, dtype, numel in saved:
        if t.dtype != dtype or t.numel() != numel:
            raise ValueError(f"a saved tensor of {numel} values of {dtype} came back as {tuple(t.shape)} of {t.dtype}")
        ops._check_device(t, "a saved tensor")


def _groups(cols: int) -> int:
    return (cols + ops.BLOCK - 1) // ops.BLOCK


def _dequantize(codes, scale_inv, dtype, saved: bool):
    if ops._gpu(codes):
        device = ops._device()
        x = ops._native.dequantize_rows(codes, scale_inv, _TYPES[dtype], saved, device, ops._raw_stream(device))
        if x is not None:
            return x
    if codes.dtype != ops.FP8 or scale_inv.dtype != torch.float32:
        raise TypeError(f"codes and scale_inv must be float8_e4m3fn and float32, got {codes.dtype} and {scale_inv.dtype}")
    ops._check_device(codes, "codes")
    ops._check_device(scale_inv, "scale_inv")
    if codes.dim() < 1:
        raise ValueError("codes must have at least one dimension")
    cols = codes.shape[-1]
    if cols and scale_inv.numel() != codes.numel() // cols * _groups(cols):
        raise ValueError(f"codes {tuple(codes.shape)} have a scale for each 128 values of a row, not {tuple(scale_inv.shape)}")
    codes, scale_inv = codes.contiguous(), scale_inv.contiguous()         # (a slice of what was made, say)
    x = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    _lib.call("hpfp8_dequantize_saved_rows" if saved else "hpfp8_dequantize_rows", ops._ptr(codes), ops._ptr(scale_inv),
              x.numel() // max(cols, 1), cols, ops._ptr(x), _TYPES[dtype], ops._stream())
    return x


def _quantize(x, saved: bool):
    """(codes, scale_inv) of x; ``saved``: with codes for infinities and NaN, for `_dequantize` with the same."""
    if ops._gpu(x):
        device = ops._device()
        made = ops._native.quantize_rows(x, saved, device, ops._raw_stream(device))
        if made is not None:
            return made
    _check_rows(x, "x")
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    cols = x.shape[-1]
    x2 = _as_rows(x, cols)
    codes = torch.empty(x.shape, dtype=ops.FP8, device=x.device)
    scale_inv = torch.empty(x.shape[:-1] + (_groups(cols),), dtype=torch.float32, device=x.device)
    _lib.call("hpfp8_quantize_saved_rows" if saved else "hpfp8_quantize_rows", ops._ptr(x2), _TYPES[x.dtype], x2.shape[0], cols, x2.stride(0),
              ops._ptr(codes), ops._ptr(scale_inv), ops._stream())
    return codes, scale_inv


class Fp8Activation(NamedTuple):
    """A tensor in 8 bits: what `quantize_activation` makes."""
    codes: torch.Tensor                 # e4m3, the tensor's shape
    scale_inv: torch.Tensor             # fp32 [..., ceil(C / 128)]
    dtype: torch.dtype                  # of the tensor it was made from

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values that the codes stand for, rounded once to ``dtype`` (default: that of the original)."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _TYPES:
            raise TypeError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
        return _dequantize(self.codes, self.scale_inv, dtype, False)

    def __repr__(self) -> str:          # (shapes, never values: see Fp8Weight)
        return f"Fp8Activation({tuple(self.codes.shape)}@{self.codes.data_ptr():#x}, {self.dtype})"


def quantize_activation(x: torch.Tensor) -> Fp8Activation:
    """x[..., C] (bfloat16, float16 or float32; any C, any strides) in 8 bits: E4M3 codes, one scale for each 128 values of the last
    dimension, the last group of a row being what is left.  For bf16 rows of a multiple of 128 values the codes and scales of
    `quantize_1x128`.  An infinity or a NaN makes its whole group NaN."""
    return Fp8Activation(*_quantize(x, False), x.dtype)


class _Saved(NamedTuple):
    """What `keep_activations_8bit` puts in a tensor's place; `_AsItIs` for those that stay."""
    codes: torch.Tensor
    scale_inv: torch.Tensor
    dtype: torch.dtype


class _AsItIs(NamedTuple):
    tensor: torch.Tensor
    version: int


def _is_parameter(t: torch.Tensor) -> bool:
    """Whether t is a parameter (frozen ones too), another leaf that requires a gradient, or a view of one: what is there anyway."""
    base = t if t._base is None else t._base
    return isinstance(base, torch.nn.Parameter) or (base.is_leaf and base.requires_grad)


def _takes_less(t: torch.Tensor) -> bool:
    """Whether codes and scales are less than what t holds: not for an expanded tensor, whose values are there once, nor for rows of a few values."""
    if t.layout != torch.strided or any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        return False
    cols = t.shape[-1]
    return cols + 4 * _groups(cols) < t.element_size() * cols


def _own(t: torch.Tensor) -> bool:
    """Whether t, just being saved, is a scale of codes or a statistic of this package's own operators, or belongs to a statistic: the
    softmax of logits that are computed again from 8 bits does not sum to 1 with the exact ones' sum, nor are values normalised by the mean
    and deviation of others."""
    level = max(ops._saving.level, ops._native.saving() if ops._native is not None else 0)
    return level == 2 or (level == 1 and t.dtype == torch.float32)


@contextlib.contextmanager
def keep_activations_8bit(min_elements: int = 1 << 16, dtypes: Sequence[torch.dtype] = (torch.bfloat16, torch.float16),
                          select: Optional[Callable[[torch.Tensor], bool]] = None):
    """Inside this context the tensors that backward nodes save are kept in 8 bits until the backward reads them.

    Kept so are GPU tensors of ``min_elements`` values and more in one of ``dtypes`` (by default the 16-bit types: an fp32 tensor is
    more often a statistic or a scale than an activation), unless they are parameters, other leaves that require a gradient, or views of
    one (a copy, such as a parameter cast to 16 bits, is none), or ``select(tensor)`` says no.  This package's own operators keep their scales and statistics as they are, and `layer_norm` and
    `linear_cross_entropy`, whose statistics are those of the exact input, their input too.  Everything else is kept as it is.  The backward may run after the context has ended.

    An expanded tensor stays as it is too, and one whose last dimension is so short (4 values of 16 bits) that the scales take what the codes save.  Each
    node that saves a tensor has codes of its own: a 16-bit tensor that two nodes save takes 2.06 bytes a value, where both share one of 2 outside.

    What the backward reads is off by 2^-4 of a value at most, or by 2^-10 of 1 / 448 of the largest finite value among its group's 128 where that is
    more; infinities and NaN (a mask's -inf, say) come back as they were."""
    for d in dtypes:
        if d not in _TYPES:
            raise TypeError(f"dtypes must be bfloat16, float16 or float32, got {d}")

    def pack(t):
        if (type(t) is not torch.Tensor or not t.is_cuda or t.dtype not in dtypes or t.dim() < 1 or t.numel() < min_elements
                or not _takes_less(t) or _own(t) or _is_parameter(t) or (select is not None and not select(t))):
            return _AsItIs(t.detach(), t._version)         # (detached: a node that saves its own result would own itself through t)
        with torch.cuda.device(t.device):
            return _Saved(*_quantize(t.detach(), True), t.dtype)

    def unpack(kept):
        if isinstance(kept, _AsItIs):
            if kept.tensor._version != kept.version:       # (torch looks at this itself where there are no hooks)
                raise RuntimeError(f"one of the variables needed for gradient computation has been modified by an inplace operation: "
                                   f"{tuple(kept.tensor.shape)} of {kept.tensor.dtype} is at version {kept.tensor._version}; expected version {kept.version}")
            return kept.tensor
        with torch.cuda.device(kept.codes.device):
            return _dequantize(kept.codes, kept.scale_inv, kept.dtype, True)

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        yield


def _forward(x2, kind: int, shape, keep: bool):
    """(y of that shape, codes, scale_inv): the last two None unless x is kept."""
    rows, cols, halves = x2.shape[0], shape[-1], 2 if kind == 3 else 1
    # (not made as rows and returned as a view of them: an autograd function's result that is a view can't be written to)
    y = torch.empty(shape, dtype=x2.dtype, device=x2.device)
    codes = scale_inv = None
    if keep:
        codes = torch.empty((rows, halves * cols), dtype=ops.FP8, device=x2.device)
        scale_inv = torch.empty((rows, halves, _groups(cols)), dtype=torch.float32, device=x2.device)
    _lib.call("hpfp8_activation_forward", ops._ptr(x2), _TYPES[x2.dtype], rows, cols, x2.stride(0), kind, ops._ptr(y), ops._ptr(codes),
              ops._ptr(scale_inv), ops._stream())
    return y, codes, scale_inv


class _Activation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kind, keep):
        cols = x.shape[-1] // (2 if kind == 3 else 1)
        y, codes, scale_inv = _forward(_as_rows(x, x.shape[-1]), kind, x.shape[:-1] + (cols,), keep)
        # (as it was: x itself, so that a write to it in between is noticed)
        ctx.save_for_backward(*((codes, scale_inv) if keep else (x,)))
        ctx.kind, ctx.keep, ctx.shape = kind, keep, x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        return _backward(grad_out, *(ctx.saved_tensors if ctx.keep else (*ctx.saved_tensors, None)), ctx.keep, ctx.kind, ctx.shape), None, None


def _backward(grad_out, kept, scale_inv, keep, kind, shape):
    """dx.  kept: x, or its codes with their scales."""
    shape = torch.Size(shape)
    halves = 2 if kind == 3 else 1
    cols = shape[-1] // halves
    x2 = None
    if keep:
        _check_saved((kept, ops.FP8, shape.numel()), (scale_inv, torch.float32, shape[:-1].numel() * halves * _groups(cols)))
        kept, scale_inv = kept.contiguous(), scale_inv.contiguous()      # (with other strides, which hooks on saved tensors may give them)
    else:
        _check_saved((kept, grad_out.dtype, shape.numel()))
        x2 = _as_rows(kept, shape[-1])
    go = grad_out.contiguous()
    dx = torch.empty(shape, dtype=go.dtype, device=go.device)
    _lib.call("hpfp8_activation_backward", ops._ptr(go), ops._ptr(x2), 0 if x2 is None else x2.stride(0), ops._ptr(kept) if keep else None,
              ops._ptr(scale_inv), _TYPES[go.dtype], go.numel() // max(cols, 1), cols, kind, ops._ptr(dx), ops._stream())
    return dx


if ops._native is not None:
    ops._native.bind_activation_backward(lambda *args: (_backward(*args),))


_ACTIVATION_DEFAULTS = dict(keep_8bit=True)


def activation(input: torch.Tensor, kind: str, *, keep_8bit: bool = True) -> torch.Tensor:
    """An activation function whose input waits for the backward in 8 bits.

    kind: "silu", "gelu", "gelu_tanh" (the tanh form), or "swiglu": input [..., 2C] = gate | up, result silu(gate) * up [..., C].
    bfloat16, float16 or float32, any width; computed in fp32 and rounded once.  The result is that of the input as it is; the
    gradient is taken where the codes are (each half of a SwiGLU input has scaling groups of its own; an infinity or a NaN in the input makes the
    gradient of its group of 128 NaN).  ``keep_8bit=False`` keeps the input itself."""
    if torch.overrides.has_torch_function((input,)):
        return _hand_off(activation, (input,), (input, kind), dict(keep_8bit=keep_8bit), _ACTIVATION_DEFAULTS)
    if kind not in KINDS:
        raise ValueError(f"kind must be one of {tuple(KINDS)}, got {kind!r}")
    if ops._gpu(input):
        device = ops._device()
        y = ops._native.activation(input, KINDS[kind], keep_8bit, device, ops._raw_stream(device))
        if y is not None:
            return y
    _check_rows(input, "input")
    if input.dim() < 1:
        raise ValueError("input must have at least one dimension")
    if kind == "swiglu" and input.shape[-1] % 2:
        raise ValueError(f"swiglu takes gate | up in the last dimension, which is {input.shape[-1]}")
    k = KINDS[kind]
    if ops._in_graph(input):
        return ops._apply(_Activation, int(bool(keep_8bit)), input, k, bool(keep_8bit))
    cols = input.shape[-1] // (2 if kind == "swiglu" else 1)
    return _forward(_as_rows(input.detach(), input.shape[-1]), k, input.shape[:-1] + (cols,), False)[0]
