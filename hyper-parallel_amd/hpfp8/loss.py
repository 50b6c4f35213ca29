"""The loss at the end of a language model: the head's linear and the softmax cross entropy over its vocabulary in one operator, which
never holds the logits."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .kept import _check_saved
from .linear import _hand_off

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
_TILE = 256
# The forward takes this many tokens at a time: its per-tile results (8 bytes for 256 columns of a row) stay at 64 MiB for 131072 columns
_FORWARD_ROWS = 16384
# What the gradient of a piece's logits may take of memory, which is there twice
_PIECE_BYTES = 512 << 20
# Elements that a piece's rows of the weight may span: the kernels address them with 31 bits
_PIECE_ELEMENTS = 0x3FFFF000


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x[..., C] as [rows, C] the kernels can read: unit stride along a row, rows 16 bytes apart and aligned."""
    x = x.reshape(-1, x.shape[-1])
    if x.stride(1) == 1 and x.stride(0) % 8 == 0 and x.shape[1] <= x.stride(0) < 1 << 21 and x.data_ptr() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)     # (contiguous() gives back a contiguous one that starts between two vectors)


def _forward(x, weight, target, ignore_index, reduction, smoothing, want_lse):
    """(loss, lse, count): loss [tokens] or 0-dim, lse None unless asked for, count None unless the loss is reduced."""
    lib = _lib.load()
    tokens, vocab = x.shape[0], weight.shape[0]
    f32 = dict(dtype=torch.float32, device=x.device)
    most = min(tokens, _FORWARD_ROWS)
    # (the last tokens may take other tiles than the others)
    parts = max((n * lib.hpfp8_cross_entropy_parts(n, x.shape[1], vocab) for n in (most, tokens % _FORWARD_ROWS)))
    stats = torch.empty((parts, 2), **f32)
    sums = torch.empty((parts,), **f32) if smoothing else None
    own = torch.empty((most,), **f32)
    loss = torch.empty((tokens,), **f32)
    lse = torch.empty((tokens,), **f32) if want_lse else None
    out = count = None
    if reduction:
        out, count = torch.empty((), **f32), torch.empty((), **f32)
    last = max(0, (tokens - 1) // _FORWARD_ROWS * _FORWARD_ROWS)
    for at in range(0, max(tokens, 1), _FORWARD_ROWS):
        n = min(tokens - at, _FORWARD_ROWS)
        whole = last == 0            # (in several pieces the losses are reduced behind the last of them, over all of them)
        _lib.call("hpfp8_linear_cross_entropy_forward", ops._ptr(x[at:]), x.stride(0), ops._ptr(weight), weight.stride(0), ops._ptr(target[at:]), n,
                  x.shape[1], vocab, ignore_index, smoothing, reduction if whole else 0, ops._ptr(stats), ops._ptr(sums), ops._ptr(own),
                  None if lse is None else ops._ptr(lse[at:]), ops._ptr(loss[at:]), ops._ptr(out), ops._ptr(count), ops._stream())
    if reduction and last:
        _lib.call("hpfp8_linear_cross_entropy_reduce", ops._ptr(loss), ops._ptr(target), tokens, ignore_index, reduction, ops._ptr(out),
                  ops._ptr(count), ops._stream())
    return (out if reduction else loss), lse, count


def _pieces(tokens: int, stride: int, vocab: int, budget: int):
    """[(first, width)]: pieces of the vocabulary, of equal width but for the last, whole tiles wide, that fit the budget.  stride: elements
    between the weight's rows."""
    padded = (tokens + _TILE - 1) // _TILE * _TILE
    most = max(_TILE, min(budget // (4 * padded), (_PIECE_ELEMENTS - 1) // stride) // _TILE * _TILE)
    count = (vocab + most - 1) // most
    width = ((vocab + count - 1) // count + _TILE - 1) // _TILE * _TILE
    return [(at, min(width, vocab - at)) for at in range(0, vocab, width)]


def _main_grad_of(param):
    """param.main_grad (None: there is none yet), which the kernels are about to add onto.  Looked at by the call and again by its backward:
    what is there then may be another tensor."""
    main_grad = getattr(param, "main_grad", None)
    if main_grad is not None:
        if main_grad.dtype != torch.float32 or main_grad.shape != param.shape or not main_grad.is_contiguous():
            raise ValueError("weight.main_grad must be a contiguous float32 tensor of the weight's shape")
        if main_grad.device != param.device:
            raise ValueError(f"weight.main_grad lives on {main_grad.device}, the weight on {param.device}")
        if main_grad.data_ptr() % 16:
            raise ValueError("weight.main_grad must start at a multiple of 16 bytes")
    return main_grad


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction, smoothing, main_grad_of):
        x2, w = _rows(x), _rows(weight)
        loss, lse, count = _forward(x2, w, target, ignore_index, reduction, smoothing, True)
        ctx.save_for_backward(x, weight, target, lse, count)
        ctx.ignore_index, ctx.reduction, ctx.smoothing, ctx.main_grad_of = ignore_index, reduction, smoothing, main_grad_of
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        return _backward(grad_out, *ctx.saved_tensors, ctx.ignore_index, ctx.reduction, ctx.smoothing, *ctx.needs_input_grad[:2],
                         ctx.main_grad_of) + (None,) * 5


def _backward(grad_out, x, weight, target, lse, count, ignore_index, reduction, smoothing, need_dx, need_dw, param=None):
    """(dx, dw); with ``param`` the weight's gradient goes to param.main_grad."""
    tokens, (vocab, hidden) = grad_out.numel() if reduction == 0 else target.numel(), weight.shape
    _check_saved((x, torch.bfloat16, tokens * hidden), (weight, torch.bfloat16, vocab * hidden), (target, torch.int64, tokens),
                 (lse, torch.float32, tokens), *(((count, torch.float32, 1),) if count is not None else ()))
    target, lse = target.contiguous(), lse.contiguous()      # (hooks on saved tensors may have handed them back with other strides)
    x2, w = _rows(x), _rows(weight)
    main_grad = None if param is None else _main_grad_of(param)
    if tokens == 0:
        if need_dw and param is not None and main_grad is None:
            param.main_grad = torch.zeros(weight.shape, dtype=torch.float32, device=w.device)
        return torch.zeros_like(x) if need_dx else None, torch.zeros_like(weight) if need_dw and param is None else None
    bf16, f32 = dict(dtype=torch.bfloat16, device=x2.device), dict(dtype=torch.float32, device=x2.device)
    # (the same for every row, as behind a sum or a mean of the losses: one factor of the sums, which the logits' gradient is not rounded with)
    same = reduction != 0 or all(n == 1 or s == 0 for n, s in zip(grad_out.shape, grad_out.stride()))
    grad = grad_out if same else grad_out.reshape(-1).contiguous()
    dw = dx = x_t = None
    splits = 1
    pieces = _pieces(tokens, w.stride(0), vocab, _PIECE_BYTES)
    width = pieces[0][1]
    row_t, row = (_lib.load().hpfp8_cross_entropy_stride(n) for n in (tokens, width))
    dl = torch.empty(((tokens + _TILE - 1) // _TILE * _TILE, row), **bf16)
    dl_t = torch.empty(((width + _TILE - 1) // _TILE * _TILE, row_t), **bf16)
    if need_dw:
        dw = torch.empty((vocab, hidden), **bf16) if param is None else main_grad
        if dw is None:
            dw = torch.empty((vocab, hidden), **f32)
        x_t = torch.empty((hidden, row_t), **bf16)
        _lib.call("hpfp8_linear_cross_entropy_rows_t", ops._ptr(x2), tokens, hidden, x2.stride(0), ops._ptr(target), ignore_index, ops._ptr(x_t),
                  row_t, ops._stream())
    if need_dx:
        splits = _lib.load().hpfp8_cross_entropy_splits(tokens, hidden, width, int(need_dw))
        dx = torch.empty((splits, tokens, hidden), **f32)
    for first, n in pieces:
        _lib.call("hpfp8_linear_cross_entropy_piece", ops._ptr(x2), x2.stride(0), ops._ptr(x_t), ops._ptr(w), w.stride(0), ops._ptr(target),
                  tokens, hidden, vocab, first, n, ignore_index, smoothing, ops._ptr(lse), ops._ptr(grad), 0 if same else 1,
                  ops._ptr(count) if reduction == 1 else None, ops._ptr(dl), ops._ptr(dl_t), ops._ptr(dx), splits, int(first > 0), ops._ptr(dw),
                  _lib.OUT_BF16 if param is None else _lib.OUT_F32, int(main_grad is not None), ops._stream())
    if need_dx:
        rounded = torch.empty(x.shape, **bf16)
        _lib.call("hpfp8_linear_cross_entropy_round", ops._ptr(dx), tokens * hidden, splits, ops._ptr(rounded), ops._stream())
        dx = rounded
    if need_dw and param is not None:
        if main_grad is None:
            param.main_grad = dw
        dw = None
    return dx, dw


if ops._native is not None:
    ops._native.bind_loss_backward(_backward)


_DEFAULTS = dict(ignore_index=-100, reduction="mean", label_smoothing=0.0, apply_grad_on_fp32_main_grad=False)


def linear_cross_entropy(input: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean", label_smoothing: float = 0.0,
                         apply_grad_on_fp32_main_grad: bool = False) -> torch.Tensor:
    """F.cross_entropy(F.linear(input, weight), target) without the logits: input [..., hidden] and weight [vocab, hidden] in bfloat16
    (hidden a multiple of 8, any vocabulary up to 2^24), target int64 of input's leading shape.

    The logits are fp32 accumulators of the tensors' products and are not rounded; the loss is fp32: [...] with reduction "none" (0 where
    target is ``ignore_index``), its sum, or its mean over the tokens that are not ignored (NaN if all are, with gradients of 0), summed in
    a fixed order.  At most 2^21 tokens in a call.
    A target that is neither ``ignore_index`` nor in [0, vocab) makes its token's loss and gradients NaN.  In the backward the logits are
    computed again, a piece of the vocabulary at a time, their gradient rounded to bfloat16 for the products of both gradients.

    ``apply_grad_on_fp32_main_grad`` as in `fp8_linear`: the weight's gradient goes to ``weight.main_grad`` (fp32, on the weight's
    device, 16-byte aligned), created by the first backward and added onto by every later one."""
    if torch.overrides.has_torch_function((input, weight, target)):
        return _hand_off(linear_cross_entropy, (input, weight, target), (input, weight, target),
                         dict(ignore_index=ignore_index, reduction=reduction, label_smoothing=label_smoothing,
                              apply_grad_on_fp32_main_grad=apply_grad_on_fp32_main_grad), _DEFAULTS)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(_REDUCTIONS)}, got {reduction!r}")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must be in [0, 1], got {label_smoothing}")
    if not apply_grad_on_fp32_main_grad and ops._gpu(input):
        device = ops._device()
        loss = ops._native.linear_cross_entropy(input, weight, target, ignore_index, _REDUCTIONS[reduction], label_smoothing, _FORWARD_ROWS,
                                                _PIECE_BYTES, _PIECE_ELEMENTS, device, ops._raw_stream(device))
        if loss is not None:
            return loss
    for name, t in (("input", input), ("weight", weight)):
        ops._check_bf16(t, name, contiguous=False)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[0] > 1 << 24:
        raise ValueError("weight must be [vocab, hidden] with 1 to 2^24 rows")
    hidden = weight.shape[1]
    if input.dim() < 1 or input.shape[-1] != hidden:
        raise ValueError(f"input {tuple(input.shape)} does not end with weight's hidden size {hidden}")
    if hidden < 8 or hidden % 8 or hidden >= 1 << 21:
        raise ValueError(f"hidden must be a multiple of 8 below 2^21, got {hidden}")
    if not isinstance(target, torch.Tensor) or target.dtype != torch.int64:
        raise TypeError("target must be an int64 tensor")
    ops._check_device(target, "target")
    if target.shape != input.shape[:-1]:
        raise ValueError(f"target must have input's leading shape {tuple(input.shape[:-1])}, got {tuple(target.shape)}")
    if target.numel() > 1 << 21:
        raise ValueError(f"at most 2^21 tokens in a call, got {target.numel()}")
    if apply_grad_on_fp32_main_grad:
        _main_grad_of(weight)
    flat = target.reshape(-1).contiguous()
    r = _REDUCTIONS[reduction]
    if ops._in_graph(input, weight):
        loss = ops._apply(_LinearCrossEntropy, 2, input, weight, flat, int(ignore_index), r, float(label_smoothing),
                                         weight if apply_grad_on_fp32_main_grad else None)
    else:
        loss = _forward(_rows(input.detach()), _rows(weight.detach()), flat, int(ignore_index), r, float(label_smoothing), False)[0]
    return loss if r else loss.reshape(target.shape)
