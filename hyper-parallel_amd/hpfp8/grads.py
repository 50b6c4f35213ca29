"""The global norm of a step's gradients, and their clipping by it: torch.nn.utils' three functions with their calling conventions.

A parameter's gradient is its ``main_grad`` where `apply_grad_on_fp32_main_grad` has made one (which torch's functions know nothing of), otherwise
its ``grad``.  The norm of all gradients is one pass over them and their clipping another, in one launch for each 250 tensors, with nothing read on
the host; tensors of bfloat16, float16 and float32 go together.  Orders other than 1, 2 and inf are refused, and ``foreach``, which chooses between
torch's two forms, is taken and changes nothing.
"""
from __future__ import annotations

import math
from typing import Iterable, List, Optional, Union

import torch

from . import _lib, ops
from .kept import _TYPES

_POWERS = {2.0: 2, 1.0: 1, math.inf: 0}


def _power(norm_type) -> int:
    norm_type = float(norm_type)
    if norm_type not in _POWERS:
        raise ValueError(f"norm_type must be 1, 2 or inf, got {norm_type}")
    return _POWERS[norm_type]


def _list_of(tensors) -> list:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _gradients(parameters) -> List[torch.Tensor]:
    """The parameters' gradients, each once however often a parameter is named."""
    found = {}
    for p in _list_of(parameters):
        grad, main_grad = p.grad, getattr(p, "main_grad", None)
        if main_grad is not None:
            if grad is not None and grad is not main_grad:
                raise ValueError("a parameter has a grad and a main_grad: its gradient is their sum, of which neither has the norm "
                                 "(add grad onto main_grad and set it to None)")
            grad = main_grad
        if grad is not None:
            found[id(grad)] = grad
    return list(found.values())


def _local(t: torch.Tensor) -> torch.Tensor:
    """This rank's part of a sharded tensor; any other as it is."""
    return t.to_local() if hasattr(t, "to_local") else t


def _check(tensors) -> None:
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"tensor {i} must be a torch.Tensor")
        if hasattr(t, "to_local"):
            raise TypeError(f"tensor {i} is sharded: take the norm of this rank's shards (to_local()), then that over the ranks, then clip_grads_with_norm_")
        if t.layout != torch.strided or t.dtype not in _TYPES:
            raise TypeError(f"tensor {i} must be a dense tensor of bfloat16, float16 or float32, got {t.dtype}, {t.layout}")
        ops._check_device(t, f"tensor {i}")


def _gapless(t: torch.Tensor) -> bool:
    """Whether t's elements are the memory from its start on, each once, in whatever order: what a norm and a factor need to know."""
    if t.is_contiguous():
        return True
    step = 1
    for stride, size in sorted((stride, size) for size, stride in zip(t.shape, t.stride()) if size > 1):
        if stride != step:
            return False
        step *= size
    return True


def _table(tensors):
    import ctypes
    n = max(len(tensors), 1)
    return ((ctypes.c_void_p * n)(*(t.data_ptr() for t in tensors)), (ctypes.c_int64 * n)(*(t.numel() for t in tensors)),
            (ctypes.c_int * n)(*(_TYPES[t.dtype] for t in tensors)), len(tensors))


def _raise_for_nonfinite(norm, norm_type) -> None:
    if not math.isfinite(float(norm)):
        raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` is non-finite, so it cannot be clipped. "
                           "To disable this error and scale the gradients by the non-finite norm anyway, set `error_if_nonfinite=False`")


@torch.no_grad()
def get_total_norm(tensors: Union[torch.Tensor, Iterable[torch.Tensor]], norm_type: float = 2.0, error_if_nonfinite: bool = False,
                   foreach: Optional[bool] = None) -> torch.Tensor:
    """torch.nn.utils.get_total_norm: the norm (of order 1, 2 or inf) of all elements of the tensors taken together, a 0-dim float32 tensor on the
    current GPU.  Sums are in 64 bits and in a fixed order: the same bits every time.  The norm over several ranks' shards is that of their norms
    (for order 2 the root of the sum of their squares): reduce it, then `clip_grads_with_norm_`."""
    tensors = _list_of(tensors)
    power = _power(norm_type)
    if torch.overrides.has_torch_function(tensors):
        return torch.overrides.handle_torch_function(get_total_norm, tensors, tensors, norm_type, error_if_nonfinite,
                                                     **({} if foreach is None else dict(foreach=foreach)))
    norm = None
    if ops._native is not None and tensors:
        device = ops._device()
        norm = ops._native.grad_norm(tensors, power, device, ops._raw_stream(device))
    if norm is None:
        ops._refuse_trace("get_total_norm", *tensors)
        _check(tensors)
        device = torch.device("cuda", torch.cuda.current_device())
        norm = torch.empty((), dtype=torch.float32, device=device)
        dense = [t if _gapless(t) else t.contiguous() for t in tensors]
        table = _table(dense)
        partial = torch.empty((_lib.load().hpfp8_grad_norm_partials(*table[1:]),), dtype=torch.float64, device=device)
        _lib.call("hpfp8_grad_norm", *table, power, ops._ptr(partial), ops._ptr(norm), ops._stream())
    if error_if_nonfinite:
        _raise_for_nonfinite(norm, norm_type)
    return norm


def _bound(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return max_norm


def _clip(grads, max_norm, total_norm) -> None:
    if torch.overrides.has_torch_function(grads):
        raise TypeError("clip_grads_with_norm_ takes local tensors: call it on the shards, with the norm over all of them")
    if not grads:
        return
    if ops._native is not None:
        device = ops._device()
        if ops._native.grad_clip(grads, total_norm, max_norm, False, device, ops._raw_stream(device)):
            return
    _check(grads)
    if hasattr(total_norm, "to_local"):
        raise TypeError("total_norm must be a number or a local tensor (full_tensor())")
    device = torch.device("cuda", torch.cuda.current_device())
    if not isinstance(total_norm, torch.Tensor):
        total_norm = torch.full((), float(total_norm), dtype=torch.float32, device=device)
    if total_norm.numel() != 1:
        raise ValueError(f"total_norm must be one number, got {tuple(total_norm.shape)}")
    norm = total_norm.detach().to(device, torch.float32)
    dense = [g if _gapless(g) else g.contiguous() for g in grads]
    torch.autograd.graph.increment_version([g for g, d in zip(grads, dense) if d is g])
    _lib.call("hpfp8_grad_clip", *_table(dense), ops._ptr(norm), max_norm, ops._stream())
    for g, d in zip(grads, dense):
        if d is not g:
            g.copy_(d)


@torch.no_grad()
def clip_grads_with_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, total_norm: torch.Tensor,
                          foreach: Optional[bool] = None) -> None:
    """torch.nn.utils.clip_grads_with_norm_: every gradient times min(1, max_norm / (total_norm + 1e-6)) in place, rounded once.  Where that is 1
    nothing is read or written (but of gradients with gaps between their elements, which are copied and copied back).  Gradients must not share memory.
    Of a sharded gradient (one with ``to_local()``) this rank's shard is scaled."""
    parameters, max_norm = _list_of(parameters), _bound(max_norm)
    if ops._native is not None and parameters and getattr(total_norm, "is_cuda", False):
        device = ops._device()
        if ops._native.grad_clip(parameters, total_norm, max_norm, True, device, ops._raw_stream(device)):
            return
    grads = [_local(g) for g in _gradients(parameters)]
    ops._refuse_trace("clip_grads_with_norm_", total_norm, *grads)
    _clip(grads, max_norm, total_norm)


@torch.no_grad()
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: Optional[bool] = None) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ for gradients in ``grad`` and in ``main_grad``: their total norm (a 0-dim float32 tensor), and the gradients
    scaled in place so that it is at most ``max_norm``.  Sharded gradients have no norm on one rank: `get_total_norm` of the shards, a reduction over
    the ranks and `clip_grads_with_norm_` take its place."""
    parameters, power, max_norm = _list_of(parameters), _power(norm_type), _bound(max_norm)
    if ops._native is not None and parameters and not error_if_nonfinite:
        device = ops._device()
        norm = ops._native.clip_grad_norm(parameters, max_norm, power, device, ops._raw_stream(device))
        if norm is not None:
            return norm
    grads = _gradients(parameters)
    ops._refuse_trace("clip_grad_norm_", *grads)
    norm = get_total_norm(grads, norm_type, error_if_nonfinite)
    _clip(grads, max_norm, norm)
    return norm
