"""What the root-mean-square norm, the linear in 8-bit integers and the gradients' norm refuse, without a GPU: arguments are looked at before
anything is launched."""
import ctypes
import math

import pytest
import torch

BF16 = torch.bfloat16


@pytest.fixture()
def p():
    buf = (ctypes.c_char * 8192)()
    yield (ctypes.cast(buf, ctypes.c_void_p).value + 255) & ~255


def c(name, *args):
    from hpfp8 import _lib
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.hpfp8_last_error().decode()


def test_rms_norm(p):
    f, b = "hpfp8_rms_norm_forward", "hpfp8_rms_norm_backward"
    assert c(f, p, 8, None, 0, 0, 4, 16385, None, 0, 1e-5, None, p, None, None)[0] == -2
    assert c(f, p, 8, None, 0, 0, 4, 1 << 40, None, 0, 1e-5, None, p, None, None)[0] == -2
    assert c(f, p, 8, None, 0, 0, 4, 0, None, 0, 1e-5, None, p, None, None)[0] == -2
    assert c(f, p, 8, None, 0, 0, -1, 8, None, 0, 1e-5, None, p, None, None)[0] == -2
    assert c(f, p, -8, None, 0, 0, 4, 8, None, 0, 1e-5, None, p, None, None)[0] == -2
    assert c(f, p, 8, p, -8, 0, 4, 8, None, 0, 1e-5, p, p, None, None)[0] == -2
    assert c(f, p, 8, None, 0, 3, 4, 8, None, 0, 1e-5, None, p, None, None)[0] == -1
    assert c(f, p, 8, None, 0, 0, 4, 8, p, -1, 1e-5, None, p, None, None)[0] == -1
    assert c(f, p, 8, p, 8, 0, 4, 8, None, 0, 1e-5, None, p, None, None)[0] == -1          # a residual without a sum
    assert c(f, p, 8, None, 0, 0, 4, 8, None, 0, 1e-5, p, p, None, None)[0] == -1
    assert c(f, None, 8, None, 0, 0, 4, 8, None, 0, 1e-5, None, p, None, None)[0] == -1
    assert c(f, p + 1, 8, None, 0, 0, 4, 8, None, 0, 1e-5, None, p, None, None)[0] == -3
    assert c(f, p, 8, p + 2, 8, 1, 4, 8, None, 0, 1e-5, p, p, None, None)[0] == -3
    assert c(f, p, 8, None, 0, 0, 4, 8, p + 2, 1, 1e-5, None, p, None, None)[0] == -3
    assert c(f, None, 8, None, 0, 0, 0, 8, None, 0, 1e-5, None, None, None, None)[0] == 0
    for q, more in (("hpfp8_rms_norm_quantize_1x128_kmajor", (0,)), ("hpfp8_rms_norm_quantize_int8", ())):
        assert c(q, p, 8, None, 0, 0, 4, 100, None, 0, 1e-5, *more, None, p, p, None)[0] == -2
        assert c(q, p, 8, None, 0, 0, 4, 16512, None, 0, 1e-5, *more, None, p, p, None)[0] == -2
        assert c(q, p, 128, None, 0, 0, 4, 128, None, 0, 1e-5, *more, None, p, None, None)[0] == -1
        assert c(q, None, 128, None, 0, 0, 0, 128, None, 0, 1e-5, *more, None, None, None, None)[0] == 0
    assert c(b, p, 8, p, 8, None, 0, p, 0, 4, 16385, None, 0, p, p, p, None)[0] == -2
    assert c(b, p, 8, p, 8, None, 0, None, 0, 4, 8, None, 0, p, p, p, None)[0] == -1
    assert c(b, p, 8, p, 8, None, 0, p, 0, 4, 8, None, 0, p, p, None, None)[0] == -1       # no workspace
    assert c(b, p, -8, p, 8, None, 0, p, 0, 4, 8, None, 0, p, p, p, None)[0] == -2
    assert c(b, p, 8, p, 8, p + 1, 8, p, 0, 4, 8, None, 0, p, p, p, None)[0] == -3
    assert c(b, p, 8, p, 8, None, 0, p, 0, 4, 8, None, 1, p, p + 2, p, None)[0] == -3
    assert c(b, None, 8, None, 8, None, 0, None, 0, 0, 8, None, 0, None, None, None, None)[0] == 0
    assert c("hpfp8_rms_norm_partials", 0, 8)[0] == 0 and c("hpfp8_rms_norm_partials", 1, 16385)[0] == 0
    assert c("hpfp8_rms_norm_partials", 1 << 40, 4096)[0] == 256 and c("hpfp8_rms_norm_partials", 1 << 40, 2048)[0] == 512


def test_int8(p):
    q, g = "hpfp8_quantize_int8", "hpfp8_gemm_int8"
    assert c(q, p, 3, 4, 128, 128, None, p, p, None)[0] == -1
    assert c(q, p, 0, 4, 100, 128, None, p, p, None)[0] == -2
    assert c(q, p, 0, 4, 131072, 131072, None, p, p, None)[0] == -2
    assert c(q, p, 0, -4, 128, 128, None, p, p, None)[0] == -2
    assert c(q, p, 0, 4, 128, -128, None, p, p, None)[0] == -2
    assert c(q, p, 0, 4, 128, 128, None, p, None, None)[0] == -1
    assert c(q, p + 1, 0, 4, 128, 128, None, p, p, None)[0] == -3
    assert c(q, p, 0, 4, 128, 128, p + 2, p, p, None)[0] == -3
    assert c(q, None, 0, 0, 128, 128, None, None, None, None)[0] == 0
    assert c(g, p, 128, p, p, 128, p, 4, 100, 128, None, p, 128, 0, None)[0] == -2
    assert c(g, p, 128, p, p, 128, p, 4, 128, 100, None, p, 128, 0, None)[0] == -2
    assert c(g, p, 131072, p, p, 131072, p, 4, 128, 131072, None, p, 128, 0, None)[0] == -2       # sums past 32 bits
    assert c(g, p, 120, p, p, 128, p, 4, 128, 128, None, p, 128, 0, None)[0] == -2
    assert c(g, p, 128, p, p, 136, p, 4, 128, 128, None, p, 128, 0, None)[0] == -2
    assert c(g, p, 128, p, p, 128, p, 4, 128, 128, None, p, 64, 0, None)[0] == -2
    assert c(g, p, 128, p, p, 128, p, 4, 128, 128, None, p, 130, 2, None)[0] == -3
    assert c(g, p, 128, p, p, 128, p, 4, 128, 128, None, p, 128, 3, None)[0] == -1
    assert c(g, p, 128, None, p, 128, p, 4, 128, 128, None, p, 128, 0, None)[0] == -1
    assert c(g, p + 1, 128, p, p, 128, p, 4, 128, 128, None, p, 128, 0, None)[0] == -3
    assert c(g, p, 128, p, p, 128, p + 4, 4, 128, 128, None, p, 128, 0, None)[0] == -3
    assert c(g, p, 128, p + 2, p, 128, p, 4, 128, 128, None, p, 128, 0, None)[0] == -3
    assert c(g, p, 128, p, p, 128, p, 4, 128, 128, p + 8, p, 128, 0, None)[0] == -3
    assert c(g, None, 128, None, None, 128, None, 0, 128, 128, None, None, 128, 0, None)[0] == 0


def table(ptrs, numels, types):
    n = max(len(ptrs), 1)
    return (ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*numels), (ctypes.c_int * n)(*types), len(ptrs)


def test_gradients(p):
    f, clip, size = "hpfp8_grad_norm", "hpfp8_grad_clip", "hpfp8_grad_norm_partials"
    one = table([p], [8], [0])
    assert c(f, *one, 3, p, p, None)[0] == -1
    assert c(f, *one, 2, None, p, None)[0] == -1
    assert c(f, *one, 2, p, None, None)[0] == -1
    assert c(f, *table([p], [8], [3]), 2, p, p, None)[0] == -1
    assert c(f, *table([p], [-8], [0]), 2, p, p, None)[0] == -2
    assert c(f, *table([p], [1 << 50], [0]), 2, p, p, None)[0] == -2
    assert c(f, *table([None], [8], [0]), 2, p, p, None)[0] == -1
    assert c(f, *table([p + 1], [8], [0]), 2, p, p, None)[0] == -3
    assert c(f, *table([p + 2], [8], [1]), 2, p, p, None)[0] == -3
    assert c(f, None, None, None, 1, 2, p, p, None)[0] == -1
    assert c(f, *one[:3], -1, 2, p, p, None)[0] == -2
    assert c(clip, *one, None, 1.0, None)[0] == -1
    assert c(clip, *table([p, p], [8, 8], [0, 0]), p, 1.0, None)[0] == -1
    assert c(clip, *table([p, p + 14], [8, 8], [0, 0]), p, 1.0, None)[0] == -1
    assert c(clip, *table([p + 64, p], [8, 20], [0, 1]), p, 1.0, None)[0] == -1
    assert "share memory" in c(clip, *table([p + 64, p], [8, 20], [0, 1]), p, 1.0, None)[1]
    assert c(clip, *table([], [], []), None, 1.0, None)[0] == 0
    assert c(clip, *table([p, p], [0, 0], [0, 1]), p, 1.0, None)[0] == 0
    assert c(size, *table([], [], [])[1:])[0] == 0 and c(size, *one[1:])[0] == 1
    _, numels, types, n = table([p] * 3, [1 << 40, 1, 0], [1, 0, 0])
    assert 1000 < c(size, numels, types, n)[0] < 20000                   # (work is dealt out by bytes)


def test_tensors_that_are_not_on_the_gpu_and_wrong_arguments():
    import hpfp8
    x, w = torch.zeros(4, 256, dtype=BF16), torch.ones(256, dtype=BF16)
    for f, error in ((lambda: hpfp8.rms_norm(x, 256, w), ValueError), (lambda: hpfp8.rms_norm(3, 256), TypeError),
                     (lambda: hpfp8.rms_norm(x.double(), 256), TypeError), (lambda: hpfp8.rms_norm_quantize_1x128(x, w), ValueError),
                     (lambda: hpfp8.rms_norm_quantize_int8(x), ValueError), (lambda: hpfp8.quantize_int8(x), ValueError),
                     (lambda: hpfp8.quantize_weight_int8(x[:3]), ValueError), (lambda: hpfp8.quantize_weight_int8(w), ValueError),
                     (lambda: hpfp8.gemm_int8(x, x, x, x), TypeError), (lambda: hpfp8.int8_linear(x, w), TypeError),
                     (lambda: hpfp8.int8_linear(x, hpfp8.Int8Weight(torch.zeros(128, 256, dtype=torch.int8), torch.ones(128))), ValueError),
                     (lambda: hpfp8.get_total_norm([x], 5), ValueError), (lambda: hpfp8.get_total_norm([x], math.nan), ValueError),
                     (lambda: hpfp8.Int8Linear(256, 100), ValueError), (lambda: hpfp8.Int8Linear(0, 128), ValueError)):
        with pytest.raises(error):
            f()


@pytest.fixture()
def as_if_on_the_gpu(monkeypatch):
    from hpfp8 import ops
    monkeypatch.setattr(ops, "_check_device", lambda *a: None)


def test_operands_that_do_not_go_together(as_if_on_the_gpu):
    import hpfp8
    x, w = torch.zeros(4, 256, dtype=BF16), torch.ones(256, dtype=BF16)
    for f, error in ((lambda: hpfp8.rms_norm(x, 128), ValueError), (lambda: hpfp8.rms_norm(x, (4, 4, 256)), ValueError),
                     (lambda: hpfp8.rms_norm(x, 256, w[:128]), ValueError), (lambda: hpfp8.rms_norm(x, 256, w.double()), TypeError),
                     (lambda: hpfp8.rms_norm(x, 256, residual=x.float()), TypeError), (lambda: hpfp8.rms_norm(x, 256, residual=x[:1]), ValueError),
                     (lambda: hpfp8.rms_norm(torch.zeros(1, 16385, dtype=BF16), 16385), ValueError),
                     (lambda: hpfp8.rms_norm_quantize_int8(x[:, :100]), ValueError), (lambda: hpfp8.rms_norm_quantize_1x128(x, w, residual=x[0]), ValueError),
                     (lambda: hpfp8.rms_norm_quantize_int8(x.clone().requires_grad_()), RuntimeError),
                     (lambda: hpfp8.rms_norm_quantize_1x128(x, w.clone().requires_grad_(), residual=x), RuntimeError)):
        with pytest.raises(error):
            f()


def test_subclasses_are_handed_the_call():
    import hpfp8
    seen = []

    class Recording(torch.Tensor):
        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            seen.append((func, len(args), kwargs))
            return "handed"
    x = torch.zeros(4, 256).as_subclass(Recording)
    y = torch.zeros(4, 256)
    w8 = hpfp8.Int8Weight(torch.zeros(128, 256, dtype=torch.int8), torch.ones(128))
    assert hpfp8.rms_norm(x, 256) == "handed" and seen[-1] == (hpfp8.rms_norm, 2, {})
    assert hpfp8.rms_norm(y, 256, eps=1e-3, residual=x) == "handed" and seen[-1] == (hpfp8.rms_norm, 2, dict(eps=1e-3, residual=x))
    assert hpfp8.int8_linear(x, w8) == "handed" and seen[-1] == (hpfp8.int8_linear, 3, {})
    assert hpfp8.get_total_norm([y, x]) == "handed" and seen[-1][0].__name__ == "get_total_norm"
    p = torch.nn.Parameter(torch.zeros(4, 256))
    p.main_grad = x
    with pytest.raises(TypeError, match="local tensors"):
        hpfp8.clip_grads_with_norm_(p, 1.0, torch.ones(()))


def test_saved_tensors_that_a_hook_handed_back_as_something_else(as_if_on_the_gpu):
    from hpfp8 import norm
    from hpfp8.int8 import _int8_backward
    go, s, rstd = torch.zeros(4, 256, dtype=BF16), torch.zeros(4, 256, dtype=BF16), torch.ones(4)
    for kept, other, weight in ((s[:3], rstd, None), (s.float(), rstd, None), (s, rstd[:2], None), (s, rstd.double(), None), (s, rstd, torch.ones(5, dtype=BF16))):
        with pytest.raises(ValueError, match="came back"):
            norm._rms_backward(go, None, kept, other, weight, 256, (4, 256), 0, None if weight is None else (256,), 0, False)
    codes, scale = torch.zeros(128, 256, dtype=torch.int8), torch.ones(128)
    for q, sc in ((codes[:64], scale), (codes.float(), scale), (codes, scale[:5]), (codes, scale.double())):
        with pytest.raises(ValueError, match="came back"):
            _int8_backward(torch.zeros(4, 128, dtype=BF16), q, sc, False, (4, 256))


@pytest.mark.parametrize("way", ["deepcopy", "copy", "pickle"])
@pytest.mark.parametrize("stale", [False, True])
def test_a_copied_int8_layer_knows_whether_its_transposed_codes_are_its_codes(way, stale):
    import copy
    import pickle

    import hpfp8
    copied = {"deepcopy": copy.deepcopy, "copy": copy.copy, "pickle": lambda layer: pickle.loads(pickle.dumps(layer))}[way]
    for writes in range(4):
        layer = hpfp8.Int8Linear(128, 256, with_transpose=True)
        layer.weight_codes.copy_(torch.arange(256 * 128).reshape(256, 128) % 251 - 125)
        for _ in range(writes):
            layer.weight_codes.add_(1)
        layer.refresh()
        if stale:
            layer.weight_codes.add_(1)
        there = copied(layer)
        assert torch.equal(there.weight_codes, layer.weight_codes) and there._up_to_date() == (not stale)
        there.load_state_dict(layer.state_dict())
        assert torch.equal(there.weight_codes_t, layer.weight_codes.t()) and there._up_to_date()
        there.weight_codes.add_(1)
        assert not there._up_to_date()
        if way != "copy":
            assert layer._up_to_date() == (not stale)


@pytest.fixture()
def launched(as_if_on_the_gpu, monkeypatch):
    """Launches written down instead of made."""
    from hpfp8 import _lib, ops
    seen = []
    monkeypatch.setattr(ops, "_native", None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_check_f32", lambda t, name: t)
    monkeypatch.setattr(_lib, "call", lambda name, *a: seen.append(name))
    return seen


def int8_calls():
    """(name, function of a tensor in 16 or 32 bits, that tensor)"""
    import hpfp8
    codes, scale = torch.zeros(128, 256, dtype=torch.int8), torch.ones(128)
    return [("quantize_int8", hpfp8.quantize_int8, torch.zeros(128, 256, dtype=BF16)),
            ("quantize_int8", lambda t: hpfp8.quantize_int8(torch.zeros(4, 256, dtype=BF16), column_scale=t), torch.ones(256)),
            ("gemm_int8", lambda t: hpfp8.gemm_int8(codes, t, codes, scale), scale), ("gemm_int8", lambda t: hpfp8.gemm_int8(codes, scale, codes, t), scale),
            ("gemm_int8", lambda t: hpfp8.gemm_int8(codes, scale, codes, None, t), torch.zeros(128, dtype=BF16))]


@pytest.mark.parametrize("case", range(5))
def test_int8_operators_have_no_place_in_a_trace_and_no_tangents(launched, case):
    """A trace would keep their empty results and none of their launches."""
    import torch.autograd.forward_ad as fwAD
    name, f, t = int8_calls()[case]
    with pytest.raises(RuntimeError, match=f"{name} has no place in a trace"):
        torch.jit.trace(f, (t,), check_trace=False)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no place in a trace"):
        torch.jit.trace(f, (t,), check_trace=False)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), fwAD.dual_level():
            with pytest.raises(RuntimeError, match=f"{name} .*forward mode"):
                f(fwAD.make_dual(t, torch.ones_like(t)))
            assert not launched
            f(t)                                             # (a level without a tangent changes nothing)
            assert launched.pop()
    f(t)
    assert launched


def test_int8_linear_in_a_trace_launches_inside_its_function(launched):
    import hpfp8
    w8 = hpfp8.Int8Weight(torch.zeros(128, 256, dtype=torch.int8), torch.ones(128))
    x = torch.zeros(4, 256, dtype=BF16)
    for grad in (True, False):
        with torch.set_grad_enabled(grad):
            traced = torch.jit.trace(lambda t: hpfp8.int8_linear(t, w8), (x,), check_trace=False)
            launched.clear()
            traced(x)
        assert launched == ["hpfp8_quantize_int8", "hpfp8_gemm_int8"]


@pytest.mark.parametrize("which", ["sa", "sb", "bias"])
def test_int8_products_have_no_gradient_for_scales_and_bias(launched, which):
    import hpfp8
    codes = torch.zeros(128, 256, dtype=torch.int8)
    given = dict(sa=torch.ones(128), sb=torch.ones(128), bias=torch.zeros(128, dtype=BF16))
    given[which].requires_grad_()
    with pytest.raises(ValueError, match=f"no gradient for {which}"):
        hpfp8.gemm_int8(codes, given["sa"], codes, given["sb"], given["bias"])
    assert not launched
    with torch.no_grad():
        assert not hpfp8.gemm_int8(codes, given["sa"], codes, given["sb"], given["bias"]).requires_grad
    if which == "sb":
        for x in (torch.zeros(4, 256, dtype=BF16), torch.zeros(4, 256, dtype=BF16).requires_grad_()):
            with pytest.raises(ValueError, match="no gradient for the weight's scales"):
                hpfp8.int8_linear(x, hpfp8.Int8Weight(codes, given["sb"]))
            with torch.no_grad():
                hpfp8.int8_linear(x, hpfp8.Int8Weight(codes, given["sb"]))


def test_gradients_norms_have_no_place_in_a_trace_and_no_tangents(launched):
    import hpfp8
    import torch.autograd.forward_ad as fwAD

    def clip(f):
        def call(t):
            p = torch.nn.Parameter(torch.zeros(8))
            p.main_grad = t
            f(p)
            return t + 1
        return call
    for name, f in (("get_total_norm", lambda t: hpfp8.get_total_norm([t])), ("clip_grads_with_norm_", clip(lambda p: hpfp8.clip_grads_with_norm_(p, 1.0, torch.ones(())))),
                    ("clip_grad_norm_", clip(lambda p: hpfp8.clip_grad_norm_(p, 1.0)))):
        with pytest.raises(RuntimeError, match=f"{name} has no place in a trace"):
            torch.jit.trace(f, (torch.ones(8),), check_trace=False)
        with fwAD.dual_level(), pytest.raises(RuntimeError, match=f"{name} .*forward mode"):
            f(fwAD.make_dual(torch.ones(8), torch.ones(8)))
    assert not launched


def test_sharded_gradients_without_a_norm_over_the_ranks_are_refused(launched):
    import hpfp8

    class Sharded(torch.Tensor):
        def to_local(self):
            return self.as_subclass(torch.Tensor)
        __torch_function__ = torch._C._disabled_torch_function_impl
    g = torch.zeros(8).as_subclass(Sharded)
    p = torch.nn.Parameter(torch.zeros(8))
    p.main_grad = g
    for f in (lambda: hpfp8.get_total_norm([torch.zeros(8), g]), lambda: hpfp8.clip_grad_norm_(p, 1.0)):
        with pytest.raises(TypeError, match="sharded"):
            f()
    with pytest.raises(TypeError, match="total_norm must be"):
        hpfp8.clip_grads_with_norm_(p, 1.0, g)
    assert not launched


def test_the_gradients_functions_take_torchs_arguments(launched):
    """By name and by place; foreach chooses between torch's own two forms and changes nothing here."""
    import inspect
    import hpfp8
    for name in ("get_total_norm", "clip_grads_with_norm_", "clip_grad_norm_"):
        ours, theirs = (inspect.signature(getattr(m, name)).parameters for m in (hpfp8, torch.nn.utils))
        assert [(p.name, p.default, p.kind) for p in ours.values()] == [(p.name, p.default, p.kind) for p in theirs.values()]
    x = torch.zeros(8, dtype=torch.float64)
    p = torch.nn.Parameter(torch.zeros(8))
    for foreach in (True, False, None):
        for f in (lambda: hpfp8.get_total_norm([x], 2.0, False, foreach), lambda: hpfp8.get_total_norm([x], foreach=foreach)):
            with pytest.raises(TypeError, match="tensor 0 must be a dense tensor"):
                f()
        assert hpfp8.clip_grads_with_norm_([p], 1.0, torch.ones(()), foreach) is None and hpfp8.clip_grads_with_norm_([p], 1.0, 1.0, foreach=foreach) is None
    assert not launched


def test_a_subclass_is_handed_the_norm_with_foreach():
    import hpfp8
    seen = []

    class Recording(torch.Tensor):
        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            seen.append((func.__name__, args[1:], kwargs))
            return "handed"
    x = torch.zeros(4).as_subclass(Recording)
    assert hpfp8.get_total_norm([x], 1.0) == "handed" and hpfp8.get_total_norm([x], 1.0, foreach=True) == "handed"
    assert seen == [("get_total_norm", (1.0, False), {}), ("get_total_norm", (1.0, False), dict(foreach=True))]
