"""The layer norm, the activations and the loss under what else torch does with a step: modes, transforms, traces, tensors of other kinds."""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu

WAYS = ["mode", "vmap", "grad", "forward_ad", "trace", "trace_inference", "batched_backward", "create_graph", "checkpoint", "reentrant", "dispatching_grad",
        "sparse_grad", "detect_anomaly", "in_place", "twice", "retained", "other_stream", "hooks"]


def randn(shape, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(torch.bfloat16).cuda()


def operator(name):
    """(function of tensors, tensors, gradient of the result)"""
    import hpfp8
    x, w = randn((48, 256), 1), randn((256,), 2)
    if name.startswith("norm"):
        return lambda a, b: hpfp8.layer_norm(a, 256, b, keep_8bit=name == "norm_kept"), (x, w), randn((48, 256), 3)
    if name.startswith("activation"):
        return lambda a: hpfp8.activation(a, "swiglu", keep_8bit=name == "activation_kept"), (x,), randn((48, 128), 4)
    head, target = randn((500, 256), 5, 0.1), torch.randint(500, (48,), generator=torch.Generator().manual_seed(6)).cuda()
    reduction = name.split("_")[1]
    go = torch.rand(48 if reduction == "none" else (), generator=torch.Generator().manual_seed(7)).cuda()
    # (the targets have a row each of a batch)
    return lambda a, b: hpfp8.linear_cross_entropy(a, b, target[:a.shape[0]], reduction=reduction, label_smoothing=0.1), (x, head), go


class Dispatching(torch.Tensor):
    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_subclass(cls, t)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raw = lambda a: a.as_subclass(torch.Tensor) if isinstance(a, cls) else a            # noqa: E731
        with torch._C._DisableTorchDispatch():
            return func(*[raw(a) for a in args], **(kwargs or {}))


def step(f, leaves, go, way):
    import torch.autograd.forward_ad as fwAD
    from torch.utils._python_dispatch import TorchDispatchMode
    from torch.utils.checkpoint import checkpoint

    class Pass(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x, rest = leaves[0], leaves[1:]
    if way == "mode":
        with Pass():
            y = f(*leaves)
            return (y, *torch.autograd.grad(y, leaves, go))
    if way == "vmap":
        return torch.func.vmap(f, in_dims=(0,) + (None,) * len(rest))(x.view(2, 24, 256), *rest)
    if way == "grad":
        return torch.func.grad(lambda a: f(a, *rest).float().sum())(x)
    if way == "forward_ad":
        with fwAD.dual_level():
            return f(fwAD.make_dual(x, torch.ones_like(x)), *rest)
    if way == "trace":
        return torch.jit.trace(f, leaves, check_trace=False)(*leaves)
    if way == "trace_inference":
        with torch.no_grad():
            traced = torch.jit.trace(f, tuple(t * 0 for t in leaves), check_trace=False)
            torch.full((1 << 20,), 7.0, device=x.device)            # (what the traced call's results may lie in)
            return traced(*leaves)
    y = checkpoint(f, *leaves, use_reentrant=way == "reentrant") if way in ("checkpoint", "reentrant") else None
    if way == "other_stream":
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = f(*leaves)
        torch.cuda.current_stream().wait_stream(side)
        y.record_stream(torch.cuda.current_stream())
    y = f(*leaves) if y is None else y
    if way == "batched_backward":
        return torch.autograd.grad(y, leaves, torch.stack((go, go)), is_grads_batched=True)
    if way == "create_graph":
        return (y, *torch.autograd.grad(y, leaves, go.requires_grad_(), create_graph=True))
    if way == "dispatching_grad":
        return torch.autograd.grad(y, leaves, Dispatching(go))
    if way == "sparse_grad":
        return torch.autograd.grad(y, leaves, go.to_sparse())
    if way == "in_place":
        y += 1
    if way in ("twice", "retained"):
        torch.autograd.grad(y, leaves, go, retain_graph=way == "retained")
    if way == "hooks":
        y.register_hook(lambda g: g * 2)
        y.grad_fn.register_hook(lambda grads_in, grads_out: tuple(None if g is None else g * 2 for g in grads_in))
    if way == "reentrant":
        for t in leaves:
            t.grad = None
        y.backward(go)
        return (y, *[t.grad for t in leaves])
    if way == "detect_anomaly":
        with torch.autograd.detect_anomaly(check_nan=True):
            return torch.autograd.grad(y, leaves, go)
    return (y, *torch.autograd.grad(y, leaves, go))


@pytest.mark.parametrize("name", ["norm", "norm_kept", "activation", "activation_kept", "loss_mean", "loss_none"])
@pytest.mark.parametrize("way", WAYS)
def test_the_native_host_path_has_the_python_functions_outcome(gpu, name, way, monkeypatch):
    """Values, or the error, are those that the Python autograd function gives by itself; where they are values, the plain step's."""
    from hpfp8 import ops
    assert ops._native is not None
    f, tensors, go = operator(name)

    def outcome(way):
        try:
            r = step(f, tuple(t.clone().requires_grad_() for t in tensors), go.detach().clone(), way)
        except Exception as e:
            return type(e), str(e).split("\n")[0].split(" is a view")[-1]       # (that message names the node, before these words)
        return [t.detach() for t in r] if isinstance(r, (tuple, list)) else [r.detach()]
    got = outcome(way)
    if way in ("mode", "trace", "trace_inference", "create_graph", "checkpoint", "reentrant", "dispatching_grad", "detect_anomaly", "retained", "other_stream",
               "in_place"):
        assert isinstance(got, list), got
        plain = outcome("plain")
        plain[0] = plain[0] + 1 if way == "in_place" else plain[0]
        plain = plain[:1] if way.startswith("trace") else (plain[1:] if len(got) < len(plain) else plain)
        assert len(got) == len(plain) and all(torch.equal(a, b) for a, b in zip(got, plain))
    monkeypatch.setattr(ops, "_native", types.SimpleNamespace(**{
        k: (lambda *a: None) if k in ("layer_norm", "activation", "linear_cross_entropy") else getattr(ops._native, k)
        for k in dir(ops._native) if not k.startswith("__")}))
    want = outcome(way)
    if isinstance(want, tuple):
        assert got == want or (way == "sparse_grad" and got[0] is want[0])           # (which of its operations comes first is the form's own)
    else:
        assert isinstance(got, list), got
        assert len(got) == len(want) and all(type(a) is type(b) and torch.equal(a, b) for a, b in zip(got, want))


def test_results_of_strided_inputs_can_be_written_to(gpu):
    """The Python forms take them; their results are no views."""
    import hpfp8
    x = randn((6, 40, 300), 8)[:, :, 3:259].requires_grad_()
    w, target = randn((50, 256), 9), torch.zeros(6, 40, dtype=torch.int64, device=gpu)
    for f in (lambda t: hpfp8.layer_norm(t, 256), lambda t: hpfp8.layer_norm(t, 256, keep_8bit=True), lambda t: hpfp8.activation(t, "silu"),
              lambda t: hpfp8.activation(t, "swiglu", keep_8bit=False), lambda t: hpfp8.linear_cross_entropy(t, w, target, reduction="none")):
        y = f(x)
        want = torch.autograd.grad(f(x).sum(), x)[0]
        y += 1
        assert torch.equal(y, f(x) + 1) and torch.equal(torch.autograd.grad(y.sum(), x)[0], want)


@pytest.mark.parametrize("name", ["norm", "norm_kept", "activation", "activation_kept", "loss_mean", "loss_none"])
@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_refused_and_not_dropped(gpu, name, grad):
    """Forward mode with tensors that require no gradient; without a tangent the level changes nothing."""
    import torch.autograd.forward_ad as fwAD
    f, tensors, _ = operator(name)
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        for i in range(len(tensors)):
            dual = [fwAD.make_dual(t, torch.ones_like(t)) if k == i else t for k, t in enumerate(tensors)]
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward mode"):
                f(*dual)
        inside = f(*tensors)
    assert torch.equal(inside, f(*tensors))
