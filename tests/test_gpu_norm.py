"""Layer norm against 64 bits, element by element, with bounds that count the roundings."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
U = 2.0 ** -24


def make(rows, cols, dtype, wdtype, seed, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, cols), generator=g) * 2 + offset).to(dtype)
    w = (1 + 0.2 * torch.randn((cols,), generator=g)).to(wdtype)
    b = (0.3 * torch.randn((cols,), generator=g)).to(wdtype)
    go = torch.randn((rows, cols), generator=g).to(dtype)
    return x, w, b, go


def reference(x, w, b, go, eps, hat=None):
    """(y, dx, dw, db, hat, rstd) in 64 bits; `hat` where the backward takes another than x's."""
    x, go = x.double(), go.double()
    w = torch.ones(x.shape[1], dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(x.shape[1], dtype=torch.float64) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    own = (x - mean) * rstd
    y = own * w + b
    hat = own if hat is None else hat
    u = go * w
    dx = rstd * (u - u.mean(1, keepdim=True) - hat * (u * hat).mean(1, keepdim=True))
    return y, dx, (go * hat).sum(0), go.sum(0), hat, rstd


def bounds(x, w, b, go, ref):
    """What fp32 sums may be off by.  A row's sum adds at most 32 values in a thread and then six steps of a tree and eight waves:
    under 64 roundings of the sizes that are added; a statistic enters every value of the row through x - mean, whose size is that of
    the row's largest |x| times rstd (`reach`).  A column's sum adds at most `chain` values one after the other."""
    y, dx, dw, db, hat, rstd = ref
    rows = x.shape[0]
    w = torch.ones(x.shape[1], dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(x.shape[1], dtype=torch.float64) if b is None else b.double()
    x, go = x.double(), go.double()
    reach = x.abs().amax(1, keepdim=True) * rstd + hat.abs()
    u = (go * w).abs()
    by = 96 * U * (w.abs() * reach + b.abs())
    bx = 192 * U * rstd * (u + u.mean(1, keepdim=True) + reach * (u * reach).mean(1, keepdim=True))
    chain = rows / 256 + 8 + 16 + 16
    bw = (chain + 96) * U * (go.abs() * reach).sum(0)
    bb = chain * U * go.abs().sum(0)
    return by, bx, bw, bb


def close(got, want, bound, dtype):
    assert got.dtype == dtype
    off = (got.double().cpu() - want).abs()
    limit = HALF[dtype] * want.abs() + bound + 2.0 ** -24 * (dtype == torch.float16)
    assert (off <= limit).all(), float((off - limit).max())


CASES = [  # rows, cols
    (1, 1), (1, 8), (5, 3), (3, 64), (9, 127), (33, 512), (20, 513), (17, 1024), (16, 1025), (300, 1027), (7, 4096), (13, 4100), (31, 7168),
    (5, 8192), (3, 8200), (9, 16384), (2, 16381), (1100, 40), (2500, 136), (40, 9), (70, 128), (33, 129), (21, 200), (65, 256), (12, 257), (11, 2047), (6, 2048), (5, 2055), (6, 8191), (3, 8193)]


@pytest.mark.parametrize("rows,cols", CASES)
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32),
                                          (torch.bfloat16, torch.float32)])
def test_forward_and_backward(gpu, rows, cols, dtype, wdtype):
    import hpfp8
    x, w, b, go = make(rows, cols, dtype, wdtype, 1)
    xg, wg, bg = (t.to(gpu).requires_grad_() for t in (x, w, b))
    y = hpfp8.layer_norm(xg, (cols,), wg, bg, 1e-5)
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), go.to(gpu))
    ref = reference(x, w, b, go, 1e-5)
    by, bx, bw, bb = bounds(x, w, b, go, ref)
    close(y.detach(), ref[0], by, dtype)
    close(dx, ref[1], bx, dtype)
    close(dw, ref[2], bw, wdtype)
    close(db, ref[3], bb, wdtype)
    with torch.no_grad():
        assert torch.equal(hpfp8.layer_norm(xg, (cols,), wg, bg, 1e-5), y)


@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 3), (9, 127), (33, 512), (20, 513), (300, 1027), (7, 4100), (31, 7168), (9, 16384), (2, 16381), (40, 9), (33, 129), (21, 253), (5, 2055)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_kept_in_8_bits(gpu, rows, cols, dtype):
    import hpfp8
    from hpfp8 import norm
    x, w, b, go = make(rows, cols, dtype, dtype, 2)
    xg, wg, bg = (t.to(gpu).requires_grad_() for t in (x, w, b))
    y = hpfp8.layer_norm(xg, (cols,), wg, bg, 1e-5, keep_8bit=True)
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), go.to(gpu))
    assert torch.equal(y.detach(), hpfp8.layer_norm(xg.detach(), (cols,), wg.detach(), bg.detach()))
    codes, scale_inv = norm._forward(xg.detach(), wg.detach(), bg.detach(), 1e-5, True, True)[3:]
    kept = (codes.float() * scale_inv.repeat_interleave(128, 1)[:, :cols]).double().cpu()
    exact = reference(x, w, b, go, 1e-5)
    # each value within half a step of E4M3 (2^-4 relative; 2^-10 of the scale below 2^-6) and of what fp32 makes of it
    reach = x.double().abs().amax(1, keepdim=True) * exact[5] + exact[4].abs()
    scale = scale_inv.double().cpu().repeat_interleave(128, 1)[:, :cols]
    assert ((kept - exact[4]).abs() <= torch.maximum(2.0 ** -4 * exact[4].abs(), 2.0 ** -10 * scale) + 128 * U * reach).all()
    ref = reference(x, w, b, go, 1e-5, hat=kept)
    by, bx, bw, bb = bounds(x, w, b, go, ref)
    close(dx, ref[1], bx, dtype)
    close(dw, ref[2], bw, dtype)
    close(db, ref[3], bb, dtype)


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_without_a_vector(gpu, weight, bias):
    import hpfp8
    x, w, b, go = make(40, 300, torch.bfloat16, torch.bfloat16, 3)
    w, b = w if weight else None, b if bias else None
    leaves = [t.to(gpu).requires_grad_() if t is not None else None for t in (x, w, b)]
    y = hpfp8.layer_norm(leaves[0], 300, leaves[1], leaves[2])
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], go.to(gpu))
    ref = reference(x, w, b, go, 1e-5)
    by, bx, bw, bb = bounds(x, w, b, go, ref)
    close(y.detach(), ref[0], by, torch.bfloat16)
    close(grads[0], ref[1], bx, torch.bfloat16)
    if weight:
        close(grads[1], ref[2], bw, torch.bfloat16)
    if bias:
        close(grads[-1], ref[3], bb, torch.bfloat16)


def test_an_offset_many_times_the_spread(gpu):
    """x = 1000 + N(0, 1) in fp32: the variance is taken around the mean, so hat is as exact as x - mean is."""
    import hpfp8
    x, w, b, go = make(16, 7168, torch.float32, torch.float32, 4)
    x = x * 0.5 + 1000.0
    y = hpfp8.layer_norm(x.to(gpu), 7168, w.to(gpu), b.to(gpu))
    ref = reference(x, w, b, go, 1e-5)
    close(y, ref[0], bounds(x, w, b, go, ref)[0], torch.float32)
    # E[x^2] - E[x]^2 in fp32 would be off by 2^-24 1e6 = 0.06 of a variance of 1
    assert float((y.double().cpu() - ref[0]).abs().max()) < 5e-3


def test_constant_rows_and_rows_that_are_not_finite(gpu):
    import hpfp8
    x, w, b, _ = make(6, 1000, torch.bfloat16, torch.bfloat16, 5)
    x[1] = 3.0
    x[2] = 0.0
    x[3, 17] = math.nan
    x[4, 999] = math.inf
    xg, wg, bg = (t.to(gpu).requires_grad_() for t in (x, w, b))
    y = hpfp8.layer_norm(xg, 1000, wg, bg)
    assert torch.equal(y[1], bg) and torch.equal(y[2], bg)
    assert y[3].isnan().all() and y[4].isnan().all() and y[[0, 5]].isfinite().all()
    dx, = torch.autograd.grad(y, xg, torch.ones_like(y))
    assert dx[3].isnan().all() and dx[[0, 1, 2, 5]].isfinite().all()


def test_several_dimensions_strides_and_starts_between_vectors(gpu):
    import hpfp8
    base = torch.randn((4, 6, 5, 77), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(gpu)
    w, b = torch.randn((5, 77)).to(torch.bfloat16).to(gpu), torch.randn((5, 77)).to(torch.bfloat16).to(gpu)
    assert torch.equal(hpfp8.layer_norm(base, (5, 77), w, b).reshape(24, 385), hpfp8.layer_norm(base.reshape(24, 385), 385, w.reshape(-1), b.reshape(-1)))
    flat = base.reshape(24, 385)
    for x in (flat[:, 1:], flat[::3, :384], flat.t()[:, :20], flat[:1].expand(7, 385)):
        c = x.shape[1]
        leaves = [t.detach().requires_grad_() for t in (x, w.reshape(-1)[:1].expand(c), b.reshape(-1)[:c])]
        copies = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in leaves]
        got, want = (hpfp8.layer_norm(t[0], c, t[1], t[2]) for t in (leaves, copies))
        assert torch.equal(got, want)
        wide = torch.randn((x.shape[0], c + 3), generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).to(gpu)
        for go in (wide[:, 3:], wide[:1, :1].expand(x.shape[0], c)):
            for p, q in zip(torch.autograd.grad(got, leaves, go, retain_graph=True), torch.autograd.grad(want, copies, go.contiguous(), retain_graph=True)):
                assert torch.equal(p, q)


def test_no_rows(gpu):
    import hpfp8
    for keep in (False, True):
        x = torch.empty((0, 256), device=gpu, dtype=torch.bfloat16, requires_grad=True)
        w, b = (torch.ones(256, device=gpu, dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
        y = hpfp8.layer_norm(x, 256, w, b, keep_8bit=keep)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
        assert dx.shape == (0, 256) and (dw == 0).all() and (db == 0).all()


def test_the_same_bits_every_time_and_module_form(gpu):
    import hpfp8
    x, w, b, go = make(5000, 640, torch.bfloat16, torch.bfloat16, 8)
    layer = hpfp8.LayerNorm(640, device=gpu)
    torch_layer = torch.nn.LayerNorm(640, device=gpu, dtype=torch.bfloat16)
    torch_layer.load_state_dict({"weight": w, "bias": b})
    layer.load_state_dict(torch_layer.state_dict())
    first = None
    for _ in range(3):
        xg = x.to(gpu).requires_grad_()
        y = layer(xg)
        grads = torch.autograd.grad(y, (xg, layer.weight, layer.bias), go.to(gpu))
        first = first or (y.detach(),) + grads
        assert all(torch.equal(p, q) for p, q in zip(first, (y.detach(),) + grads))
    assert "keep_8bit" in repr(layer)


def test_gradients_of_only_some_inputs(gpu):
    import hpfp8
    x, w, b, go = (t.to(gpu) for t in make(30, 256, torch.bfloat16, torch.bfloat16, 9))
    whole = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(hpfp8.layer_norm(whole[0], 256, whole[1], whole[2]), whole, go)
    for k in range(3):
        some = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(hpfp8.layer_norm(some[0], 256, some[1], some[2]), some[k], go)
        assert torch.equal(got, want[k])


def test_gradient_against_differences(gpu):
    import hpfp8
    x, w, b, go = (t.to(gpu) for t in make(2, 24, torch.float32, torch.float32, 10))
    x.requires_grad_()
    dx, = torch.autograd.grad(hpfp8.layer_norm(x, 24, w, b), x, go)
    step = 1e-2
    with torch.no_grad():
        for c in range(24):
            e = torch.zeros_like(x)
            e[:, c] = step
            d = ((hpfp8.layer_norm(x + e, 24, w, b) - hpfp8.layer_norm(x - e, 24, w, b)) * go).sum(1) / (2 * step)
            # fp32 results of size 4 by 24 summands off by 2^-22 each, over 2 step; curvature: step^2 times third derivatives (below 2 per unit of go)
            assert ((d - dx[:, c]).abs() <= 24 * 4 * 4 * 2.0 ** -22 / (2 * step) + 2 * step ** 2 * go.abs().sum(1)).all()


@pytest.mark.parametrize("keep", [False, True])
def test_the_python_form_and_other_ways_through_the_graph(gpu, keep, monkeypatch):
    """Without the native host path, under a dispatch mode, and with hooks on saved tensors: the same results."""
    import hpfp8
    from hpfp8 import ops
    from torch.utils._python_dispatch import TorchDispatchMode

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x, w, b, go = (t.to(gpu) for t in make(33, 300, torch.bfloat16, torch.float32, 11))

    def step(around_forward=None, around_backward=None):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        if around_forward is None:
            y = hpfp8.layer_norm(leaves[0], 300, leaves[1], leaves[2], keep_8bit=keep)
        else:
            with around_forward:
                y = hpfp8.layer_norm(leaves[0], 300, leaves[1], leaves[2], keep_8bit=keep)
        if around_backward is None:
            grads = torch.autograd.grad(y, leaves, go)
        else:
            with around_backward:
                grads = torch.autograd.grad(y, leaves, go)
        return (y.detach(),) + grads
    want = step()
    hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(gpu))
    strided = torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.stack((t, t), -1)[..., 0])
    for got in (step(Mode()), step(None, Mode()), step(hooks), step(strided) if not keep else want):
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    with torch.no_grad():
        monkeypatch.setattr(ops, "_native", None)
        assert torch.equal(hpfp8.layer_norm(x, 300, w, b), want[0])
    assert all(torch.equal(p, q) for p, q in zip(step(), want))


@pytest.mark.parametrize("native", [True, False])
def test_second_derivatives_are_refused_and_writes_in_between_noticed(gpu, native, monkeypatch):
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    x = torch.randn((4, 64), device=gpu, requires_grad=True)
    go = torch.ones((4, 64), device=gpu, requires_grad=True)
    for f in (lambda t: hpfp8.layer_norm(t, 64), lambda t: hpfp8.activation(t, "silu")):
        g, = torch.autograd.grad(f(x), x, go, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            g.sum().backward()
    t = x * 1.0
    y = hpfp8.layer_norm(t, 64)
    t.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("keep", [False, True])
def test_more_than_2_31_values(gpu, keep):
    """The last rows of a tensor that large have the bits that they have alone."""
    import hpfp8
    cols = 4100
    rows = (1 << 31) // cols + 100
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device=gpu).normal_().requires_grad_()
    w = torch.empty((cols,), dtype=torch.bfloat16, device=gpu).normal_()
    y = hpfp8.layer_norm(x, cols, w, keep_8bit=keep)
    go = torch.empty_like(y).normal_()
    dx, = torch.autograd.grad(y, x, go)
    last = x.detach()[-150:].clone().requires_grad_()
    y_last = hpfp8.layer_norm(last, cols, w, keep_8bit=keep)
    assert torch.equal(y[-150:], y_last) and torch.equal(dx[-150:], torch.autograd.grad(y_last, last, go[-150:])[0])
