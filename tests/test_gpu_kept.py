"""Activations kept in 8 bits: codes against a CPU restatement bit for bit, values and gradients against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}        # half a step, relative
LEAST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -126}     # below it: absolute
U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def randn(shape, seed, dtype, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def quantized(x):
    """(codes, scale_inv) of x[R, C] on the CPU: IEEE fp32 operations and torch's own cast."""
    r, c = x.shape
    g = (c + 127) // 128
    full = torch.zeros((r, g * 128))
    full[:, :c] = x.float()
    full = full.view(r, g, 128)
    amax = full.abs().amax(-1, keepdim=True)
    amax = torch.where(amax < 1e-12, torch.full_like(amax, 1e-12), amax)
    most = torch.full_like(amax, 448.0)         # (torch divides a number by a tensor as number * reciprocal: tensors, for one IEEE division)
    codes = (full * (most / amax)).to(torch.float8_e4m3fn)
    return codes.view(r, g * 128)[:, :c], (amax / most).squeeze(-1)


def values(codes, scale_inv):
    """What codes[R, C] with scales [R, G] stand for, in 64 bits from fp32 products."""
    c = codes.shape[-1]
    return (codes.float() * scale_inv.float().repeat_interleave(128, -1)[..., :c]).double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (1, 128), (5, 129), (17, 1000), (64, 896), (2, 3, 333), (70, 2049)])
def test_codes_scales_and_values_are_the_cpu_restatements(gpu, dtype, shape):
    import hpfp8
    x = randn(shape, 1, dtype, 3.0)
    kept = hpfp8.quantize_activation(x.to(gpu))
    codes, scale_inv = quantized(x.reshape(-1, shape[-1]))
    assert kept.codes.shape == x.shape and kept.scale_inv.shape == x.shape[:-1] + ((shape[-1] + 127) // 128,)
    assert torch.equal(kept.codes.cpu().view(torch.uint8).reshape(codes.shape), codes.view(torch.uint8))
    assert torch.equal(kept.scale_inv.cpu().reshape(scale_inv.shape), scale_inv)
    for to in DTYPES:
        want = (codes.float() * scale_inv.repeat_interleave(128, -1)[:, :shape[-1]]).to(to).reshape(shape)
        assert torch.equal(kept.dequantize(to).cpu(), want)
    assert kept.dequantize().dtype == dtype


def test_whole_groups_have_the_bits_of_the_activation_quantizer(gpu):
    import hpfp8
    x = randn((130, 1152), 2, torch.bfloat16).to(gpu)
    kept, (q, s) = hpfp8.quantize_activation(x), hpfp8.quantize_1x128(x)
    assert torch.equal(kept.codes.view(torch.uint8), q.view(torch.uint8)) and torch.equal(kept.scale_inv, s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_starts_between_vectors(gpu, dtype):
    import hpfp8
    base = randn((40, 700), 3, dtype).to(gpu)
    for x in (base[:, 3:600], base[1::2, 5:], base.t()[2:, :33], base[:1].expand(9, 700), base.reshape(-1)[1:1 + 39 * 700].view(39, 700)):
        got = hpfp8.quantize_activation(x)
        want = hpfp8.quantize_activation(x.clone(memory_format=torch.contiguous_format))
        assert torch.equal(got.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(got.scale_inv, want.scale_inv)


def test_non_finite_and_tiny_groups(gpu):
    import hpfp8
    x = randn((6, 300), 4, torch.float32)
    x[0, 5], x[1, 130], x[2, 299] = math.nan, math.inf, -math.inf
    x[3] = 0.0
    x[4] = 1e-30
    x[5] = 3e38
    kept = hpfp8.quantize_activation(x.to(gpu))
    v = kept.dequantize().cpu()
    assert v[0, :128].isnan().all() and v[0, 128:].isfinite().all()
    assert v[1, 128:256].isnan().all() and v[2, 256:].isnan().all() and v[1, :128].isfinite().all()
    assert (v[3] == 0).all() and (v[4] == 0).all()
    assert ((v[5] - x[5]).abs() <= 2.0 ** -4 * x[5]).all()
    codes, scale_inv = quantized(x)
    assert torch.equal(kept.codes.cpu().view(torch.uint8)[3:], codes.view(torch.uint8)[3:]) and torch.equal(kept.scale_inv.cpu()[3:], scale_inv[3:])


def normal_cdf(x):
    """(through erfc: torch.special.ndtr is 1 + erf on the left too, 2e-2 off at -8 in 64 bits)"""
    return 0.5 * torch.special.erfc(-x * math.sqrt(0.5))


def f64(kind, x):
    if kind == "swiglu":
        gate, up = x.chunk(2, -1)
        return gate * torch.sigmoid(gate) * up
    if kind == "silu":
        return x * torch.sigmoid(x)
    if kind == "gelu":
        return x * normal_cdf(x)
    return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))      # (1 + tanh(u) = 2 sigmoid(2 u), without the cancellation)


def relative_error(kind, x):
    """What fp32 makes of one value or derivative, in units of 2^-24, relative: a handful of operations of one to two units each, and an
    exponential whose argument is rounded: that many units times the argument."""
    x = x[..., :x.shape[-1] // 2] if kind == "swiglu" else x
    argument = {"silu": x.abs(), "swiglu": x.abs(), "gelu": x * x / 2, "gelu_tanh": 1.6 * x.abs() + 0.0714 * x.abs() ** 3}[kind]
    return 24 + 4 * argument.clamp(max=200.0)       # (beyond 200 the exponential is 0 or the function linear)


def gradient(kind, x, go):
    x = x.detach().requires_grad_()
    return torch.autograd.grad(f64(kind, x), x, go)[0]


def within(got, want, limit):
    off = (got.double() - want).abs()
    k = int((off - limit).argmax())
    assert (off <= limit).all(), (k, float(got.reshape(-1)[k]), float(want.reshape(-1)[k]), float(limit.reshape(-1)[k]))


def check_activation(kind, x, go, y, dx, at):
    """at: where the derivative is taken (64 bits)."""
    h, least = HALF[x.dtype], LEAST[x.dtype]
    x64, go64 = x.double(), go.double()
    want = f64(kind, x64)
    err = relative_error(kind, x64)
    within(y, want, h * want.abs() + U * err * want.abs() + least * (1 + x64[..., -want.shape[-1]:].abs()))
    want = gradient(kind, at, go64)
    err = relative_error(kind, at)
    if kind == "swiglu":
        gate, up = at.chunk(2, -1)
        # silu' is a sum of two terms, each with the relative error above
        size = torch.cat(((go64 * up).abs() * (1 + gate.abs()) * torch.sigmoid(gate), (go64 * gate).abs() * torch.sigmoid(gate)), -1)
        err = torch.cat((err, err), -1)
    else:
        scale = torch.sigmoid(at) if kind == "silu" else (normal_cdf(at) + torch.exp(-at * at / 2) if kind == "gelu"
                                                         else torch.sigmoid(1.6 * at + 0.0714 * at ** 3) * (1 + at * at))
        size = go64.abs() * scale * (1 + at.abs())
    within(dx, want, h * want.abs() + U * err * size + least * (1 + go64.abs().max() * (1 + at.abs().max())))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("rows,cols,keep", [(1, 8, True), (3, 130, True), (37, 1000, True), (65, 514, False), (200, 2048, True)])
def test_activation_and_its_gradient(gpu, dtype, kind, rows, cols, keep):
    import hpfp8
    x = randn((rows, cols), 5, dtype, 2.0)
    x[0, 0], x[-1, -1] = 11.0, -30.0
    out = cols // 2 if kind == "swiglu" else cols
    go = randn((rows, out), 6, dtype)
    xg = x.to(gpu).requires_grad_()
    y = hpfp8.activation(xg, kind, keep_8bit=keep)
    assert y.dtype == dtype and y.shape == (rows, out)
    dx, = torch.autograd.grad(y, xg, go.to(gpu))
    at = x.double()
    if keep:
        parts = x.chunk(2, 1) if kind == "swiglu" else (x,)
        at = torch.cat([values(*quantized(t)) for t in parts], 1)
    check_activation(kind, x, go, y.detach().cpu(), dx.cpu(), at)
    with torch.no_grad():
        assert torch.equal(hpfp8.activation(xg, kind), y)


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh", "swiglu"])
def test_derivative_against_differences(gpu, kind):
    import hpfp8
    x = torch.linspace(-6, 6, 512).to(gpu).requires_grad_()
    up = torch.full((512,), 1.5, device=gpu)
    step = 1e-2

    def at(t):
        return hpfp8.activation(torch.cat((t, up)) if kind == "swiglu" else t, kind, keep_8bit=False)
    dx, = torch.autograd.grad(at(x).sum(), x)
    with torch.no_grad():
        # third derivatives are below 4: the central difference is off by 4 / 6 step^2; fp32 results (below 9) by 2^-24 * 32 each
        difference = (at(x + step) - at(x - step)) / (2 * step)
    assert ((dx - difference).abs() <= 4 / 6 * step ** 2 + 2 * 9 * 32 * U / (2 * step)).all()


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh", "swiglu"])
def test_activation_of_extremes(gpu, kind):
    import hpfp8
    g = torch.tensor([math.inf, -math.inf, 1e30, -1e30, 0.0, -0.0, math.nan, -200.0], device=gpu)
    x = torch.cat((g, torch.ones(8, device=gpu))) if kind == "swiglu" else g
    x.requires_grad_()
    y = hpfp8.activation(x, kind, keep_8bit=False)
    dx, = torch.autograd.grad(y, x, torch.ones(8, device=gpu))
    y = y.detach().cpu()
    assert y[0] == math.inf and y[1] == 0 and y[2] == 1e30 and y[3] == 0 and y[4] == 0 and y[5] == 0 and y[6].isnan() and y[7] == 0
    assert dx.cpu()[:4].tolist() == [1, 0, 1, 0] and dx[6].isnan() and dx[7] == 0
    assert abs(float(dx[4]) - 0.5) <= 24 * U * 0.5        # (gelu: the polynomial of Phi is fitted to 4.5e-7 = 7.5 units, at 0 too)


def test_empty_inputs_strided_inputs_and_gradients(gpu):
    import hpfp8
    for shape in ((0, 256), (4, 0)):
        x = torch.empty(shape, device=gpu, dtype=torch.bfloat16, requires_grad=True)
        y = hpfp8.activation(x, "silu")
        assert torch.autograd.grad(y, x, torch.empty_like(y))[0].shape == shape
        assert hpfp8.quantize_activation(x.detach()).dequantize().shape == shape
    base = randn((2, 30, 520), 7, torch.bfloat16).to(gpu)
    x = base[:, ::2, 4:516]
    a, b = x.detach().requires_grad_(), x.detach().clone().requires_grad_()
    for t in (a, b):
        hpfp8.activation(t, "swiglu").sum().backward()       # (an expanded gradient)
    assert torch.equal(a.grad, b.grad)


def test_saved_tensors_are_kept_in_8_bits(gpu):
    import hpfp8
    x = randn((300, 512), 8, torch.bfloat16).to(gpu).requires_grad_()
    w = randn((256, 512), 9, torch.bfloat16, 0.05).to(gpu).requires_grad_()
    seen = []

    def select(t):
        seen.append(t.shape)
        return True
    with hpfp8.keep_activations_8bit(min_elements=1000, select=select):
        h = torch.nn.functional.linear(x * 1.0, w)
        y = torch.nn.functional.silu(h)
    go = randn((300, 256), 10, torch.bfloat16).to(gpu)
    dx, dw = torch.autograd.grad(y, (x, w), go)
    assert seen and all(s != w.shape for s in seen)         # (neither the weight nor its transposed view)
    # the same graph by hand, on what the codes stand for
    kept_x, kept_h = hpfp8.quantize_activation(x.detach()).dequantize(), hpfp8.quantize_activation(h.detach()).dequantize()
    s = torch.sigmoid(kept_h.double())
    dh = go.double() * s * (1 + kept_h.double() * (1 - s))
    # torch rounds dh to bf16, then each result: 2^-8 of the summands' sizes twice, and one rounding of what comes out
    for got, want, size in ((dw, dh.t() @ kept_x.double(), dh.abs().t() @ kept_x.double().abs()),
                            (dx, dh @ w.detach().double(), dh.abs() @ w.detach().double().abs())):
        assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * size).all()
    # small tensors, other types and leaves stay as they are
    with hpfp8.keep_activations_8bit():
        z = (w.detach().requires_grad_() ** 2).sum()
    assert z.grad_fn is not None
    f = randn((300, 512), 11, torch.float32).to(gpu).requires_grad_()
    with hpfp8.keep_activations_8bit(min_elements=1):
        loss = ((f * 1.0) ** 3).sum()
    g, = torch.autograd.grad(loss, f)
    assert torch.allclose(g, 3 * f.detach() ** 2, rtol=1e-6)


def test_an_fp8_linear_inside_the_context_has_its_own_results(gpu):
    """Its saved codes and scales are neither 16-bit nor activations: nothing changes."""
    import hpfp8
    x, w = randn((256, 512), 12, torch.bfloat16).to(gpu), randn((384, 512), 13, torch.bfloat16, 0.05).to(gpu)
    grads = []
    for inside in (False, True):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        if inside:
            with hpfp8.keep_activations_8bit(min_elements=1):
                y = hpfp8.fp8_linear(a, b)
        else:
            y = hpfp8.fp8_linear(a, b)
        y.backward(torch.ones_like(y))
        grads.append((a.grad, b.grad))
    assert all(torch.equal(p, q) for p, q in zip(*grads))


def test_second_derivatives_are_refused(gpu):
    import hpfp8
    x = randn((4, 64), 14, torch.float32).to(gpu).requires_grad_()
    g, = torch.autograd.grad(hpfp8.activation(x, "silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("keep", [False, True])
def test_the_python_form_and_hooks_on_what_is_saved(gpu, keep, monkeypatch):
    import hpfp8
    from hpfp8 import ops
    x, go = randn((21, 390), 15, torch.float16).to(gpu), randn((21, 195), 16, torch.float16).to(gpu)

    def step():
        a = x.clone().requires_grad_()
        y = hpfp8.activation(a, "swiglu", keep_8bit=keep)
        return y.detach(), torch.autograd.grad(y, a, go)[0]
    want = step()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(gpu)):
        got = step()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    kept = hpfp8.quantize_activation(x)
    monkeypatch.setattr(ops, "_native", None)
    assert all(torch.equal(p, q) for p, q in zip(step(), want))
    again = hpfp8.quantize_activation(x)
    assert torch.equal(again.codes.view(torch.uint8), kept.codes.view(torch.uint8)) and torch.equal(again.dequantize(), kept.dequantize())


def test_codes_of_a_part_and_wrong_ones(gpu):
    """Slices of what was made are read with their strides; scales that do not belong to the codes are refused."""
    import hpfp8
    from hpfp8.kept import Fp8Activation
    made = hpfp8.quantize_activation(torch.randn(12, 5, 200, device=gpu).to(torch.bfloat16))
    whole = made.dequantize()
    for part in ((slice(None, None, 2),), (slice(None), 3), (slice(3, 7), slice(1, 4))):
        assert torch.equal(Fp8Activation(made.codes[part], made.scale_inv[part], made.dtype).dequantize(), whole[part])
    for codes, scale_inv in ((made.codes, made.scale_inv[:6]), (made.codes[..., :100], made.scale_inv), (made.codes[0, 0, 0], made.scale_inv)):
        with pytest.raises(ValueError):
            Fp8Activation(codes, scale_inv, torch.bfloat16).dequantize()
    for codes, scale_inv in ((whole, made.scale_inv), (made.codes, made.scale_inv.half())):
        with pytest.raises(TypeError):
            Fp8Activation(codes, scale_inv, torch.bfloat16).dequantize()


@pytest.mark.parametrize("kind,cols", [("silu", 8200), ("swiglu", 4100)])
def test_more_than_2_31_values(gpu, kind, cols):
    """The last rows of a tensor that large have the bits that they have alone."""
    import hpfp8
    width = 2 * cols if kind == "swiglu" else cols
    rows = (1 << 31) // width + 100
    x = torch.empty((rows, width), dtype=torch.bfloat16, device=gpu).normal_().requires_grad_()
    y = hpfp8.activation(x, kind)
    go = torch.empty_like(y).normal_()
    dx, = torch.autograd.grad(y, x, go)
    last = x.detach()[-150:].clone().requires_grad_()
    y_last = hpfp8.activation(last, kind)
    assert torch.equal(y[-150:], y_last) and torch.equal(dx[-150:], torch.autograd.grad(y_last, last, go[-150:])[0])
    made, made_last = hpfp8.quantize_activation(x.detach()), hpfp8.quantize_activation(last.detach())
    assert torch.equal(made.codes[-150:].view(torch.uint8), made_last.codes.view(torch.uint8)) and torch.equal(made.scale_inv[-150:], made_last.scale_inv)
    assert torch.equal(made.dequantize()[-150:], made_last.dequantize())


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 7, 128, 300])
def test_what_a_backward_saved_comes_back_with_its_infinities(gpu, dtype, cols, native, monkeypatch):
    """Infinities and NaN as they were; every other value as if 0 stood in their places."""
    from hpfp8 import kept, ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    x = randn((50, cols), 17, dtype, 2.0)
    x[1], x[2], x[3] = math.inf, -math.inf, math.nan
    pick = torch.rand((50, cols), generator=torch.Generator().manual_seed(18))
    x[4:] = torch.where(pick[4:] < 0.1, -math.inf, torch.where(pick[4:] < 0.15, math.inf, torch.where(pick[4:] < 0.2, math.nan, x[4:].float()))).to(dtype)
    x[40:44] = torch.where(pick[40:44] < 0.5, -math.inf, 0.0).to(dtype)
    x[44:46] = torch.where(pick[44:46] < 0.5, torch.finfo(dtype).min, 0.0).to(dtype)             # (a mask of the type's lowest value)
    x[46] = torch.where(pick[46] < 0.5, -1e-30, 3.0).to(dtype)                                   # (values that round to -0)
    finite = torch.where(x.isfinite(), x, 0.0)
    codes, scale_inv = quantized(finite)
    want = (codes.float() * scale_inv.repeat_interleave(128, -1)[:, :cols]).to(dtype)
    want = torch.where(x.isfinite(), want, x)
    made = kept._quantize(x.to(gpu), True)
    assert torch.equal(made[1].cpu(), scale_inv)
    got = kept._dequantize(*made, dtype, True).cpu()
    assert torch.equal(got.isnan(), x.isnan()) and torch.equal(got.nan_to_num(0.0, math.inf, -math.inf), want.nan_to_num(0.0, math.inf, -math.inf))


def test_saved_tensors_with_infinities_have_finite_gradients(gpu):
    """log_softmax of masked scores saves its result, -inf where the mask is; the gradient is that of the result as it is kept."""
    import hpfp8
    from hpfp8 import kept
    x = randn((300, 500), 19, torch.bfloat16, 2.0)
    mask = torch.rand((300, 500), generator=torch.Generator().manual_seed(20)) < 0.3
    x = x.masked_fill(mask, -math.inf).to(gpu).requires_grad_()
    go = randn((300, 500), 21, torch.bfloat16).masked_fill(mask, 0.0).to(gpu)
    with hpfp8.keep_activations_8bit(min_elements=1000):
        y = torch.log_softmax(x, -1)
    dx, = torch.autograd.grad(y, x, go)
    at = kept._dequantize(*kept._quantize(y.detach(), True), torch.bfloat16, True).double()
    p = torch.exp(at)
    want = go.double() - p * go.double().sum(1, keepdim=True)
    assert dx.isfinite().all() and (dx[mask.to(gpu)] == 0).all()
    # bf16's rounding of the result; fp32 sums of 500 summands, an exponential of an argument below 128
    size = go.double().abs() + p * go.double().abs().sum(1, keepdim=True)
    assert ((dx.double() - want).abs() <= 2.0 ** -8 * want.abs() + U * (500 + 256) * size).all()


def inside(f, leaves, go, **context):
    """(result, gradients) of f(*leaves), inside keep_activations_8bit(**context) if there is one."""
    import contextlib
    import hpfp8
    leaves = [v.clone().requires_grad_() for v in leaves]
    with hpfp8.keep_activations_8bit(**context) if context else contextlib.nullcontext():
        y = f(*leaves)
    return (y.detach(),) + torch.autograd.grad(y, leaves, go)


ALL = dict(min_elements=1, dtypes=(torch.bfloat16, torch.float16, torch.float32))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("context", [dict(min_elements=1), ALL])
def test_statistics_and_what_belongs_to_them_stay_exact(gpu, context, native, monkeypatch):
    """A loss whose targets have almost all of the probability, a norm of rows far from zero: as outside the context, bit for bit."""
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    w = randn((1000, 256), 22, torch.bfloat16, 0.1)
    t = torch.randint(1000, (200,), generator=torch.Generator().manual_seed(23))
    x = (w[t].float() * 8 + randn((200, 256), 24, torch.float32, 0.1)).to(torch.bfloat16)            # (losses around 1e-3)

    def loss(x, w):
        return hpfp8.linear_cross_entropy(x * 1, w, t.to(gpu))          # (no leaf: an activation)
    leaves, go = (x.to(gpu), w.to(gpu)), torch.ones((), device=gpu)
    want, got = inside(loss, leaves, go), inside(loss, leaves, go, **context)
    assert want[0] < 0.1 and all(torch.equal(p, q) for p, q in zip(got, want))
    for dtype in DTYPES:
        x, v = (randn((64, 384), 25, torch.float32) + 100).to(dtype).to(gpu), randn((384,), 26, dtype).to(gpu)
        go = randn((64, 384), 27, dtype).to(gpu)
        for keep in (False, True):
            def norm(x, w, b):
                return hpfp8.layer_norm(x * 1, 384, w, b, keep_8bit=keep)
            want, got = inside(norm, (x, v, v), go), inside(norm, (x, v, v), go, **context)
            assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("native", [True, False])
def test_scales_of_codes_stay_exact(gpu, native, monkeypatch):
    """Linears, experts and activations keep codes: with fp32 tensors in 8 bits too their results are those outside the context."""
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    x, w, go = randn((200, 256), 28, torch.bfloat16).to(gpu), randn((384, 256), 29, torch.bfloat16, 0.1).to(gpu), randn((200, 384), 30, torch.bfloat16).to(gpu)
    experts, offs = randn((3, 384, 256), 31, torch.bfloat16, 0.1).to(gpu), torch.tensor([50, 128, 200], dtype=torch.int32, device=gpu)
    cases = [(lambda x, w: hpfp8.fp8_linear(x * 1, w), (x, w), go), (lambda x, w: hpfp8.fp8_linear(x * 1, w, recipe="per_tensor"), (x, w), go),
             (lambda x, w: hpfp8.fp8_grouped_linear(x * 1, w, offs), (x, experts), go),
             (lambda x: hpfp8.activation(x * 1, "gelu"), (x,), x)]
    for f, leaves, g in cases:
        want, got = inside(f, leaves, g), inside(f, leaves, g, **ALL)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    # the MLP's gate/up output is no statistic's: it is kept in 8 bits, as keep_8bit does
    wgu, wd = randn((512, 256), 33, torch.bfloat16, 0.1).to(gpu), randn((256, 256), 34, torch.bfloat16, 0.1).to(gpu)
    want = inside(lambda *t: hpfp8.fp8_swiglu_mlp(*t, keep_8bit=True), (x, wgu, wd), x)
    got = inside(lambda *t: hpfp8.fp8_swiglu_mlp(*t), (x, wgu, wd), x, **ALL)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert not torch.equal(want[1], inside(lambda *t: hpfp8.fp8_swiglu_mlp(*t), (x, wgu, wd), x)[1])


def test_frozen_parameters_are_parameters(gpu):
    """Neither they nor views of them are kept in 8 bits: the gradient of the input is that outside the context."""
    import hpfp8
    lin = torch.nn.Linear(512, 768, bias=False, device=gpu, dtype=torch.bfloat16).requires_grad_(False)
    x, go = randn((300, 512), 35, torch.bfloat16).to(gpu), randn((300, 768), 36, torch.bfloat16).to(gpu)
    scale = torch.nn.Parameter(randn((300, 1536), 37, torch.bfloat16).to(gpu), requires_grad=False)
    seen = []

    def f(x):
        return lin(x) * scale[:, ::2]
    want = inside(f, (x,), go)
    got = inside(f, (x,), go, min_elements=1000, select=lambda t: seen.append(t) or True)
    assert not seen and all(torch.equal(p, q) for p, q in zip(got, want))


def test_tensors_that_would_take_more_in_8_bits_stay_as_they_are(gpu):
    """Expanded ones, rows of a few values, sparse ones; of all others the context holds the codes and scales instead."""
    import hpfp8
    seen = []
    context = dict(ALL, select=lambda t: seen.append(tuple(t.shape)) or True)
    v, x = randn((512,), 38, torch.bfloat16).to(gpu), randn((300, 512), 39, torch.bfloat16).to(gpu)
    cases = [(lambda x: x * v.expand(300, 512), x)]
    for cols, dtype in ((1, torch.bfloat16), (4, torch.bfloat16), (4, torch.float16), (1, torch.float32)):
        u = randn((700, cols), 40, dtype).to(gpu)
        cases.append((lambda x, u=u: x * (u * 1), u))
    sparse = torch.eye(300, device=gpu).to_sparse()
    cases.append((lambda x: torch.sparse.mm(sparse, x), x.float()))
    for f, leaf in cases:
        want, got = inside(f, (leaf,), torch.ones_like(leaf)), inside(f, (leaf,), torch.ones_like(leaf), **context)
        assert not seen and all(torch.equal(p, q) for p, q in zip(got, want))
    for cols, dtype in ((5, torch.bfloat16), (5, torch.float16), (2, torch.float32)):
        u = randn((700, cols), 41, dtype).to(gpu)
        inside(lambda x: x * (u * 1), (u,), u, **context)
        assert seen.pop() == (700, cols) and not seen


def test_what_the_context_holds(gpu):
    """A chain of nodes that each save one tensor: its codes and scales, to the byte."""
    import hpfp8
    x = randn((1024, 2048), 42, torch.bfloat16).to(gpu).requires_grad_()

    def held(context):
        with context:
            before = torch.cuda.memory_stats()["requested_bytes.all.current"]
            y = torch.nn.functional.silu(torch.nn.functional.silu(x * 2) * 2)       # (saves the products, not the results)
            return torch.cuda.memory_stats()["requested_bytes.all.current"] - before, y
    n = 1024 * 2048
    held(torch.enable_grad()), held(hpfp8.keep_activations_8bit())
    assert held(torch.enable_grad())[0] - held(hpfp8.keep_activations_8bit())[0] == 2 * (2 * n - n - n // 128 * 4)
