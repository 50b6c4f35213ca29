"""Root-mean-square norm against 64 bits, element by element, with bounds that count the roundings; its outputs in 8 bits."""
import math
import types

import pytest
import torch

from test_gpu_operators_in_torch import WAYS, randn, step

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
U = 2.0 ** -24
EPS = 1e-6


def make(rows, cols, dtype, wdtype, seed):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp(torch.randn((cols,), generator=g) * 0.7)
    x = (torch.randn((rows, cols), generator=g) * size + 0.3).to(dtype)
    r = (torch.randn((rows, cols), generator=g) * size).to(dtype)
    w = (1 + 0.2 * torch.randn((cols,), generator=g)).to(wdtype)
    go = torch.randn((rows, cols), generator=g).to(dtype)
    gs = torch.randn((rows, cols), generator=g).to(dtype)
    return x, r, w, go, gs


def reference(s, w, go, gs, eps=EPS):
    """(y, ds, dw, hat, rstd) in 64 bits of the values s that are normalised."""
    s, go = s.double(), go.double()
    w = torch.ones(s.shape[1], dtype=torch.float64) if w is None else w.double()
    rstd = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    hat = s * rstd
    u = go * w
    ds = rstd * (u - hat * (u * hat).mean(1, keepdim=True)) + (0 if gs is None else gs.double())
    return hat * w, ds, (go * hat).sum(0), hat, rstd


def bounds(s, w, go, gs, ref):
    """What fp32 may be off by.  A row's sum adds at most 32 values in a thread, then six steps of a tree and eight waves, each a rounding, and
    has one more for each product: 47 of its size, and rstd, a root of it, half of that and its own three: 28.  y takes two products more.  A
    column's sum adds its rows one after the other in at least 256 places, or in fewer places fewer rows, then at most 32 teams and 48 partial
    sums."""
    y, ds, dw, hat, rstd = ref
    w = torch.ones(s.shape[1], dtype=torch.float64) if w is None else w.double()
    go = go.double()
    u = (go * w).abs()
    by = 48 * U * y.abs()
    bs = 128 * U * rstd * (u + hat.abs() * (u * hat.abs()).mean(1, keepdim=True)) + (0 if gs is None else 2 * U * gs.double().abs())
    bw = (s.shape[0] / 256 + 128 + 32) * U * (go * hat).abs().sum(0)
    return by, bs, bw


def close(got, want, bound, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    off = (got.double().cpu() - want).abs()
    limit = HALF[dtype] * (want.abs() + bound) + bound + 2.0 ** -24 * (dtype == torch.float16)
    assert (off <= limit).all(), float((off - limit).max())


CASES = [  # rows, cols
    (1, 1), (1, 8), (5, 3), (3, 64), (9, 127), (33, 512), (20, 513), (17, 1024), (16, 1025), (300, 1027), (7, 4096), (13, 4100), (31, 7168),
    (5, 8192), (3, 8200), (9, 16384), (2, 16381), (1100, 40), (2500, 136), (40, 9), (70, 128), (33, 129), (21, 200), (65, 256), (12, 257), (11, 2047),
    (6, 2048), (5, 2055), (6, 8191), (3, 8193), (700, 2048), (1300, 384)]
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32), (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("rows,cols", CASES)
@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
def test_forward_and_backward(gpu, rows, cols, dtype, wdtype, residual):
    import hpfp8
    x, r, w, go, gs = make(rows, cols, dtype, wdtype, 1)
    xg, rg, wg = (t.to(gpu).requires_grad_() for t in (x, r, w))
    if not residual:
        y = hpfp8.rms_norm(xg, cols, wg, EPS)
        ds, dw = torch.autograd.grad(y, (xg, wg), go.to(gpu))
        s, gs = x, None
    else:
        y, total = hpfp8.rms_norm(xg, (cols,), wg, EPS, residual=rg)
        ds, dr, dw = torch.autograd.grad((y, total), (xg, rg, wg), (go.to(gpu), gs.to(gpu)))
        assert torch.equal(ds, dr)
        s = x + r                                            # (one rounding of the exact sum: the same bits)
        assert torch.equal(total.detach().cpu(), s)
    ref = reference(s, w, go, gs)
    by, bs, bw = bounds(s, w, go, gs, ref)
    close(y.detach(), ref[0], by, dtype)
    close(ds, ref[1], bs, dtype)
    close(dw, ref[2], bw, wdtype)
    with torch.no_grad():                                    # inference: the same bits
        out = hpfp8.rms_norm(xg, cols, wg, EPS, residual=rg if residual else None)
    assert torch.equal(out[0] if residual else out, y)
    if residual:
        assert torch.equal(out[1], total)


@pytest.mark.parametrize("residual", [False, True])
def test_without_a_weight_and_the_default_eps(gpu, residual):
    import hpfp8
    x, r, _, go, gs = make(12, 256, torch.bfloat16, torch.bfloat16, 2)
    x = x * 1e-4
    r = r * 1e-4
    xg, rg = x.to(gpu).requires_grad_(), r.to(gpu).requires_grad_()
    s = x + r if residual else x
    out = hpfp8.rms_norm(xg, 256, residual=rg if residual else None)
    eps = torch.finfo(torch.float32).eps
    ref = reference(s, None, go, gs if residual else None, eps)
    by, bs, _ = bounds(s, None, go, gs if residual else None, ref)
    close((out[0] if residual else out).detach(), ref[0], by, torch.bfloat16)
    ds, = torch.autograd.grad(out, (xg,), (go.to(gpu), gs.to(gpu)) if residual else go.to(gpu))
    close(ds, ref[1], bs, torch.bfloat16)
    want = torch.nn.functional.rms_norm(s.float(), (256,))
    assert (want.double() - ref[0]).abs().max() < 1e-5       # (torch's own default)


@pytest.mark.parametrize("native", [True, False])
def test_only_one_of_the_results_is_used(gpu, native, monkeypatch):
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    x, r, w, go, gs = (t.to(gpu) for t in make(9, 640, torch.bfloat16, torch.bfloat16, 3))
    x, r, w = (t.requires_grad_() for t in (x, r, w))
    y, s = hpfp8.rms_norm(x, 640, w, residual=r)
    dx, dr, dw = torch.autograd.grad(s, (x, r, w), gs, allow_unused=True)
    assert torch.equal(dx, gs) and torch.equal(dr, gs) and dw is None
    y, s = hpfp8.rms_norm(x, 640, w, residual=r)
    dx, dr, dw = torch.autograd.grad(y, (x, r, w), go)
    want = torch.autograd.grad(hpfp8.rms_norm(s.detach().requires_grad_(), 640, w), w, go)[0]
    assert torch.equal(dx, dr) and torch.equal(dw, want)
    s2 = s.detach().requires_grad_()
    assert torch.equal(dx, torch.autograd.grad(hpfp8.rms_norm(s2, 640, w), s2, go)[0])
    # backward into leaves: each has a gradient of its own
    y, s = hpfp8.rms_norm(x, 640, w, residual=r)
    (y.float().sum() + s.float().sum()).backward()
    assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()


@pytest.mark.parametrize("which", [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
def test_gradients_of_only_some_inputs(gpu, which):
    import hpfp8
    x, r, w, go, gs = (t.to(gpu) for t in make(33, 384, torch.float16, torch.float16, 4))
    full = [t.clone().requires_grad_() for t in (x, r, w)]
    want = torch.autograd.grad(hpfp8.rms_norm(full[0], 384, full[2], residual=full[1]), full, (go, gs))
    some = [t.clone().requires_grad_(q) for t, q in zip((x, r, w), which)]
    out = hpfp8.rms_norm(some[0], 384, some[2], residual=some[1])
    got = torch.autograd.grad(out, [t for t in some if t.requires_grad], (go, gs), allow_unused=True)
    for g, e in zip(got, [e for e, q in zip(want, which) if q]):
        assert torch.equal(g, e)


def test_gradient_against_differences(gpu):
    """fp32, a direction at a time: (f(x + h d) - f(x - h d)) / 2h in 64 bits of the formula against <grad, d>."""
    import hpfp8
    x, r, w, go, gs = make(6, 96, torch.float32, torch.float32, 5)
    xg, rg, wg = (t.to(gpu).requires_grad_() for t in (x, r, w))
    out = hpfp8.rms_norm(xg, 96, wg, EPS, residual=rg)
    grads = torch.autograd.grad(out, (xg, rg, wg), (go.to(gpu), gs.to(gpu)))

    def f(x, r, w):
        s = x + r
        y = s / torch.sqrt((s * s).mean(1, keepdim=True) + EPS) * w
        return (y * go.double()).sum() + (s * gs.double()).sum()
    at = [t.double() for t in (x, r, w)]
    g = torch.Generator().manual_seed(6)
    for i in range(3):
        d = torch.randn(at[i].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * d, at[i] - h * d
        slope = (f(*up) - f(*down)) / (2 * h)
        got = (grads[i].double().cpu() * d).sum()
        size = (grads[i].double().cpu() * d).abs().sum()
        assert abs(float(got - slope)) < 1e-5 * float(size)  # (fp32 gradients: 256 roundings of 2^-24; the differences: h^2)


def test_several_dimensions_strides_and_starts_between_vectors(gpu):
    import hpfp8
    g = torch.Generator().manual_seed(7)
    wide = torch.randn((4, 6, 700), generator=g).to(torch.bfloat16).to(gpu)
    other = torch.randn((700, 4, 6), generator=g).to(torch.bfloat16).to(gpu)
    x, r = wide[:, :, 3:515], other.permute(1, 2, 0)[:, :, 100:612]
    w = torch.randn((515,), generator=g).to(torch.bfloat16).to(gpu)[3:]
    want = hpfp8.rms_norm(x.contiguous(), 512, w.clone(), residual=r.contiguous())
    got = hpfp8.rms_norm(x, 512, w, residual=r)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x2 = wide[0, :, :640].reshape(6, 5, 128)
    w2 = torch.randn((5, 128), generator=g).to(torch.bfloat16).to(gpu)
    assert torch.equal(hpfp8.rms_norm(x2, (5, 128), w2), hpfp8.rms_norm(x2.reshape(6, 640), 640, w2.view(-1)).view(6, 5, 128))
    # gradients that come with other strides, and broadcast inputs
    xl = torch.randn((1, 384), generator=g).to(torch.bfloat16).to(gpu).requires_grad_()
    y, s = hpfp8.rms_norm(xl.expand(5, 384), 384, residual=r.reshape(24, 512)[:5, :384])
    go = torch.randn((384, 5), generator=g).to(torch.bfloat16).to(gpu).t()
    got, = torch.autograd.grad((y, s), xl, (go, go))
    xe = xl.detach().expand(5, 384).contiguous().requires_grad_()
    y, s = hpfp8.rms_norm(xe, 384, residual=r.reshape(24, 512)[:5, :384].contiguous())
    want, = torch.autograd.grad((y, s), xe, (go.contiguous(), go.contiguous()))
    assert torch.equal(got, want.sum(0, keepdim=True))
    y = hpfp8.rms_norm(xe, 384)
    assert torch.equal(torch.autograd.grad(y.sum(), xe)[0], torch.autograd.grad(hpfp8.rms_norm(xe, 384), xe, torch.ones_like(y))[0])    # (an expanded one)


def test_rows_of_zeros_and_rows_that_are_not_finite(gpu):
    import hpfp8
    x = torch.ones((5, 256), dtype=torch.float32, device=gpu)
    x[0] = 0
    x[1, 7] = math.inf
    x[2, 9] = math.nan
    y = hpfp8.rms_norm(x, 256, eps=1e-6)
    want = torch.nn.functional.rms_norm(x, (256,), eps=1e-6)
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and (y[0] == 0).all()
    assert torch.equal(y[3:], torch.nn.functional.rms_norm(x[3:], (256,), eps=1e-6))
    assert torch.isnan(hpfp8.rms_norm(x, 256, eps=0.0)[0]).all()        # (0 / 0, as torch's)
    codes, scale = hpfp8.rms_norm_quantize_int8(x, eps=1e-6)
    assert torch.isnan(scale[1:3]).all() and (codes[:3] == 0).all() and torch.isfinite(scale[[0, 3, 4]]).all()
    codes, scale = hpfp8.rms_norm_quantize_1x128(x, eps=1e-6)
    assert torch.isnan(scale[1, 0]) and torch.isnan(scale[2]).all() and scale[1, 1] == torch.tensor(1e-12) / 448
    assert (codes[0].float() == 0).all()


def test_no_rows(gpu):
    import hpfp8
    x = torch.zeros((0, 256), dtype=torch.bfloat16, device=gpu, requires_grad=True)
    w = torch.ones(256, dtype=torch.bfloat16, device=gpu, requires_grad=True)
    y, s = hpfp8.rms_norm(x, 256, w, residual=x.detach())
    dx, dw = torch.autograd.grad((y, s), (x, w), (torch.zeros_like(y), torch.zeros_like(s)))
    assert dx.shape == (0, 256) and (dw == 0).all() and dw.shape == (256,)
    with torch.no_grad():
        for f, shape in ((hpfp8.rms_norm_quantize_1x128, (0, 2)), (hpfp8.rms_norm_quantize_int8, (0,))):
            codes, scale, total = f(x, w, residual=x)
            assert codes.shape == (0, 256) and scale.shape == shape and total.shape == (0, 256)


@pytest.mark.parametrize("rows,cols", [(1, 128), (7, 256), (33, 384), (19, 1024), (300, 2048), (8, 7168), (517, 7168), (5, 16384), (3, 8320)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
def test_output_in_8_bits(gpu, rows, cols, dtype, residual):
    """What a code stands for is off by half a step (E4M3: 2^-4 of the value, 2^-10 scales below the smallest normal; int8: half a scale) of
    a y that is off by what the norm's own roundings are."""
    import hpfp8
    x, r, w, go, _ = make(rows, cols, dtype, dtype, 8)
    s = x + r if residual else x
    y, _, _, _, _ = reference(s, w, go, None)
    to = lambda t: t.to(gpu)          # noqa: E731
    kw = dict(residual=to(r)) if residual else {}
    for pow2 in (False, True):
        out = hpfp8.rms_norm_quantize_1x128(to(x), to(w), EPS, pow2=pow2, **kw)
        codes, scale = out[0].double().cpu(), out[1].double().cpu()
        assert out[0].dtype == torch.float8_e4m3fn and scale.shape == (rows, cols // 128) and out[1].stride(0) == 1
        groups = y.view(rows, -1, 128)
        want = groups.abs().amax(2).clamp_min(1e-12) / 448
        if pow2:
            assert (torch.log2(scale) == torch.log2(scale).round()).all()
            assert (scale >= want * (1 - 64 * U)).all() and (scale < 2 * want * (1 + 64 * U)).all()
        else:
            assert ((scale - want).abs() <= 64 * U * want).all()
        off = (codes.view(rows, -1, 128) * scale.unsqueeze(2) - groups).abs()
        assert (off <= (2.0 ** -4 + 128 * U) * groups.abs() + 2.0 ** -10 * scale.unsqueeze(2)).all()
        if residual:
            assert torch.equal(out[2].cpu(), s)
    out = hpfp8.rms_norm_quantize_int8(to(x), to(w), EPS, **kw)
    scale = out[1].double().cpu()
    want = y.abs().amax(1).clamp_min(1e-12) / 127
    assert out[0].dtype == torch.int8 and ((scale - want).abs() <= 64 * U * want).all()
    assert ((out[0].double().cpu() * scale.unsqueeze(1) - y).abs() <= scale.unsqueeze(1) * (0.5 + 127 * 128 * U)).all()
    assert (out[0].cpu().int().abs().amax(1) == 127).all()
    if residual:
        assert torch.equal(out[2].cpu(), s)


@pytest.mark.parametrize("rows,cols", [(5, 128), (40, 1024), (130, 7168)])
def test_codes_are_the_quantizers_where_the_norm_is_exact(gpu, rows, cols):
    """Rows of +-1 and eps 0: rstd is 1 and y the weight's values with signs, which quantize_1x128 and quantize_int8 take to the same codes."""
    import hpfp8
    g = torch.Generator().manual_seed(9)
    x = (torch.randint(2, (rows, cols), generator=g) * 2 - 1).to(torch.bfloat16).to(gpu)
    w = torch.randn((cols,), generator=g).to(torch.bfloat16).to(gpu)
    y = x * w
    for pow2 in (False, True):
        codes, scale = hpfp8.rms_norm_quantize_1x128(x, w, 0.0, pow2=pow2)
        want, want_scale = hpfp8.quantize_1x128(y, kmajor=True, pow2=pow2)
        assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scale, want_scale)
    codes, scale = hpfp8.rms_norm_quantize_int8(x, w, 0.0)
    want, want_scale = hpfp8.quantize_int8(y)
    assert torch.equal(codes, want) and torch.equal(scale, want_scale)


def test_three_dimensions_and_strided_inputs_in_8_bits(gpu):
    import hpfp8
    g = torch.Generator().manual_seed(10)
    wide = torch.randn((2, 5, 300), generator=g).to(torch.float16).to(gpu)
    x, r = wide[:, :, 1:257], wide[:, :, 7:263]
    w = torch.randn((256,), generator=g).to(gpu)
    for f in (hpfp8.rms_norm_quantize_1x128, hpfp8.rms_norm_quantize_int8):
        got = f(x, w, residual=r)
        want = f(x.reshape(10, 256).clone(), w, residual=r.reshape(10, 256).clone())
        assert torch.equal(got[0].view(torch.uint8).view(10, 256), want[0].view(torch.uint8)) and torch.equal(got[2].view(10, 256), want[2])
        assert torch.equal(got[1].reshape(want[1].shape), want[1]) and got[1].shape[:2] == (2, 5)
        same = f(x.contiguous(), w, residual=r.contiguous())          # (the native form)
        assert torch.equal(got[0].view(torch.uint8), same[0].view(torch.uint8)) and torch.equal(got[1], same[1]) and got[1].shape == same[1].shape


def test_the_same_bits_every_time_and_module_form(gpu):
    import hpfp8
    x, r, w, go, gs = (t.to(gpu) for t in make(3000, 1152, torch.bfloat16, torch.bfloat16, 11))
    norm = hpfp8.RMSNorm(1152, 1e-6, device=gpu)
    theirs = torch.nn.RMSNorm(1152, 1e-6, device=gpu, dtype=torch.bfloat16)
    theirs.weight.data.copy_(w)
    norm.load_state_dict(theirs.state_dict())
    assert list(norm.state_dict()) == ["weight"] and "1152" in repr(norm)
    runs = []
    for _ in range(3):
        xl, rl = x.clone().requires_grad_(), r.clone().requires_grad_()
        y, s = norm(xl, rl)
        runs.append((y, s, *torch.autograd.grad((y, s), (xl, rl, norm.weight), (go, gs))))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
    assert torch.equal(norm(x), hpfp8.rms_norm(x, 1152, w, 1e-6))
    plain = hpfp8.RMSNorm(1152, elementwise_affine=False)
    assert torch.equal(plain(x), hpfp8.rms_norm(x, 1152))


def operator(name):
    import hpfp8
    x, r, w = randn((48, 256), 1), randn((48, 256), 2), randn((256,), 3)
    if name == "plain":
        return lambda a, b: hpfp8.rms_norm(a, 256, b), (x, w), randn((48, 256), 4)

    def both(a, b, c):
        y, s = hpfp8.rms_norm(a, 256, c, residual=b.expand(a.shape) if b.dim() != a.dim() else b)
        return y * s
    return both, (x, r[0] if name == "one_row" else r, w), randn((48, 256), 4)


@pytest.mark.parametrize("name", ["plain", "residual"])
@pytest.mark.parametrize("way", [w for w in WAYS if w != "vmap"] + ["vmap"])
def test_the_native_host_path_has_the_python_functions_outcome(gpu, name, way, monkeypatch):
    """Values, or the error, are those that the Python autograd function gives by itself; where they are values, the plain step's."""
    from hpfp8 import ops
    assert ops._native is not None
    f, tensors, go = operator(name if way != "vmap" or name == "plain" else "one_row")

    def outcome(way):
        try:
            r = step(f, tuple(t.clone().requires_grad_() for t in tensors), go.detach().clone(), way)
        except Exception as e:
            return type(e), str(e).split("\n")[0].split(" is a view")[-1]
        return [t.detach() for t in r] if isinstance(r, (tuple, list)) else [r.detach()]
    got = outcome(way)
    values = ("mode", "trace", "trace_inference", "create_graph", "checkpoint", "reentrant", "dispatching_grad", "detect_anomaly", "retained", "other_stream",
              "in_place")
    if way in values and not (name == "residual" and way == "dispatching_grad"):
        assert isinstance(got, list), got
        plain = outcome("plain")
        plain[0] = plain[0] + 1 if way == "in_place" else plain[0]
        plain = plain[:1] if way.startswith("trace") else (plain[1:] if len(got) < len(plain) else plain)
        assert len(got) == len(plain) and all(torch.equal(a, b) for a, b in zip(got, plain))
    monkeypatch.setattr(ops, "_native", types.SimpleNamespace(**{
        k: (lambda *a: None) if k == "rms_norm" else getattr(ops._native, k) for k in dir(ops._native) if not k.startswith("__")}))
    want = outcome(way)
    if isinstance(want, tuple):
        assert got == want or (way == "sparse_grad" and got[0] is want[0])
    else:
        assert isinstance(got, list), got
        assert len(got) == len(want) and all(type(a) is type(b) and torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("native", [True, False])
def test_second_derivatives_are_refused_and_writes_in_between_noticed(gpu, native, monkeypatch):
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    x, r, w = (t.requires_grad_() for t in (randn((16, 128), 1), randn((16, 128), 2), randn((128,), 3)))
    y, s = hpfp8.rms_norm(x, 128, w, residual=r)
    go = randn((16, 128), 4).requires_grad_()
    dx, = torch.autograd.grad((y, s), x, (go, go), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        dx.float().sum().backward()
    y, s = hpfp8.rms_norm(x, 128, w, residual=r)
    total = y + 0                                            # (y is not saved: it may be written to)
    y += 1
    torch.autograd.grad(total.float().sum(), x)
    y, s = hpfp8.rms_norm(x, 128, w, residual=r)
    z = (y * 2).float().sum()
    s += 1                                                   # (the sum is)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_a_tangent_is_refused_and_not_dropped(gpu):
    import hpfp8
    import torch.autograd.forward_ad as fwAD
    x, r, w = randn((16, 128), 1), randn((16, 128), 2), randn((128,), 3)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), fwAD.dual_level():
            for i in range(3):
                a, b, c = (fwAD.make_dual(t, torch.ones_like(t)) if k == i else t for k, t in enumerate((x, r, w)))
                with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward mode"):
                    hpfp8.rms_norm(a, 128, c, residual=b)
                with pytest.raises(RuntimeError, match="for inference"):
                    hpfp8.rms_norm_quantize_int8(a, c, residual=b)


def test_inputs_of_kept_activations_stay_as_they_are(gpu):
    import hpfp8
    x, r, w, go, gs = (t.to(gpu) for t in make(64, 512, torch.bfloat16, torch.bfloat16, 12))

    def grads(native):
        xl, rl, wl = (t.clone().requires_grad_() for t in (x, r, w))
        out = hpfp8.rms_norm(xl if native else xl.t().contiguous().t(), 512, wl, residual=rl)
        return torch.autograd.grad(out, (xl, rl, wl), (go, gs))
    want = grads(True)
    for native in (True, False):
        with hpfp8.keep_activations_8bit(min_elements=1):
            got = grads(native)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_with_its_backward_and_replayed(gpu):
    import hpfp8
    x, r, w, go, gs = (t.to(gpu) for t in make(513, 1024, torch.bfloat16, torch.bfloat16, 13))
    xs, rs = x.clone().requires_grad_(), r.clone().requires_grad_()
    ws = w.clone().requires_grad_()

    def run():
        y, s = hpfp8.rms_norm(xs, 1024, ws, residual=rs)
        with torch.no_grad():
            q = hpfp8.rms_norm_quantize_1x128(xs, ws, residual=rs)
            i = hpfp8.rms_norm_quantize_int8(xs, ws, residual=rs)
        return (y.detach(), s.detach(), *torch.autograd.grad((y, s), (xs, rs, ws), (go, gs)), q[0].view(torch.uint8), q[1], i[0], i[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for k in range(4):
        with torch.no_grad():
            xs.copy_(x * (k + 1))
            rs.copy_(r - k)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, run()))


@pytest.mark.parametrize("form", ["own", "train", "e4m3", "int8"])
def test_more_than_2_31_values(gpu, form):
    import hpfp8
    rows, cols = (1 << 31) // 4096 + 64, 4096
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device=gpu)
    part = randn((64, cols), 14)
    x.view(-1, 64, cols)[:] = part
    few = part.clone()
    if form == "own":
        with torch.no_grad():
            y, s = hpfp8.rms_norm(x, cols, residual=x)
            ey, es = hpfp8.rms_norm(few, cols, residual=few)
        for at in (0, rows - 64):
            assert torch.equal(y[at:at + 64], ey) and torch.equal(s[at:at + 64], es)
    elif form == "train":
        x.requires_grad_()
        y = hpfp8.rms_norm(x, cols)
        dx, = torch.autograd.grad(y, x, x.detach())
        few.requires_grad_()
        want, = torch.autograd.grad(hpfp8.rms_norm(few, cols), few, few.detach())
        for at in (0, rows - 64):
            assert torch.equal(dx[at:at + 64], want)
    else:
        f = hpfp8.rms_norm_quantize_1x128 if form == "e4m3" else hpfp8.rms_norm_quantize_int8
        codes, scale = f(x)
        want, want_scale = f(few)
        for at in (0, rows - 64):
            assert torch.equal(codes[at:at + 64].view(torch.uint8), want.view(torch.uint8)) and torch.equal(scale[at:at + 64], want_scale)


def test_hooks_on_saved_tensors(gpu):
    """What a hook hands back is looked at: as it was or packed elsewhere and back it is used, anything else is refused."""
    import hpfp8
    x, r, w, go, gs = (t.to(gpu) for t in make(32, 384, torch.bfloat16, torch.bfloat16, 15))
    leaves = [t.requires_grad_() for t in (x, r, w)]
    f = lambda: hpfp8.rms_norm(leaves[0], 384, leaves[2], residual=leaves[1])          # noqa: E731
    want = torch.autograd.grad(f(), leaves, (go, gs))
    with torch.autograd.graph.save_on_cpu():
        out = f()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, (go, gs)), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t):
        out = f()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, (go, gs)), want))
    for wrong in (lambda t: t.double(), lambda t: t[:-1], lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, wrong):
            out = f()
        with pytest.raises((ValueError, TypeError)):
            torch.autograd.grad(out, leaves, (go, gs))


def test_gradient_penalty_through_what_follows_and_accumulation(gpu):
    """Two uses of the stream: their gradients add up before they reach the norm's node; .backward twice accumulates."""
    import hpfp8
    x, r, w, go, gs = (t.to(gpu) for t in make(40, 256, torch.float32, torch.float32, 16))
    leaves = [t.requires_grad_() for t in (x, r, w)]
    for t in leaves:
        t.grad = None
    for _ in range(2):
        y, s = hpfp8.rms_norm(leaves[0], 256, leaves[2], EPS, residual=leaves[1])
        y2, s2 = hpfp8.rms_norm(y, 256, leaves[2], EPS, residual=s)
        ((y2 * go).sum() + (s2 * gs).sum() + (s * go).sum()).backward()
    a, b, c = (t.detach().double().requires_grad_() for t in leaves)

    def norm(v):
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + EPS) * c
    s = a + b
    s2 = norm(s) + s
    ((norm(s2) * go.double()).sum() + (s2 * gs.double()).sum() + (s * go.double()).sum()).backward()
    for t, u in zip(leaves, (a, b, c)):
        assert (t.grad.double() - 2 * u.grad).norm() <= 1e-5 * u.grad.norm()       # (a few hundred roundings of 2^-24)
