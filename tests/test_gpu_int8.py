"""The linear in 8-bit integers: codes, scales and products bit for bit (sums of integers are exact), the input's gradient against 64 bits."""
import math
import types

import numpy as np
import pytest
import torch

from test_gpu_operators_in_torch import WAYS, step

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def quantized(v):
    """(codes, scale_inv) of the rows of v[R, C] in numpy fp32: each operation rounded once."""
    v = np.asarray(v, dtype=np.float32)
    amax = np.abs(v).max(1, keepdims=True) if v.size else np.zeros((v.shape[0], 1), np.float32)
    amax = np.where(amax < np.float32(1e-12), np.float32(1e-12), amax).astype(np.float32)
    with np.errstate(all="ignore"):
        scale = np.float32(127.0) / amax
        codes = np.rint(v * scale)
        codes = np.where(np.isfinite(amax), codes, 0).astype(np.int8)
    return codes, (amax / np.float32(127.0))[:, 0]


def product(a, sa, b, sb, bias, dtype):
    """The bits of the result: the sum as an integer, rounded to fp32, times one scale, times the other, plus the bias, rounded to the type."""
    c = torch.from_numpy(a.astype(np.int64)).double() @ torch.from_numpy(b.astype(np.int64)).double().t()      # (below 2^53: exact)
    c = c.numpy().astype(np.float32) * np.float32(sa)[:, None]
    if sb is not None:
        c = c * np.float32(sb)[None, :]
    if bias is not None:
        c = c + bias.float().numpy()[None, :]
    return torch.from_numpy(c.astype(np.float32)).to(dtype)


def values(rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g)
    x[:, ::max(1, cols // 7)] *= 20
    return x.to(dtype)


def same(a, b):
    return torch.equal(a.cpu(), b) and a.dtype == b.dtype


@pytest.mark.parametrize("rows,cols", [(1, 128), (5, 256), (33, 384), (20, 1024), (9, 1152), (300, 2048), (7, 7168), (3, 8192), (4, 16384), (2, 16512), (3, 40960),
                                       (1, 130944)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("columns", [False, True])
def test_codes_and_scales_bit_for_bit(gpu, rows, cols, dtype, columns):
    import hpfp8
    x = values(rows, cols, dtype, 1)
    by = torch.rand((cols,), generator=torch.Generator().manual_seed(2)) * 0.01 if columns else None
    v = x.float().numpy() if by is None else x.float().numpy() * by.numpy()[None, :]
    codes, scale = quantized(v)
    got, got_scale = hpfp8.quantize_int8(x.to(gpu), column_scale=None if by is None else by.to(gpu))
    assert same(got, torch.from_numpy(codes)) and same(got_scale, torch.from_numpy(scale))


@pytest.mark.parametrize("cols", [128, 512, 2048, 16512])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_at_the_edges(gpu, cols, dtype):
    """Zeros, values below the smallest scale, subnormals, the type's largest, ties, infinities and NaN."""
    import hpfp8
    top = torch.finfo(dtype).max
    x = torch.zeros((9, cols), dtype=torch.float64)
    x[1, 3] = 1e-14
    x[2, 5], x[2, 9] = -1e-39, 5e-40
    x[3, 0], x[3, 1] = top, -top
    x[4] = torch.arange(cols, dtype=torch.float64) % 255 - 127           # (amax 127: every value a code)
    x[5, 0], x[5, 1:5] = 127, torch.tensor([0.5, 1.5, -2.5, 126.5])      # ties
    x[6, 2] = math.inf
    x[7, 2], x[7, 4] = -math.inf, math.nan
    x[8, cols - 1] = math.nan
    x = x.to(dtype)
    codes, scale = quantized(x.float().numpy())
    got, got_scale = hpfp8.quantize_int8(x.to(gpu))
    assert same(got, torch.from_numpy(codes))
    assert torch.equal(torch.isnan(got_scale.cpu()), torch.tensor([False] * 7 + [True] * 2)) and math.isinf(float(got_scale[6]))
    assert np.array_equal(got_scale.cpu().numpy()[:7], scale[:7])
    w = hpfp8.quantize_weight_int8(torch.ones((128, cols), dtype=dtype, device=gpu))
    y = hpfp8.int8_linear(x.to(gpu), w)
    assert torch.isnan(y[6:].float()).all() and (y[:2].float() == 0)[:1].all() and torch.isfinite(y[4:6].float()).all()


def test_strides_dimensions_and_no_rows_quantized(gpu):
    import hpfp8
    wide = values(24, 700, torch.bfloat16, 3).to(gpu)
    x = wide.view(4, 6, 700)[:, :, 5:517]
    want = hpfp8.quantize_int8(x.reshape(24, 512).clone())
    got = hpfp8.quantize_int8(x)
    assert torch.equal(got[0].view(24, 512), want[0]) and torch.equal(got[1].view(24), want[1]) and got[1].shape == (4, 6)
    t = values(256, 40, torch.float16, 4).to(gpu).t()
    assert torch.equal(hpfp8.quantize_int8(t)[0], hpfp8.quantize_int8(t.contiguous())[0])
    by = torch.rand((1027,), device=gpu)[3:515]                          # (starts between two vectors)
    a, b = hpfp8.quantize_int8(x, column_scale=by), hpfp8.quantize_int8(x.contiguous(), column_scale=by.clone())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    one = hpfp8.quantize_int8(x[0, 0])
    assert one[0].shape == (512,) and one[1].shape == ()
    none = hpfp8.quantize_int8(x[:0])
    assert none[0].shape == (0, 6, 512) and none[1].shape == (0, 6)


SHAPES = [(1, 128, 128), (3, 128, 384), (8, 7168, 512), (16, 256, 2048), (37, 1024, 1024), (64, 640, 4096), (65, 640, 1024), (130, 384, 640), (200, 1280, 2048),
          (300, 256, 128), (515, 2048, 1152), (1000, 1152, 256), (1531, 4096, 384)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [False, True])
def test_product_bit_for_bit(gpu, m, n, k, dtype, bias):
    import hpfp8
    g = torch.Generator().manual_seed(m + n + k)
    a = torch.randint(-128, 128, (m, k), generator=g).to(torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=g).to(torch.int8)
    sa, sb = torch.rand((m,), generator=g) * 0.01, torch.rand((n,), generator=g) * 0.01
    bi = torch.randn((n,), generator=g).to(dtype) if bias else None
    want = product(a.numpy(), sa.numpy(), b.numpy(), sb.numpy(), bi, dtype)
    to = lambda t: None if t is None else t.to(gpu)          # noqa: E731
    assert same(hpfp8.gemm_int8(to(a), to(sa), to(b), to(sb), to(bi), out_dtype=dtype), want)
    want = product(a.numpy(), sa.numpy(), b.numpy(), None, bi, dtype)
    assert same(hpfp8.gemm_int8(to(a), to(sa), to(b), None, to(bi), out_dtype=dtype), want)


@pytest.mark.parametrize("form", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_tile_shape_has_the_same_bits(gpu, form, dtype):
    import hpfp8
    from hpfp8 import _lib
    g = torch.Generator().manual_seed(form)
    m, n, k = 700, 1408, 640
    a = torch.randint(-127, 128, (m, k), generator=g).to(torch.int8)
    b = torch.randint(-127, 128, (n, k), generator=g).to(torch.int8)
    sa, sb, bias = torch.rand((m,), generator=g), torch.rand((n,), generator=g), torch.randn((n,), generator=g).to(dtype) * 1000
    want = product(a.numpy(), sa.numpy(), b.numpy(), sb.numpy(), bias, dtype)
    ops = [t.to(gpu) for t in (a, sa, b, sb, bias)]
    lib = _lib.load()
    lib.hpfp8_debug_set_small_gemm(form)
    try:
        for rows in (m, 256, 70, 5):
            got = hpfp8.gemm_int8(ops[0][:rows], ops[1][:rows], *ops[2:4], bias=ops[4], out_dtype=dtype)
            assert same(got, want[:rows])
    finally:
        lib.hpfp8_debug_set_small_gemm(0)
    assert same(hpfp8.gemm_int8(*ops[:4], bias=ops[4], out_dtype=dtype), want)


@pytest.mark.parametrize("m", [5, 100])
def test_the_longest_contraction_of_the_largest_codes(gpu, m):
    """-128 times -128 over 130944: 2145386496, just below 2^31."""
    import hpfp8
    a = torch.full((m, 130944), -128, dtype=torch.int8, device=gpu)
    b = torch.full((128, 130944), -128, dtype=torch.int8, device=gpu)
    b[1::2] = 127
    one = torch.ones((m,), device=gpu)
    c = hpfp8.gemm_int8(a, one, b, None, out_dtype=torch.float32)
    want = torch.tensor([130944 * 16384, -130944 * 128 * 127], dtype=torch.float64).float()
    assert (c[:, 0::2].cpu() == want[0]).all() and (c[:, 1::2].cpu() == want[1]).all()


def test_strided_codes_and_results_past_2_31_elements(gpu):
    import hpfp8
    g = torch.Generator().manual_seed(5)
    wide = torch.randint(-127, 128, (300, 1024), generator=g).to(torch.int8).to(gpu)
    a, b = wide[:100, 16:528], wide[100:228, 256:768]
    sa, sb = torch.rand((100,), device=gpu), torch.rand((131,), device=gpu)[3:]
    assert torch.equal(hpfp8.gemm_int8(a, sa, b, sb), hpfp8.gemm_int8(a.contiguous(), sa, b.contiguous(), sb.clone()))
    rows, n = 70000, 36864
    few = torch.randint(-127, 128, (700, 128), generator=g).to(torch.int8).to(gpu)
    a = few.repeat(100, 1)
    w = torch.randint(-127, 128, (n, 128), generator=g).to(torch.int8).to(gpu)
    sa = torch.rand((700,), device=gpu)
    c = hpfp8.gemm_int8(a, sa.repeat(100), w, None)
    want = hpfp8.gemm_int8(few, sa, w, None)
    assert c.numel() > 1 << 31 and rows == c.shape[0]
    for at in (0, 34300, 69300):
        assert torch.equal(c[at:at + 700], want)


@pytest.mark.parametrize("tokens", [1, 8, 37, 65, 300, 1531])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [False, True])
def test_linear_and_its_input_gradient(gpu, tokens, dtype, bias):
    """Codes and products bit for bit; then both against the weight's own values in 64 bits: a row's codes are each off by half a scale."""
    import hpfp8
    k, n = 640, 384
    x, w = values(tokens, k, dtype, 6), values(n, k, dtype, 7) * 0.02
    b = values(1, n, dtype, 8)[0] if bias else None
    go = values(tokens, n, dtype, 9)
    w8 = hpfp8.quantize_weight_int8(w.to(gpu))
    codes, sw = quantized(w.float().numpy())
    assert same(w8.codes, torch.from_numpy(codes)) and same(w8.scale_inv, torch.from_numpy(sw))
    xl = x.to(gpu).requires_grad_()
    y = hpfp8.int8_linear(xl, w8, None if b is None else b.to(gpu))
    xq, sx = quantized(x.float().numpy())
    assert same(y.detach(), product(xq, sx, codes, sw, b, dtype))
    dx, = torch.autograd.grad(y, xl, go.to(gpu), retain_graph=True)
    gq, sg = quantized(go.float().numpy() * sw[None, :])
    assert same(dx, product(gq, sg, np.ascontiguousarray(codes.T), None, None, dtype))
    # with transposed codes at hand, without a graph, in three dimensions: the same
    t8 = hpfp8.quantize_weight_int8(w.to(gpu), with_transpose=True)
    y2 = hpfp8.int8_linear(xl, t8, None if b is None else b.to(gpu))
    assert torch.equal(torch.autograd.grad(y2, xl, go.to(gpu))[0], dx) and torch.equal(t8.codes_t, w8.codes.t())
    with torch.no_grad():
        assert torch.equal(hpfp8.int8_linear(xl.view(1, tokens, k), w8, None if b is None else b.to(gpu))[0], y)
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    wv = torch.from_numpy(codes).double() * torch.from_numpy(sw).double()[:, None]
    exact = x.double() @ wv.t() + (0 if b is None else b.double())
    bound = torch.from_numpy(sx).double()[:, None] * 0.5001 * wv.abs().sum(1) + 2 * half * exact.abs() + 1e-6 * (x.double().abs() @ wv.abs().t() + 1)
    assert ((y.detach().double().cpu() - exact).abs() <= bound).all()
    exact = go.double() @ wv
    bound = torch.from_numpy(sg).double()[:, None] * 0.5001 * torch.from_numpy(codes).double().abs().sum(0) + 2 * half * exact.abs() \
        + 1e-6 * (go.double().abs() @ wv.abs() + 1)
    assert ((dx.double().cpu() - exact).abs() <= bound).all()


def test_gradient_against_differences(gpu):
    """The gradient is the straight one through the codes' steps: along a direction it is the slope of x W^T with the codes' weight, which is
    linear, but for the gradient's own codes (half a scale each)."""
    import hpfp8
    x, w, go, d = values(24, 256, torch.float32, 1), values(128, 256, torch.float32, 2), values(24, 128, torch.float32, 3), values(24, 256, torch.float32, 4)
    w8 = hpfp8.quantize_weight_int8(w.to(gpu))
    xl = x.to(gpu).requires_grad_()
    dx, = torch.autograd.grad(hpfp8.int8_linear(xl, w8), xl, go.to(gpu))
    wv = w8.dequantize(torch.float64).cpu()
    f = lambda t: ((t @ wv.t()) * go.double()).sum()          # noqa: E731
    h = 2.0 ** -10
    slope = (f(x.double() + h * d.double()) - f(x.double() - h * d.double())) / (2 * h)
    _, sg = quantized(go.numpy() * w8.scale_inv.cpu().numpy()[None, :])
    spread = 0.5001 * (torch.from_numpy(sg).double()[:, None] * (w8.codes.cpu().double().abs().sum(0)) * d.double().abs()).sum()
    assert abs(float((dx.cpu().double() * d.double()).sum() - slope)) <= float(spread) + 1e-6 * abs(float(slope))


def test_no_tokens(gpu):
    import hpfp8
    w8 = hpfp8.quantize_weight_int8(values(128, 256, torch.bfloat16, 1).to(gpu))
    x = torch.zeros((0, 3, 256), dtype=torch.bfloat16, device=gpu, requires_grad=True)
    y = hpfp8.int8_linear(x, w8)
    dx, = torch.autograd.grad(y, x, torch.zeros_like(y))
    assert y.shape == (0, 3, 128) and dx.shape == x.shape
    with torch.no_grad():
        assert hpfp8.int8_linear(x, w8).shape == (0, 3, 128)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("with_transpose", [False, True])
def test_module_form(gpu, bias, with_transpose):
    import hpfp8
    linear = torch.nn.Linear(256, 384, bias=bias, device=gpu, dtype=torch.bfloat16)
    made = hpfp8.Int8Linear.from_linear(linear, with_transpose=with_transpose)
    x = values(40, 256, torch.bfloat16, 2).to(gpu).requires_grad_()
    w8 = hpfp8.quantize_weight_int8(linear.weight)
    y = made(x)
    b = None if not bias else linear.bias.detach()
    assert torch.equal(y, hpfp8.int8_linear(x, w8, b)) and (made.weight_codes_t is not None) == with_transpose
    go = values(40, 384, torch.bfloat16, 3).to(gpu)
    want, = torch.autograd.grad(hpfp8.int8_linear(x, w8, b), x, go)
    assert torch.equal(torch.autograd.grad(y, x, go)[0], want)
    assert list(made.state_dict()) == ["weight_codes", "weight_scale_inv"] + ["bias"] * bias
    other = hpfp8.Int8Linear(256, 384, bias=bias, with_transpose=with_transpose, device=gpu)
    other(x)                                                 # (its transposed codes are those of zeros)
    other.load_state_dict(made.state_dict())
    assert torch.equal(torch.autograd.grad(other(x), x, go)[0], want)
    with torch.no_grad():
        other.weight_codes.neg_()
    assert torch.equal(torch.autograd.grad(other(x), x, go)[0], -want)
    other.weight_codes = w8.codes.clone()
    assert torch.equal(torch.autograd.grad(other(x), x, go)[0], want)
    other.refresh()
    assert torch.equal(torch.autograd.grad(other(x), x, go)[0], want)
    assert not list(made.parameters()) and "in_features=256" in repr(made)
    there = made.cpu().to(gpu)                               # (codes and transposed codes move together)
    assert torch.equal(torch.autograd.grad(there(x), x, go)[0], want)
    half = made.to(torch.float16)
    assert half.weight_scale_inv.dtype == torch.float32 and half.weight_codes.dtype == torch.int8
    assert torch.equal(half(x.detach().half()), hpfp8.int8_linear(x.detach().half(), w8, None if b is None else b.half()))
    import copy
    twin = copy.deepcopy(there).to(torch.bfloat16)
    assert torch.equal(torch.autograd.grad(twin(x), x, go)[0], want)
    with torch.inference_mode():
        served = hpfp8.Int8Linear.from_linear(linear, with_transpose=with_transpose)
        assert torch.equal(served(x.detach()), y)
    fp8 = hpfp8.Fp8Linear(256, 384, device=gpu)
    assert hpfp8.Int8Linear.from_linear(fp8)(x.detach()).shape == (40, 384)


def operator():
    import hpfp8
    w8 = hpfp8.quantize_weight_int8(values(128, 256, torch.bfloat16, 1).cuda())
    return lambda a: hpfp8.int8_linear(a, w8), (values(48, 256, torch.bfloat16, 2).cuda(),), values(48, 128, torch.bfloat16, 3).cuda()


@pytest.mark.parametrize("way", WAYS)
def test_under_what_else_torch_does_with_a_step(gpu, way, monkeypatch):
    from hpfp8 import ops
    f, tensors, go = operator()

    def outcome(way):
        try:
            r = step(f, tuple(t.clone().requires_grad_() for t in tensors), go.detach().clone(), way)
        except Exception as e:
            return type(e), str(e).split("\n")[0].split(" is a view")[-1]
        return [t.detach() for t in r] if isinstance(r, (tuple, list)) else [r.detach()]
    got = outcome(way)
    if way in ("mode", "trace", "trace_inference", "create_graph", "checkpoint", "reentrant", "detect_anomaly", "retained", "other_stream", "in_place"):
        assert isinstance(got, list), got
        plain = outcome("plain")
        plain[0] = plain[0] + 1 if way == "in_place" else plain[0]
        plain = plain[:1] if way.startswith("trace") else (plain[1:] if len(got) < len(plain) else plain)
        assert len(got) == len(plain) and all(torch.equal(a, b) for a, b in zip(got, plain))
    monkeypatch.setattr(ops, "_native", types.SimpleNamespace(**{
        k: (lambda *a: None) if k in ("int8_linear", "quantize_int8", "gemm_int8") else getattr(ops._native, k)
        for k in dir(ops._native) if not k.startswith("__")}))
    want = outcome(way)
    if isinstance(want, tuple):
        assert got == want or got[0] is want[0]
    else:
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_tangent_is_refused_and_not_dropped(gpu):
    import torch.autograd.forward_ad as fwAD
    f, (x,), _ = operator()
    for grad in (True, False):
        with torch.set_grad_enabled(grad), fwAD.dual_level():
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward mode"):
                f(fwAD.make_dual(x, torch.ones_like(x)))
            inside = f(x)
        assert torch.equal(inside, f(x))


def test_a_write_to_the_codes_in_between_is_noticed_and_kept_activations_leave_them(gpu):
    import hpfp8
    w8 = hpfp8.quantize_weight_int8(values(128, 256, torch.bfloat16, 1).to(gpu))
    x, go = values(48, 256, torch.bfloat16, 2).to(gpu).requires_grad_(), values(48, 128, torch.bfloat16, 3).to(gpu)
    want, = torch.autograd.grad(hpfp8.int8_linear(x, w8), x, go)
    with hpfp8.keep_activations_8bit(min_elements=1):
        got, = torch.autograd.grad(hpfp8.int8_linear(x, w8), x, go)
    assert torch.equal(got, want)
    y = hpfp8.int8_linear(x, w8)
    w8.codes.neg_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, go)


def test_captured_and_replayed(gpu):
    import hpfp8
    w8 = hpfp8.quantize_weight_int8(values(1024, 512, torch.bfloat16, 1).to(gpu), with_transpose=True)
    x0, go = values(700, 512, torch.bfloat16, 2).to(gpu), values(700, 1024, torch.bfloat16, 3).to(gpu)
    x = x0.clone().requires_grad_()

    def run():
        y = hpfp8.int8_linear(x, w8)
        with torch.no_grad():
            few = hpfp8.int8_linear(x[:8], w8)
        return y.detach(), torch.autograd.grad(y, x, go)[0], few
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
            x.copy_(x0 * (k + 1) + k)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, run()))


def test_refused(gpu):
    import hpfp8
    w = values(128, 256, torch.bfloat16, 1).to(gpu)
    w8 = hpfp8.quantize_weight_int8(w)
    x = values(4, 256, torch.bfloat16, 2).to(gpu)
    bias = torch.zeros(128, dtype=torch.bfloat16, device=gpu)
    for wrong, error in (((x, w), TypeError), ((x[:, :128], w8), ValueError), ((x.double(), w8), TypeError), ((x, w8, bias.float()), TypeError),
                         ((x, w8, bias[:64]), ValueError), ((x, w8, bias.clone().requires_grad_()), ValueError), ((x.cpu(), w8), ValueError),
                         ((x, w8._replace(scale_inv=w8.scale_inv[:64])), ValueError), ((x, w8._replace(codes=w8.codes.float())), TypeError),
                         ((x, w8._replace(codes_t=w8.codes)), ValueError), ((x, w8._replace(scale_inv=w8.scale_inv.double())), TypeError)):
        with pytest.raises(error):
            hpfp8.int8_linear(*wrong)
    for f in (lambda: hpfp8.quantize_int8(x[:, :100]), lambda: hpfp8.quantize_int8(x, column_scale=torch.ones(128, device=gpu)),
              lambda: hpfp8.gemm_int8(w8.codes, w8.scale_inv, w8.codes[:64], None), lambda: hpfp8.gemm_int8(w8.codes, w8.scale_inv[:5], w8.codes, None),
              lambda: hpfp8.gemm_int8(w8.codes.t(), w8.scale_inv, w8.codes, None), lambda: hpfp8.quantize_weight_int8(w[:100]),
              lambda: hpfp8.Int8Linear(100, 128)):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(TypeError):
        hpfp8.gemm_int8(w, w8.scale_inv, w8.codes, None)
    with pytest.raises(TypeError):
        hpfp8.gemm_int8(w8.codes, w8.scale_inv, w8.codes, None, out_dtype=torch.float64)
    with torch.no_grad():
        assert hpfp8.int8_linear(x, w8, bias.clone().requires_grad_()).shape == (4, 128)


def test_more_than_2_31_values_quantized_and_codes_of_a_weight_past_2_31(gpu):
    import hpfp8
    rows, cols = (1 << 31) // 4096 + 64, 4096
    part = values(64, cols, torch.bfloat16, 1).to(gpu)
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device=gpu)
    x.view(-1, 64, cols)[:] = part
    by = torch.rand((cols,), device=gpu)
    codes, scale = hpfp8.quantize_int8(x, column_scale=by)
    want, want_scale = hpfp8.quantize_int8(part, column_scale=by)
    for at in (0, rows - 64):
        assert torch.equal(codes[at:at + 64], want) and torch.equal(scale[at:at + 64], want_scale)
    del x
    one = torch.ones((5,), device=gpu)
    assert rows % 128 == 64
    w = codes[:rows - 64]                                    # [524288, 4096]
    for a in (want[:5], want):
        s = torch.ones((a.shape[0],), device=gpu)
        c = hpfp8.gemm_int8(a, s, w, None)
        few = hpfp8.gemm_int8(a, s, want.repeat(2, 1), None)
        for at in (0, w.shape[0] - 128):
            assert torch.equal(c[:, at:at + 128], few)
    del one


def test_hooks_on_saved_tensors(gpu):
    """What a hook hands back is looked at: as it was or packed elsewhere and back it is used, anything else is refused."""
    import hpfp8
    f, (x,), go = operator()
    xl = x.clone().requires_grad_()
    want, = torch.autograd.grad(f(xl), xl, go)
    with torch.autograd.graph.save_on_cpu():
        y = f(xl)
    assert torch.equal(torch.autograd.grad(y, xl, go)[0], want)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t):
        y = f(xl)
    assert torch.equal(torch.autograd.grad(y, xl, go)[0], want)
    for wrong in (lambda t: t.float(), lambda t: t[:-1], lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, wrong):
            y = f(xl)
        with pytest.raises((ValueError, TypeError)):
            torch.autograd.grad(y, xl, go)


def test_steps_of_several_threads_at_once(gpu):
    import threading
    import hpfp8
    w8 = hpfp8.quantize_weight_int8(values(512, 1024, torch.bfloat16, 1).to(gpu))
    norm_w = torch.ones(1024, dtype=torch.bfloat16, device=gpu)
    xs = [values(200 + 50 * i, 1024, torch.bfloat16, 10 + i).to(gpu) for i in range(4)]

    def run(i):
        x = xs[i].clone().requires_grad_()
        y, s = hpfp8.rms_norm(x, 1024, norm_w, residual=xs[i])
        z = hpfp8.int8_linear(y, w8)
        dx, = torch.autograd.grad((z, s), x, (torch.ones_like(z), torch.ones_like(s)))
        p = torch.nn.Parameter(torch.zeros_like(x))
        p.grad = dx.clone()
        norm = hpfp8.clip_grad_norm_([p], 1.0)
        return z.detach(), dx, norm, p.grad
    want = [run(i) for i in range(4)]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = run(i)
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("with_transpose", [True, False])
def test_small_gradients_scale_along(gpu, dtype, native, with_transpose, monkeypatch):
    """Every step from dy to dx (times a scale, the row's largest, its codes, their integer sum times the row's scale) commutes with a power of two while
    nothing is subnormal: the gradient of 2^-k dy is 2^-k times that of dy, bit for bit, each row by a k of its own."""
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    w8 = hpfp8.quantize_weight_int8((values(384, 256, torch.bfloat16, 1) * 0.02).to(gpu), with_transpose)
    x = values(96, 256, dtype, 2).to(gpu).requires_grad_()
    go = values(96, 384, dtype, 3).to(gpu)
    # (2^-84 of dy, which is 1e-5 at its least, times a scale of 1e-3 is 1e-34: a normal number, and the row's largest is above 2^-118)
    by = torch.exp2(-torch.arange(96, device=gpu).float() * 84 / 95).log2().round().exp2().unsqueeze(1)
    want, = torch.autograd.grad(hpfp8.int8_linear(x, w8), x, go)
    got, = torch.autograd.grad(hpfp8.int8_linear(x, w8), x, go * by.to(dtype))
    assert by.min() == 2.0 ** -84 and (want != 0).any(1).all()
    assert torch.equal(got, want * by.to(dtype))


def test_gradients_of_zeros_subnormals_and_no_numbers(gpu):
    import hpfp8
    w8 = hpfp8.quantize_weight_int8((values(384, 256, torch.bfloat16, 1) * 0.02).to(gpu))
    x = values(7, 256, torch.float32, 2).to(gpu).requires_grad_()
    go = torch.zeros((7, 384), device=gpu)
    go[1, 5], go[2], go[3, 1] = 1e-45, 2.0 ** -140, 1e-38
    go[4, 0], go[5, 3], go[6] = math.inf, math.nan, 3e38
    dx, = torch.autograd.grad(hpfp8.int8_linear(x, w8), x, go)
    assert (dx[0] == 0).all() and torch.isfinite(dx[:4]).all() and dx[:4].abs().max() < 1e-35 and torch.isnan(dx[4:6]).all()
    # the largest: 3e38 times the channels' scales, codes and one scale for the row, which an fp32 holds
    wv = w8.dequantize(torch.float64)
    assert torch.isfinite(dx[6][(wv.sum(0).abs() * 3e38) < 1e38]).all()


@pytest.mark.parametrize("cols", [128, 2048, 16512])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_codes_of_small_rows_with_column_scales(gpu, cols, dtype):
    """A row's largest value behind the columns' scales is held from below by 2^-118 alone, where 127 / amax and amax / 127 are both normal numbers."""
    import hpfp8
    x = values(6, cols, dtype, 1) * torch.tensor([0.0, 2.0 ** -34, 2.0 ** -60, 2.0 ** -90, 2.0 ** -110, 2.0 ** -120])[:, None].to(dtype)
    by = torch.rand((cols,), generator=torch.Generator().manual_seed(2)) * 0.01
    v = x.float().numpy() * by.numpy()[None, :]
    amax = np.maximum(np.abs(v).max(1, keepdims=True), np.float32(2.0 ** -118))
    codes = np.rint(v * (np.float32(127.0) / amax)).astype(np.int8)
    got, scale = hpfp8.quantize_int8(x.to(gpu), column_scale=by.to(gpu))
    assert same(got, torch.from_numpy(codes)) and same(scale, torch.from_numpy((amax / np.float32(127.0))[:, 0]))
    assert got[1:5].abs().amax(1).eq(127).all() and not got[0].any()


@pytest.mark.parametrize("native", [True, False])
def test_traces_and_tangents_of_the_operators_by_themselves_are_refused(gpu, native, monkeypatch):
    import hpfp8
    import torch.autograd.forward_ad as fwAD
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    x, w8 = values(48, 256, torch.bfloat16, 1).to(gpu), hpfp8.quantize_weight_int8(values(128, 256, torch.bfloat16, 2).to(gpu))
    codes, scale = hpfp8.quantize_int8(x)
    bias = torch.zeros((128,), dtype=torch.bfloat16, device=gpu)
    for name, f, t in (("quantize_int8", hpfp8.quantize_int8, x), ("gemm_int8", lambda t: hpfp8.gemm_int8(codes, t, w8.codes, w8.scale_inv), scale),
                       ("gemm_int8", lambda t: hpfp8.gemm_int8(codes, scale, w8.codes, w8.scale_inv, t), bias)):
        with torch.no_grad(), pytest.raises(RuntimeError, match=f"{name} has no place in a trace"):
            torch.jit.trace(f, (t,), check_trace=False)
        with fwAD.dual_level():
            with pytest.raises(RuntimeError, match="forward mode"):
                f(fwAD.make_dual(t, torch.ones_like(t)))
            inside = f(t)
        after = f(t)
        assert all(torch.equal(a, b) for a, b in zip(inside, after))


@pytest.mark.parametrize("native", [True, False])
def test_gradients_that_a_product_does_not_have_are_refused_and_not_lost(gpu, native, monkeypatch):
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    w8 = hpfp8.quantize_weight_int8(values(128, 256, torch.bfloat16, 1).to(gpu))
    codes, scale = hpfp8.quantize_int8(values(8, 256, torch.bfloat16, 2).to(gpu))
    bias = torch.ones((128,), dtype=torch.bfloat16, device=gpu)
    want = hpfp8.gemm_int8(codes, scale, w8.codes, w8.scale_inv, bias)
    learned = lambda t: t.clone().requires_grad_()           # noqa: E731
    for sa, sb, b in ((learned(scale), w8.scale_inv, bias), (scale, learned(w8.scale_inv), bias), (scale, w8.scale_inv, learned(bias))):
        with pytest.raises(ValueError, match="no gradient"):
            hpfp8.gemm_int8(codes, sa, w8.codes, sb, b)
        with torch.no_grad():
            assert torch.equal(hpfp8.gemm_int8(codes, sa, w8.codes, sb, b), want)
    x = values(8, 256, torch.bfloat16, 2).to(gpu)
    for t in (x, learned(x)):
        with pytest.raises(ValueError, match="no gradient"):
            hpfp8.int8_linear(t, w8._replace(scale_inv=learned(w8.scale_inv)), bias)


@pytest.mark.parametrize("out", [256, 384])
@pytest.mark.parametrize("form", ["transposed", "module", "plain", "strided"])
def test_the_native_backward_takes_the_codes_that_the_package_makes(gpu, out, form):
    """Transposed codes of an even multiple of 128 outputs have rows with a gap behind them; codes that are a slice have one too."""
    import hpfp8
    from hpfp8 import int8, ops
    k = 512
    w = (values(out, k, torch.bfloat16, 1) * 0.02).to(gpu)
    w8 = hpfp8.quantize_weight_int8(w, with_transpose=form == "transposed")
    assert form != "transposed" or w8.codes_t.is_contiguous() == (out == 384)
    f = lambda t: hpfp8.int8_linear(t, w8)                   # noqa: E731
    if form == "strided":
        wide = torch.zeros((out, k + 256), dtype=torch.int8, device=gpu)
        wide[:, 128:128 + k] = w8.codes
        w8 = w8._replace(codes=wide[:, 128:128 + k])
    elif form == "module":
        linear = torch.nn.Linear(k, out, bias=False, device=gpu, dtype=torch.bfloat16)
        linear.weight.data.copy_(w)
        f = hpfp8.Int8Linear.from_linear(linear, with_transpose=True)
        assert not f.weight_codes_t.is_contiguous() or out == 384
    x, go = values(70, k, torch.bfloat16, 2).to(gpu).requires_grad_(), values(70, out, torch.bfloat16, 3).to(gpu)
    codes, sw = quantized(w.float().cpu().numpy())
    gq, sg = quantized(go.float().cpu().numpy() * sw[None, :])
    want = product(gq, sg, np.ascontiguousarray(codes.T), None, None, torch.bfloat16)

    def python(*a):
        raise AssertionError("the native backward left this to Python")
    ops._native.bind_int8_backward(python)
    try:
        dx, = torch.autograd.grad(f(x), x, go)
    finally:
        ops._native.bind_int8_backward(int8._int8_backward)
    assert same(dx, want)


@pytest.mark.parametrize("cols", [128, 512, 2048, 16512])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [9, 99])
def test_products_of_rows_at_the_edges(gpu, cols, dtype, tokens):
    """Bit for bit from the codes, with a weight whose rows cancel the largest values of a type or let them overflow to an infinity, as one rounding
    to the type does; tokens: few rows, and tiles."""
    import hpfp8
    top = torch.finfo(dtype).max
    x = torch.zeros((tokens, cols), dtype=torch.float64)
    x[1, 3] = 1e-14
    x[2, 5], x[2, 9] = -1e-39, 5e-40
    x[3, 0], x[3, 1] = top, -top
    x[4] = torch.arange(cols, dtype=torch.float64) % 255 - 127
    x[5, 0], x[5, 1:5] = 127, torch.tensor([0.5, 1.5, -2.5, 126.5])
    x[6, 0], x[6, 1] = top, top
    x = x.to(dtype)
    w = torch.ones((128, cols), dtype=dtype)
    w[1::2, 1] = -1
    w[2::4] *= 0.001
    codes, scale = quantized(x.float().numpy())
    wq, sw = quantized(w.float().numpy())
    with np.errstate(over="ignore"):
        want = product(codes, scale, wq, sw, None, dtype)
    y = hpfp8.int8_linear(x.to(gpu), hpfp8.quantize_weight_int8(w.to(gpu)))
    assert same(y, want)
    assert (want[0] == 0).all() and torch.isinf(want[3, 1]) and want[3, 0] == 0 and torch.isfinite(want[[1, 2, 4, 5]].float()).all()
