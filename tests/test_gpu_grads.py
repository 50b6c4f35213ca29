"""The global norm of gradients and their clipping: the norm against 64 bits, the clipped values bit for bit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def tensors(sizes, seed, std=1.0, dtypes=TYPES):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn((n,), generator=g) * std).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def norm64(ts, p):
    flat = torch.cat([t.double().reshape(-1) for t in ts]) if ts else torch.zeros(0, dtype=torch.float64)
    return torch.linalg.vector_norm(flat, p) if flat.numel() else torch.zeros((), dtype=torch.float64)


def near(got, want):
    """Sums of up to 2^32 terms in 64 bits are off by 2^-53 of each addition: one rounding to fp32 is all that is left."""
    assert got.dtype == torch.float32 and got.shape == () and got.is_cuda
    assert abs(float(got) - float(want)) <= 2.0 ** -24 * 1.0001 * float(want), (float(got), float(want))


def params(ts):
    """Parameters of 16 bits with their grads; of fp32 ones with main_grads."""
    out = []
    for t in ts:
        if t.dtype == torch.float32:
            p = torch.nn.Parameter(torch.zeros(t.shape, dtype=torch.bfloat16, device=t.device))
            p.main_grad = t
        else:
            p = torch.nn.Parameter(torch.zeros(t.shape, dtype=t.dtype, device=t.device))
            p.grad = t
        out.append(p)
    return out


def clipped(ts, norm, max_norm):
    factor = torch.clamp(torch.tensor(max_norm, dtype=torch.float32) / (norm.cpu() + torch.tensor(1e-6, dtype=torch.float32)), max=1.0)
    return [(t.float() * factor).to(t.dtype) for t in ts]


SIZES = [[1], [7, 1, 3], [0, 5, 0], [4096], [8191, 8192, 8193], [16384 * 3 + 5, 1, 100000], [1000003], list(range(1, 400)), [17] * 161, [2] * 320, [3 << 20, 5, 1 << 21]]


@pytest.mark.parametrize("sizes", SIZES, ids=[str(i) for i in range(len(SIZES))])
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("native", [True, False])
def test_norm_and_clipping(gpu, sizes, p, native, monkeypatch):
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    ts = tensors(sizes, 1)
    on = [t.to(gpu) for t in ts]
    want = norm64(ts, p)
    norm = hpfp8.get_total_norm(on, p)
    near(norm, want)
    assert torch.equal(norm, hpfp8.get_total_norm(tuple(on), p))
    for share in (0.3, 3.0):
        ps = params([t.clone() for t in on])
        max_norm = share * float(want)
        got = hpfp8.clip_grad_norm_(ps, max_norm, p)
        assert torch.equal(got, norm)
        expected = clipped(ts, norm, max_norm)
        for q, t in zip(ps, expected):
            assert torch.equal((q.grad if q.grad is not None else q.main_grad).cpu(), t)


def test_against_torchs_own(gpu):
    import hpfp8
    ts = [t.to(gpu) for t in tensors([1000, 64 * 128, 5], 2, dtypes=[torch.float32])]
    a = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts]
    b = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts]
    for p, q, t in zip(a, b, ts):
        p.grad, q.grad = t.clone(), t.clone()
    x, y = hpfp8.clip_grad_norm_(iter(a), 1.5), torch.nn.utils.clip_grad_norm_(b, 1.5)
    assert abs(float(x) - float(y)) < 1e-6 * float(y)
    for p, q in zip(a, b):
        assert ((p.grad - q.grad).abs() <= 1e-6 * q.grad.abs()).all()
    near(hpfp8.clip_grad_norm_(a[0], 1e9), norm64([a[0].grad.cpu()], 2.0))
    hpfp8.clip_grads_with_norm_(a, 1.0, torch.tensor(2.0, device=gpu))
    hpfp8.clip_grads_with_norm_(b, 1.0, 2.0)
    torch.nn.utils.clip_grads_with_norm_(b, 1.0, torch.tensor(0.5, device=gpu))
    for p, q in zip(a, b):
        assert ((p.grad - q.grad).abs() <= 1e-6 * q.grad.abs()).all()


def test_values_whose_squares_32_bits_do_not_hold(gpu):
    import hpfp8
    for size in (1e30, 1e-30, 2.0 ** 127, 2.0 ** -126):
        for dtype in (torch.float32, torch.bfloat16):
            t = torch.full((1 if size > 1e38 else 300,), size, dtype=dtype)
            near(hpfp8.get_total_norm([t.to(gpu)]), norm64([t], 2.0))
    big = torch.full((9,), 3e38, device=gpu)
    assert math.isinf(float(hpfp8.get_total_norm([big])))                # (the norm itself does not fit)
    near(hpfp8.get_total_norm([big], math.inf), torch.tensor(3e38).double())


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_infinities_and_nan(gpu, p):
    import hpfp8
    for bad in (math.inf, -math.inf, math.nan):
        ts = [t.to(gpu) for t in tensors([1000, 30000, 5], 3)]
        ts[1][12345] = bad
        norm = hpfp8.get_total_norm(ts, p)
        assert (math.isnan(float(norm)) if math.isnan(bad) else float(norm) == math.inf)
        ps = params([t.clone() for t in ts])
        with pytest.raises(RuntimeError, match="non-finite"):
            hpfp8.clip_grad_norm_(ps, 1.0, p, error_if_nonfinite=True)
        assert all(torch.equal(torch.nan_to_num(q.grad if q.grad is not None else q.main_grad), torch.nan_to_num(t)) for q, t in zip(ps, ts))
        hpfp8.clip_grad_norm_(ps, 1.0, p)
        for q, t in zip(ps, ts):                                         # (what torch's makes of it: times 0, or NaN)
            got = q.grad if q.grad is not None else q.main_grad
            want = t.float() * torch.clamp(1.0 / (norm + 1e-6), max=1.0)
            assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want.to(got.dtype)))
    both = torch.tensor([math.nan, math.inf], device=gpu)
    assert math.isnan(float(hpfp8.get_total_norm([both], p))) and math.isnan(float(hpfp8.get_total_norm([both.flip(0)], p)))


def test_starts_between_vectors_and_what_lies_around(gpu):
    """Views of one buffer at every offset: neighbours keep their bits."""
    import hpfp8
    for dtype in TYPES:
        buffer = torch.randn((9000,), generator=torch.Generator().manual_seed(4)).to(dtype)
        on = buffer.to(gpu)
        spans = [(1, 8), (9, 4105), (4107, 4108), (4113, 8990)]
        parts = [on[a:b] for a, b in spans]
        norm = hpfp8.get_total_norm(parts)
        near(norm, norm64([buffer[a:b] for a, b in spans], 2.0))
        ps = []
        for t in parts:
            p = torch.nn.Parameter(torch.zeros(t.shape, dtype=dtype, device=gpu))
            p.grad = t
            ps.append(p)
        hpfp8.clip_grads_with_norm_(ps, 2.0, norm)
        want = buffer.clone()
        for a, b in spans:
            want[a:b] = clipped([buffer[a:b]], norm, 2.0)[0]
        assert torch.equal(on.cpu(), want)


def test_strides(gpu):
    import hpfp8
    g = torch.Generator().manual_seed(5)
    base = torch.randn((64, 96), generator=g).to(gpu)
    wide = torch.randn((64, 200), generator=g).to(torch.bfloat16).to(gpu)
    grads = [base.t(), wide[:, 3:90], torch.randn((2, 3, 4, 5), generator=g).to(gpu).to(memory_format=torch.channels_last)]
    cpu = [t.cpu() for t in grads]
    around = wide.clone()
    norm = hpfp8.get_total_norm(grads)
    near(norm, norm64(cpu, 2.0))
    ps = []
    for t in grads:
        p = torch.nn.Parameter(torch.zeros(t.shape, dtype=t.dtype, device=gpu))
        p.grad = t
        ps.append(p)
    hpfp8.clip_grads_with_norm_(ps, 1.0, norm)
    for p, w in zip(ps, clipped(cpu, norm, 1.0)):
        assert torch.equal(p.grad.cpu(), w)
    assert torch.equal(wide[:, :3], around[:, :3]) and torch.equal(wide[:, 90:], around[:, 90:])


def test_gradients_that_are_shared_or_missing(gpu):
    import hpfp8
    t = torch.randn((1000,), device=gpu)
    p, q, empty = (torch.nn.Parameter(torch.zeros(1000, device=gpu)) for _ in range(3))
    p.grad = t.clone()
    q.grad = p.grad
    norm = hpfp8.clip_grad_norm_([p, p, q, empty], 1.0)                  # one gradient, named three times
    near(norm, norm64([t.cpu()], 2.0))
    assert torch.equal(p.grad.cpu(), clipped([t.cpu()], norm, 1.0)[0])
    q.grad = p.grad[:]                                                   # the same memory as another tensor
    before = p.grad.clone()
    for a, b in ((0, 1000), (0, 999), (1, 1000), (500, 501)):
        q = torch.nn.Parameter(torch.zeros(b - a, device=gpu))
        q.grad = p.grad[a:b]
        with pytest.raises(hpfp8._lib.Hpfp8Error, match="share memory"):
            hpfp8.clip_grad_norm_([p, q], 1e-3)
    assert torch.equal(p.grad, before)
    zero = hpfp8.clip_grad_norm_([empty], 1.0)
    assert float(zero) == 0 and zero.is_cuda and float(hpfp8.get_total_norm([])) == 0
    assert hpfp8.clip_grads_with_norm_([], 1.0, zero) is None
    # a main gradient is the gradient
    main = torch.nn.Parameter(torch.zeros(1000, dtype=torch.bfloat16, device=gpu))
    main.main_grad = t.clone()
    near(hpfp8.clip_grad_norm_(main, 1.0), norm64([t.cpu()], 2.0))
    assert torch.equal(main.main_grad.cpu(), clipped([t.cpu()], norm, 1.0)[0])
    main.grad = torch.zeros(1000, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(ValueError, match="main_grad"):
        hpfp8.clip_grad_norm_([main], 1.0)
    same = torch.nn.Parameter(torch.zeros(1000, device=gpu))
    same.grad = same.main_grad = t.clone()
    near(hpfp8.clip_grad_norm_([same], 1.0), norm64([t.cpu()], 2.0))
    assert torch.equal(same.grad.cpu(), clipped([t.cpu()], norm, 1.0)[0])


@pytest.mark.parametrize("native", [True, False])
def test_autograd_sees_the_write(gpu, native, monkeypatch):
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    x = torch.randn((64,), device=gpu, requires_grad=True)
    g = torch.randn((64,), device=gpu)
    y = x * g                                                # (saves g)
    p = torch.nn.Parameter(torch.zeros(64, device=gpu))
    p.grad = g
    hpfp8.clip_grad_norm_([p], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refused(gpu):
    import hpfp8
    p = torch.nn.Parameter(torch.zeros(8, device=gpu))
    p.grad = torch.ones(8, device=gpu)
    for f in (lambda: hpfp8.get_total_norm([p.grad], 3.0), lambda: hpfp8.get_total_norm([p.grad], -math.inf), lambda: hpfp8.get_total_norm([p.grad], 0),
              lambda: hpfp8.clip_grad_norm_([p], -1.0), lambda: hpfp8.clip_grad_norm_([p], math.nan), lambda: hpfp8.get_total_norm([torch.ones(3)]),
              lambda: hpfp8.clip_grads_with_norm_([p], 1.0, torch.ones(2, device=gpu))):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: hpfp8.get_total_norm([p.grad.double()]), lambda: hpfp8.get_total_norm([3]), lambda: hpfp8.get_total_norm([p.grad.to_sparse()]),
              lambda: hpfp8.get_total_norm([p.grad.to(torch.float8_e4m3fn)])):
        with pytest.raises(TypeError):
            f()
    assert (p.grad == 1).all()


def test_the_same_bits_every_time_captured_and_on_another_stream(gpu):
    import hpfp8
    source = [t.to(gpu) for t in tensors([1 << 20, 70001, 3, 5000] + [900] * 200, 6)]
    held = [t.clone() for t in source]
    ps = params(held)

    def run():
        return hpfp8.clip_grad_norm_(ps, 10.0)
    want_norm = run()
    want = [t.clone() for t in held]
    side = torch.cuda.Stream()
    for t, s in zip(held, source):
        t.copy_(s)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, want_norm) and all(torch.equal(a, b) for a, b in zip(held, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = run()
    for k in range(4):
        for t, s in zip(held, source):
            t.copy_(s * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        got, got_norm = [t.clone() for t in held], norm.clone()
        for t, s in zip(held, source):
            t.copy_(s * (k + 1))
        assert torch.equal(run(), got_norm) and all(torch.equal(a, b) for a, b in zip(held, got))
        assert k or (torch.equal(got_norm, want_norm) and all(torch.equal(a, b) for a, b in zip(got, want)))


def test_more_than_2_31_elements(gpu):
    import hpfp8
    n = (1 << 31) + 77
    t = torch.zeros((n,), dtype=torch.bfloat16, device=gpu)
    t[0], t[1 << 30], t[-1] = 3.0, 4.0, 12.0
    assert float(hpfp8.get_total_norm([t])) == 13.0 and float(hpfp8.get_total_norm([t], 1)) == 19.0 and float(hpfp8.get_total_norm([t], math.inf)) == 12.0
    p = torch.nn.Parameter(torch.zeros((1,), dtype=torch.bfloat16, device=gpu).expand(n))
    p.grad = t
    hpfp8.clip_grads_with_norm_(p, 6.5, torch.tensor(13.0, device=gpu))
    assert [float(t[i]) for i in (0, 1 << 30, n - 1)] == [1.5, 2.0, 6.0] and int((t != 0).sum()) == 3


@pytest.mark.parametrize("p", [2.0, math.inf])
def test_more_than_the_caches_hold(gpu, p):
    """Streamed: over 256 MiB, in more tensors than a launch takes, odd sizes of every type, starts between vectors."""
    import hpfp8
    sizes = [40_000_003, 30_000_001, 33_333_333] + [1009 + 7 * i for i in range(170)]
    flats = {d: torch.randn((sum(sizes[i::3]) + 1,), generator=torch.Generator().manual_seed(7)).to(d) for i, d in enumerate(TYPES)}
    on = {d: t.to(gpu) for d, t in flats.items()}
    before = {d: t.clone() for d, t in flats.items()}
    ps, at = [], dict.fromkeys(TYPES, 1)
    for i, n in enumerate(sizes):
        d = TYPES[i % 3]
        q = torch.nn.Parameter(torch.zeros((1,), dtype=d, device=gpu).expand(n))
        q.grad = on[d][at[d]:at[d] + n]
        at[d] += n
        ps.append(q)
    assert sum(q.grad.numel() * q.grad.element_size() for q in ps) > 256 << 20
    want = norm64([t[1:] for t in flats.values()], p)
    norm = hpfp8.get_total_norm([q.grad for q in ps], p)
    near(norm, want)
    assert torch.equal(hpfp8.clip_grad_norm_(ps, 10 * float(want), p), norm)
    assert all(torch.equal(on[d].cpu(), before[d]) for d in TYPES)       # (the bound holds)
    assert torch.equal(hpfp8.clip_grad_norm_(ps, 0.25 * float(want), p), norm)
    for d in TYPES:
        got = on[d].cpu()
        assert torch.equal(got[1:], clipped([before[d][1:]], norm, 0.25 * float(want))[0]) and got[0] == before[d][0]


def test_around_the_size_that_is_streamed(gpu):
    """The same values in one form and in the other have the same norm and become the same."""
    import hpfp8
    n = (256 << 20) // 4
    t = torch.randn((n + 5000,), device=gpu, generator=torch.Generator(device=gpu).manual_seed(8))
    for m in (n - 1, n, n + 1, n + 4097):
        part = t[:m].clone()
        q = torch.nn.Parameter(torch.zeros((1,), device=gpu).expand(m))
        q.grad = part
        norm = hpfp8.clip_grad_norm_(q, 100.0)
        assert abs(float(norm) - float(torch.linalg.vector_norm(t[:m].double()))) <= 2.0 ** -23 * float(norm)
        factor = torch.tensor(100.0, device=gpu) / (norm + 1e-6)
        assert torch.equal(part, t[:m] * factor)


@pytest.mark.parametrize("native", [True, False])
def test_tensors_made_in_inference_mode(gpu, native, monkeypatch):
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    with torch.inference_mode():
        g = torch.full((1000,), 2.0, device=gpu)
        q = torch.nn.Parameter(torch.zeros(1000, device=gpu))
        q.main_grad = g
        near(hpfp8.clip_grad_norm_([q], 1e9), torch.tensor(2.0 * 1000 ** 0.5, dtype=torch.float64))
        hpfp8.clip_grads_with_norm_([q], 1.0, torch.tensor(2.0, device=gpu))
        assert torch.equal(g, torch.full_like(g, 2.0) * (1.0 / (torch.tensor(2.0, device=gpu) + 1e-6)))


def test_half_a_parameters_gradient_in_each_place(gpu):
    """Weights with main gradients beside biases with ordinary ones, in whatever containers."""
    import hpfp8
    linear = hpfp8.Fp8Linear(128, 256, device=gpu, apply_grad_on_fp32_main_grad=True)
    x = torch.randn((32, 128), device=gpu).to(torch.bfloat16)
    linear(x).float().square().sum().backward()
    grads = [linear.weight.main_grad.clone(), linear.bias.grad.clone()]
    want = norm64([t.cpu() for t in grads], 2.0)
    for given in (linear.parameters(), tuple(linear.parameters()), [linear.bias, linear.weight], {p: 0 for p in linear.parameters()}):
        near(hpfp8.clip_grad_norm_(given, 1e9), want)
    norm = hpfp8.clip_grad_norm_(linear.parameters(), 1.0)
    for got, t in zip((linear.weight.main_grad, linear.bias.grad), clipped([t.cpu() for t in grads], norm, 1.0)):
        assert torch.equal(got.cpu(), t)
    # the next backward adds onto what was clipped
    before = linear.weight.main_grad.clone()
    linear(x).float().square().sum().backward()
    assert (linear.weight.main_grad - before - grads[0]).abs().max() <= 1e-5 * grads[0].abs().max()


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("count", [1, 249, 250, 251, 500, 501])
def test_clipping_by_a_given_norm(gpu, count, native, monkeypatch):
    """Tables of 250 tensors, tensors without elements among them; the norm in every form in which it comes; a parameter named twice is clipped once."""
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    ts = tensors([(e * 37) % 300 for e in range(1, count + 1)], 2)
    norm = torch.tensor(7.0)
    expected = clipped(ts, norm, 2.0)
    for given in (norm.to(gpu), norm, norm.to(gpu, torch.bfloat16), norm.to(gpu).reshape(1), 7.0):
        ps = params([t.to(gpu) for t in ts])
        assert hpfp8.clip_grads_with_norm_(iter(ps + ps[:3]), 2.0, given) is None
        for q, t in zip(ps, expected):
            assert torch.equal((q.grad if q.grad is not None else q.main_grad).cpu(), t)
    near(hpfp8.get_total_norm([q.grad if q.grad is not None else q.main_grad for q in ps]), norm64(expected, 2.0))


@pytest.mark.parametrize("native", [True, False])
def test_traces_and_tangents_are_refused(gpu, native, monkeypatch):
    """A trace would keep an empty norm and no launch; a tangent would be dropped."""
    import hpfp8
    import torch.autograd.forward_ad as fwAD
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)

    def clip(f):
        def call(t):
            p = torch.nn.Parameter(torch.zeros(8, device=gpu))
            p.main_grad = t
            f(p)
            return t + 1
        return call
    two = torch.full((), 2.0, device=gpu)
    for name, f in (("get_total_norm", lambda t: hpfp8.get_total_norm([t])), ("clip_grads_with_norm_", clip(lambda p: hpfp8.clip_grads_with_norm_(p, 1.0, two))),
                    ("clip_grad_norm_", clip(lambda p: hpfp8.clip_grad_norm_(p, 1.0)))):
        g = torch.ones(8, device=gpu)
        with pytest.raises(RuntimeError, match=f"{name} has no place in a trace"):
            torch.jit.trace(f, (g,), check_trace=False)
        with fwAD.dual_level():
            with pytest.raises(RuntimeError, match=f"{name} .*forward mode"):
                f(fwAD.make_dual(g, torch.ones_like(g)))
            assert (g == 1).all()
            inside = f(g.clone())
        assert torch.equal(inside, f(g.clone()))


@pytest.fixture()
def mesh(gpu):
    """Two ranks of which this process is the first; nothing is ever sent."""
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.testing._internal.distributed.fake_pg import FakeStore
    dist.init_process_group("fake", store=FakeStore(), rank=0, world_size=2)
    try:
        yield init_device_mesh("cuda", (2,))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("kind", ["torch", "reference"])
def test_shards(gpu, mesh, kind):
    """The recipe for sharded gradients: the norm of the shards, that of the ranks' norms, and the parameters clipped by it, each gradient's own shard in
    place.  torch's tensors over a mesh, and those that hand every call to a dispatcher; main gradients that are shards too; local gradients among them."""
    import hpfp8
    from torch.distributed.tensor import DTensor, Shard
    import _hp_standin as S

    def sharded(local):
        if kind == "torch":
            return DTensor.from_local(local, mesh, [Shard(0)], run_check=False)
        return S.DTensor(local, S.Layout((2,), ("dp",))("dp", "None"))
    S.DTensor.DISPATCHER = S.Dispatcher()
    g = torch.Generator().manual_seed(3)
    locals_ = [torch.randn(n, 6, generator=g).to(d).to(gpu) for n, d in ((40, torch.float32), (7, torch.bfloat16), (1, torch.float32))]
    before = [t.cpu() for t in locals_]
    with torch._C.DisableTorchFunctionSubclass():
        grads = [sharded(t) for t in locals_[:2]] + [locals_[2]]
        if kind == "torch":
            a = torch.nn.Parameter(sharded(torch.zeros_like(locals_[0])))
        else:
            a = torch.nn.Parameter(torch.zeros_like(locals_[0]))
        a.grad = grads[0]
        b = torch.nn.Parameter(torch.zeros(3, device=gpu))
        b.main_grad = grads[1]
        c = torch.nn.Parameter(torch.zeros_like(locals_[2]))
        c.grad = grads[2]
    shards = [t.to_local() if hasattr(t, "to_local") else t for t in grads]
    n = hpfp8.get_total_norm(shards)
    near(n, norm64(before, 2.0))
    n = (2 * n.square()).sqrt()                              # (the other rank's shards have the same norm)
    for share in (2.0, 0.5):
        assert hpfp8.clip_grads_with_norm_([a, b, c], share * float(n), n) is None
        for t, w in zip(locals_, clipped(before, n, share * float(n))):
            assert torch.equal(t.cpu(), w)
    with pytest.raises((TypeError, RuntimeError), match="shard|parallel layout"):
        hpfp8.clip_grad_norm_([a, b, c], 1.0)
    with pytest.raises((TypeError, RuntimeError), match="shard|parallel layout"):
        hpfp8.get_total_norm(grads)
    assert all(torch.equal(t.cpu(), w) for t, w in zip(locals_, clipped(before, n, 0.5 * float(n))))


@pytest.mark.parametrize("native", [True, False])
def test_gradients_in_another_order_are_read_and_written_where_they_are(gpu, native, monkeypatch):
    """Transposed and channels_last gradients are memory without gaps: no copy of one is made, whether there is something to clip or not; with gaps
    between the elements, or elements that lie on one another, it is."""
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    g = torch.Generator().manual_seed(5)
    grads = [torch.randn((1024, 2050), generator=g).to(gpu).t(), torch.randn((16, 64, 33, 35), generator=g).half().to(gpu).to(memory_format=torch.channels_last),
             torch.randn((5, 7, 3, 1), generator=g).to(gpu).to(torch.bfloat16).permute(2, 3, 0, 1)]
    cpu = [t.cpu() for t in grads]
    ps = []
    for t in grads:
        p = torch.nn.Parameter(torch.zeros((1,), dtype=t.dtype, device=gpu).expand(t.shape))
        p.grad = t
        ps.append(p)
    at = [(t.data_ptr(), t.stride()) for t in grads]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    norm = hpfp8.get_total_norm(grads)
    held = hpfp8.clip_grad_norm_(ps, 1e9)
    hpfp8.clip_grads_with_norm_(ps, 2e9, norm)
    assert torch.cuda.max_memory_allocated() - before < 1 << 17          # (the smallest two copies would be 2 MiB)
    near(norm, norm64(cpu, 2.0))
    assert torch.equal(held, norm) and all(torch.equal(t.cpu(), c) for t, c in zip(grads, cpu))
    hpfp8.clip_grad_norm_(ps, 1.0)
    hpfp8.clip_grads_with_norm_(ps, 1.0, torch.tensor(2.0, device=gpu))
    assert torch.cuda.max_memory_allocated() - before < 1 << 17
    want = clipped(clipped(cpu, norm, 1.0), torch.tensor(2.0), 1.0)
    assert all(torch.equal(t.cpu(), w) for t, w in zip(grads, want)) and at == [(t.data_ptr(), t.stride()) for t in grads]
    # gaps, and one value for a whole row: the norm counts elements, not memory
    wide = torch.randn((64, 200), generator=g).to(gpu)
    around = wide.clone()
    apart = [wide.t()[3:90], wide[:, 100:101].expand(64, 9), wide[:, 120], torch.zeros((0, 4), device=gpu).t()]
    near(hpfp8.get_total_norm(apart), norm64([t.cpu() for t in apart], 2.0))
    q = torch.nn.Parameter(torch.zeros((1,), device=gpu).expand(87, 64))
    q.grad = apart[0]
    norm = hpfp8.clip_grad_norm_([q], 1.0)
    near(norm, norm64([around.t()[3:90].cpu()], 2.0))
    around.t()[3:90] = clipped([around.t()[3:90].cpu()], norm, 1.0)[0].to(gpu)
    assert torch.equal(wide, around)


@pytest.mark.parametrize("foreach", [None, True, False])
def test_foreach_changes_nothing(gpu, foreach):
    import hpfp8
    ts = [t.to(gpu) for t in tensors([1000, 70, 5], 2)]
    norm = hpfp8.get_total_norm(ts, foreach=foreach)
    near(norm, norm64([t.cpu() for t in ts], 2.0))
    one, other = params([t.clone() for t in ts]), params([t.clone() for t in ts])
    assert torch.equal(hpfp8.clip_grad_norm_(one, 1.0, 2.0, False, foreach), norm)
    hpfp8.clip_grads_with_norm_(other, 1.0, norm, foreach=foreach)
    for a, b, w in zip(one, other, clipped([t.cpu() for t in ts], norm, 1.0)):
        a, b = (q.grad if q.grad is not None else q.main_grad for q in (a, b))
        assert torch.equal(a.cpu(), w) and torch.equal(b.cpu(), w)
