"""Softmax cross entropy of a linear, without its logits, against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

IGNORE = -100
H = 2.0 ** -8        # half a step of bf16, relative
U = 2.0 ** -24


def make(tokens, hidden, vocab, seed, ignored=0.1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, hidden), generator=g).to(torch.bfloat16)
    w = (torch.randn((vocab, hidden), generator=g) * 2 / math.sqrt(hidden)).to(torch.bfloat16)
    t = torch.randint(vocab, (tokens,), generator=g)
    if tokens > 1:
        t = torch.where(torch.rand((tokens,), generator=g) < ignored, IGNORE, t)
        t[0] = vocab - 1
    return x, w, t


def reference(x, w, t, smoothing, coefficient):
    """(loss per row, dx, dw, bounds of the three) in 64 bits; coefficient [tokens]: each row's share of the loss's gradient.
    A logit is a chain of hidden / 32 accumulations of 32 products each, at most a step of fp32 lost in each: `off`."""
    x, w = x.double(), w.double()
    vocab, hidden = w.shape
    l = x @ w.t()
    off = (hidden / 32 + 32) * 2 * U * (x.abs() @ w.abs().t()).amax(1)
    lse = torch.logsumexp(l, 1)
    counted = t != IGNORE
    at = torch.where(counted, t, 0)
    rows = lse - (1 - smoothing) * l.gather(1, at[:, None])[:, 0] - smoothing * l.mean(1)
    rows = torch.where(counted, rows, 0.0)
    # the logits' error reaches lse and the target's logit; 64 roundings of sums of exponentials (relative: absolute in lse); a few of the result's
    b_rows = 2 * off + 64 * U + 8 * U * (lse.abs() + l.abs().amax(1)) + (vocab / 256 + 64) * U * smoothing * l.abs().mean(1)
    p = torch.exp(l - lse[:, None])
    c = torch.where(counted, coefficient.double(), 0.0)[:, None]
    dl = p - smoothing / vocab
    dl.scatter_add_(1, at[:, None], torch.full_like(dl, -(1 - smoothing))[:, :1])
    size = (p + smoothing / vocab)
    size.scatter_add_(1, at[:, None], torch.full_like(dl, 1 - smoothing)[:, :1])
    # dl: rounded to bf16; its probability is off by the logits' and lse's errors, relative
    b_dl = H * dl.abs() + size * (4 * off[:, None] + 64 * U + 4 * U * l.abs().amax())
    dl, b_dl = c * dl, c.abs() * b_dl * 1.01
    dx, dw = dl @ w, dl.t() @ x
    b_dx = b_dl @ w.abs() + (vocab / 32 + 64) * 2 * U * (dl.abs() @ w.abs())
    b_dw = b_dl.t() @ x.abs() + (x.shape[0] / 32 + 64) * 2 * U * (dl.abs().t() @ x.abs())
    return rows, dx, dw, b_rows, b_dx, b_dw


def within(got, want, bound, half=0.0):
    off = (got.double().cpu() - want).abs()
    limit = half * want.abs() + bound
    assert (off <= limit).all(), float((off - limit).max())


SIZES = [(1, 8, 1), (1, 64, 256), (2, 8, 300), (5, 128, 1000), (64, 72, 257), (255, 256, 511), (256, 512, 512), (300, 200, 1111), (513, 320, 2049)]


@pytest.mark.parametrize("tokens,hidden,vocab", SIZES)
@pytest.mark.parametrize("reduction,smoothing", [("mean", 0.0), ("sum", 0.1), ("none", 0.0), ("none", 0.3)])
def test_loss_and_gradients(gpu, tokens, hidden, vocab, reduction, smoothing):
    import hpfp8
    x, w, t = make(tokens, hidden, vocab, 1)
    xg, wg = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
    loss = hpfp8.linear_cross_entropy(xg, wg, t.to(gpu), reduction=reduction, label_smoothing=smoothing)
    assert loss.dtype == torch.float32
    counted = t != IGNORE
    go = torch.randn((tokens,), generator=torch.Generator().manual_seed(2)) if reduction == "none" else torch.tensor(0.7)
    coefficient = go if reduction == "none" else (go / counted.sum() if reduction == "mean" else go).expand(tokens)
    dx, dw = torch.autograd.grad(loss, (xg, wg), go.to(gpu))
    rows, rdx, rdw, b_rows, b_dx, b_dw = reference(x, w, t, smoothing, coefficient)
    if reduction == "none":
        within(loss.detach(), rows, b_rows)
        assert (loss.detach().cpu()[~counted] == 0).all()
    else:
        n = counted.sum() if reduction == "mean" else 1
        within(loss.detach(), rows.sum() / n, (b_rows * counted).sum() / n + U * (rows.sum() / n).abs())
    within(dx, rdx, b_dx, H)
    within(dw, rdw, b_dw, H)
    assert (dx.cpu()[~counted] == 0).all()
    with torch.no_grad():
        assert torch.equal(hpfp8.linear_cross_entropy(xg, wg, t.to(gpu), reduction=reduction, label_smoothing=smoothing), loss)


@pytest.mark.parametrize("budget", [1 << 20, 1 << 16])
def test_pieces_of_the_vocabulary(gpu, budget, monkeypatch):
    """Several pieces, a last one that is no whole tile: the weight's gradient has the bits of one piece, x's is summed in fp32."""
    import hpfp8
    from hpfp8 import loss as module
    x, w, t = make(130, 256, 2000, 3)
    assert len(module._pieces(130, 256, 2000, budget)) > 1
    both = []
    for b in (1 << 30, budget):
        monkeypatch.setattr(module, "_PIECE_BYTES", b)
        xg, wg = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
        both.append(torch.autograd.grad(hpfp8.linear_cross_entropy(xg, wg, t.to(gpu)), (xg, wg)))
    _, rdx, _, _, b_dx, _ = reference(x, w, t, 0.0, torch.full((130,), 1.0) / (t != IGNORE).sum())
    within(both[1][0], rdx, b_dx, H)
    assert torch.equal(both[0][1], both[1][1])


def test_pieces_cover_the_vocabulary_once():
    from hpfp8.loss import _pieces
    for tokens, hidden, vocab, budget in ((1, 8, 1, 1), (4096, 7168, 131072, 512 << 20), (1 << 22, 8, 1 << 24, 512 << 20), (300, 64, 50001, 1 << 20)):
        pieces = _pieces(tokens, hidden, vocab, budget)
        assert pieces[0][0] == 0 and sum(n for _, n in pieces) == vocab
        assert all(a + n == b for (a, n), (b, _) in zip(pieces, pieces[1:])) and all(n % 256 == 0 for _, n in pieces[:-1])


def test_tokens_in_several_forwards(gpu, monkeypatch):
    import hpfp8
    from hpfp8 import loss as module
    x, w, t = (v.to(gpu) for v in make(600, 64, 500, 4))
    want = [hpfp8.linear_cross_entropy(x, w, t, reduction=r, label_smoothing=0.1) for r in ("none", "mean", "sum")]
    monkeypatch.setattr(module, "_FORWARD_ROWS", 256)
    got = [hpfp8.linear_cross_entropy(x, w, t, reduction=r, label_smoothing=0.1) for r in ("none", "mean", "sum")]
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_rows_that_are_ignored_may_hold_anything(gpu):
    import hpfp8
    x, w, t = make(100, 128, 700, 5, 0.3)
    grads = []
    for junk in (0.0, math.nan, math.inf):
        y = x.clone()
        y[t == IGNORE] = junk
        xg, wg = y.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
        loss = hpfp8.linear_cross_entropy(xg, wg, t.to(gpu))
        grads.append((loss.detach(),) + torch.autograd.grad(loss, (xg, wg)))
    for other in grads[1:]:
        assert all(torch.equal(p, q) for p, q in zip(grads[0], other))


def test_all_rows_ignored_and_no_rows(gpu):
    import hpfp8
    x, w, t = make(20, 64, 100, 6)
    for n in (20, 0):
        xg, wg = x[:n].to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
        tg = torch.full((n,), IGNORE, device=gpu)
        assert hpfp8.linear_cross_entropy(xg, wg, tg).isnan()
        loss = hpfp8.linear_cross_entropy(xg, wg, tg, reduction="sum")
        dx, dw = torch.autograd.grad(loss, (xg, wg))
        assert loss == 0 and dx.shape == (n, 64) and (dx == 0).all() and (dw == 0).all()
        assert hpfp8.linear_cross_entropy(xg, wg, tg, reduction="none").shape == (n,)


def test_targets_out_of_range_and_logits_that_are_not_finite(gpu):
    import hpfp8
    x, w, t = make(40, 64, 300, 7, 0.0)
    t[3], t[4] = 300, -5
    x[7, 0] = math.nan
    xg = x.to(gpu).requires_grad_()
    loss = hpfp8.linear_cross_entropy(xg, w.to(gpu), t.to(gpu), reduction="none")
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[3, 4, 7]] = True
    assert torch.equal(loss.isnan().cpu(), bad)
    dx, = torch.autograd.grad(loss.sum(), xg)
    assert torch.equal(dx.isnan().any(1).cpu(), bad)
    # another value that is ignored
    t[3], t[4] = 7, 7
    loss = hpfp8.linear_cross_entropy(x.to(gpu), w.to(gpu), t.to(gpu), reduction="none", ignore_index=7)
    assert (loss.cpu()[t == 7] == 0).all()


def test_large_logits(gpu):
    """Logits of +-500: the largest is subtracted before the exponential."""
    import hpfp8
    x, w, t = make(50, 64, 400, 8)
    x = x * 60
    loss = hpfp8.linear_cross_entropy(x.to(gpu), w.to(gpu), t.to(gpu), reduction="none")
    rows, _, _, b_rows, _, _ = reference(x, w, t, 0.0, torch.ones(50))
    within(loss, rows, b_rows)


def test_shapes_strides_and_starts_between_vectors(gpu):
    import hpfp8
    g = torch.Generator().manual_seed(9)
    base = torch.randn((6, 50, 80), generator=g).to(torch.bfloat16).to(gpu)
    weight = torch.randn((333, 96), generator=g).to(torch.bfloat16).to(gpu)
    t = torch.randint(333, (6, 50), generator=g).to(gpu)
    for x, w in ((base[:, :, :64], weight[:, :64]), (base[:, :, 3:67], weight[:, 1:65]), (base[::2, 5:20, 16:], weight[:, 32:]),
                 (base.transpose(0, 1)[:, :, 8:72], weight[:, 8:72])):
        tt = t.reshape(-1)[:x.shape[0] * x.shape[1]].reshape(x.shape[:2])
        a = [v.detach().requires_grad_() for v in (x, w)]
        b = [v.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for v in (x, w)]
        got, want = hpfp8.linear_cross_entropy(*a, tt, reduction="none"), hpfp8.linear_cross_entropy(*b, tt, reduction="none")
        assert got.shape == tt.shape and torch.equal(got, want)
        for p, q in zip(torch.autograd.grad(got.sum(), a), torch.autograd.grad(want.sum(), b)):
            assert torch.equal(p, q)


def test_gradient_of_one_alone_and_main_grad(gpu):
    import hpfp8
    x, w, t = (v.to(gpu) for v in make(70, 64, 900, 10))
    leaves = [v.clone().requires_grad_() for v in (x, w)]
    dx, dw = torch.autograd.grad(hpfp8.linear_cross_entropy(*leaves, t), leaves)
    for k in range(2):
        some = [v.clone().requires_grad_(i == k) for i, v in enumerate((x, w))]
        assert torch.equal(torch.autograd.grad(hpfp8.linear_cross_entropy(*some, t), some[k])[0], (dx, dw)[k])
    p = torch.nn.Parameter(w.clone())
    xg = x.clone().requires_grad_()
    for step in (1, 2):
        hpfp8.linear_cross_entropy(xg, p, t, apply_grad_on_fp32_main_grad=True).backward()
        assert p.grad is None and p.main_grad.dtype == torch.float32
        if step == 1:
            once = p.main_grad.clone()
            assert torch.equal(once.to(torch.bfloat16), dw)
    assert ((p.main_grad - 2 * once).abs() <= 4 * U * once.abs()).all()


def test_gradient_against_differences(gpu):
    import hpfp8
    x, w, t = make(3, 16, 50, 11, 0.0)
    xg = x.to(gpu).requires_grad_()
    dx, = torch.autograd.grad(hpfp8.linear_cross_entropy(xg, w.to(gpu), t.to(gpu), reduction="sum"), xg)
    with torch.no_grad():
        for c in range(16):
            up, down = x.clone(), x.clone()
            up[:, c] += 0.0625
            down[:, c] -= 0.0625
            step = (up[:, c].double() - down[:, c].double())
            d = (hpfp8.linear_cross_entropy(up.to(gpu), w.to(gpu), t.to(gpu), reduction="none")
                 - hpfp8.linear_cross_entropy(down.to(gpu), w.to(gpu), t.to(gpu), reduction="none")).double().cpu() / step
            # the loss's third derivative along c is below 8 (a moment of weights below 2); bf16 rounds dl's 50 summands
            limit = 8 / 6 * 0.0625 ** 2 * 1.2 + 2.0 ** -7 * 2 * float(w.abs().max()) + 1e-4 + (step - 0.125).abs() * 8
            assert ((d - dx.double().cpu()[:, c]).abs() <= limit).all()


@pytest.mark.parametrize("reduction,smoothing", [("mean", 0.1), ("none", 0.0)])
def test_the_python_form_and_other_ways_through_the_graph(gpu, reduction, smoothing, monkeypatch):
    """Without the native host path, under a dispatch mode and with hooks on saved tensors, in one piece and in several: the same results."""
    import hpfp8
    from hpfp8 import loss as module, ops
    from torch.utils._python_dispatch import TorchDispatchMode

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x, w, t = (v.to(gpu) for v in make(90, 64, 1500, 12))
    x, t = x.reshape(3, 30, 64), t.reshape(3, 30)
    go = torch.rand(t.shape if reduction == "none" else (), device=gpu)

    def step(hooks=None, mode=None):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        with hooks or torch.enable_grad():
            loss = hpfp8.linear_cross_entropy(a, b, t, reduction=reduction, label_smoothing=smoothing)
        with mode or torch.enable_grad():
            return (loss.detach(),) + torch.autograd.grad(loss, (a, b), go)
    for budget in (1 << 30, 1 << 19):
        monkeypatch.setattr(module, "_PIECE_BYTES", budget)
        want = step()
        hooks = torch.autograd.graph.saved_tensors_hooks(lambda v: v.cpu(), lambda v: v.to(gpu))
        strided = torch.autograd.graph.saved_tensors_hooks(lambda v: v, lambda v: torch.stack((v, v), -1)[..., 0])
        for got in (step(hooks), step(strided), step(None, Mode()), step(Mode())):
            assert all(torch.equal(p, q) for p, q in zip(got, want))
        with monkeypatch.context() as m:
            m.setattr(ops, "_native", None)
            assert all(torch.equal(p, q) for p, q in zip(step(), want))


@pytest.mark.parametrize("main_grad", [False, True])
def test_the_mean_over_no_rows_is_nan_and_its_gradients_are_zero(gpu, main_grad):
    """A micro-batch of padding alone, as in torch."""
    import hpfp8
    x, w, _ = make(20, 64, 300, 8)
    xg, wg = x.to(gpu).requires_grad_(), torch.nn.Parameter(w.to(gpu))
    loss = hpfp8.linear_cross_entropy(xg, wg, torch.full((20,), IGNORE, device=gpu), apply_grad_on_fp32_main_grad=main_grad)
    loss.backward()
    dw = wg.main_grad if main_grad else wg.grad
    assert loss.isnan() and (xg.grad == 0).all() and dw.shape == w.shape and (dw == 0).all()


@pytest.mark.parametrize("tokens,hidden,vocab", [(2100, 1024, 20000), (1100, 520, 33000)])
def test_several_rounds_of_the_largest_tiles(gpu, tokens, hidden, vocab):
    """More tiles of 256 rows than compute units, the last of each side cut; the reference on the GPU, in 64 bits too."""
    import hpfp8
    x, w, t = (v.to(gpu) for v in make(tokens, hidden, vocab, 9))
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = hpfp8.linear_cross_entropy(xg, wg, t, label_smoothing=0.1)
    dx, dw = torch.autograd.grad(loss, (xg, wg))
    n = int((t != IGNORE).sum())
    rows, rdx, rdw, b_rows, b_dx, b_dw = (v.cpu() for v in reference(x, w, t, 0.1, torch.full((tokens,), 1.0 / n, device=gpu, dtype=torch.float64)))
    within(loss.detach(), rows.sum() / n, (b_rows * (t != IGNORE).cpu()).sum() / n + U * (rows.sum() / n).abs())
    within(dx, rdx, b_dx, H)
    within(dw, rdw, b_dw, H)


def test_as_many_tokens_as_a_call_takes(gpu):
    """2^21 rows: workspaces whose rows have a column for each of them."""
    import hpfp8
    tokens, hidden, vocab = 1 << 21, 8, 300
    g = torch.Generator(device=gpu).manual_seed(10)
    x = torch.randn((tokens, hidden), generator=g, device=gpu).to(torch.bfloat16)
    w = torch.randn((vocab, hidden), generator=g, device=gpu).to(torch.bfloat16)
    t = torch.randint(vocab, (tokens,), generator=g, device=gpu)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = hpfp8.linear_cross_entropy(xg, wg, t, reduction="none")
    go = torch.randn((tokens,), generator=g, device=gpu)
    dx, dw = torch.autograd.grad(loss, (xg, wg), go)
    rdw, b_dw = torch.zeros((vocab, hidden), dtype=torch.float64), torch.zeros((vocab, hidden), dtype=torch.float64)
    for at in range(0, tokens, 1 << 18):
        part = slice(at, at + (1 << 18))
        rows, rdx, dw_part, b_rows, b_dx, b_part = (v.cpu() for v in reference(x[part], w, t[part], 0.0, go[part]))
        within(loss[part].detach(), rows, b_rows)
        within(dx[part], rdx, b_dx, H)
        rdw += dw_part
        b_dw += b_part * 8            # (the sum's roundings are bounded by the number of all tokens, here by that of a part's)
    within(dw, rdw, b_dw, H)
    with pytest.raises(ValueError, match="2\\^21 tokens"):
        hpfp8.linear_cross_entropy(x.new_zeros(tokens + 1, hidden), w, t.new_zeros(tokens + 1))


def test_a_weight_of_more_than_2_31_values(gpu):
    import hpfp8
    tokens, hidden, vocab = 70, 8192, 270000
    g = torch.Generator(device=gpu).manual_seed(11)
    x = torch.randn((tokens, hidden), generator=g, device=gpu).to(torch.bfloat16)
    w = torch.empty((vocab, hidden), dtype=torch.bfloat16, device=gpu).normal_(0.0, 0.02, generator=g)
    t = torch.randint(vocab, (tokens,), generator=g, device=gpu)
    t[0] = vocab - 1
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = hpfp8.linear_cross_entropy(xg, wg, t, reduction="none")
    dx, dw = torch.autograd.grad(loss.sum(), (xg, wg))
    x64 = x.double()
    l = torch.cat([x64 @ w[a:a + 30000].double().t() for a in range(0, vocab, 30000)], 1)
    size = max(float((x64.abs() @ w[a:a + 30000].double().abs().t()).max()) for a in range(0, vocab, 30000))
    off = (hidden / 32 + 32) * 2 * U * size             # a logit's error, as in `reference`
    lse = torch.logsumexp(l, 1)
    at = torch.arange(tokens, device=gpu)
    within(loss.detach(), (lse - l[at, t]).cpu(), 2 * off + 64 * U + 8 * U * (lse.abs() + l.abs().amax(1)).cpu())
    p = torch.exp(l - lse[:, None])
    p[at, t] -= 1
    b_p = H * p.abs() + (p.abs() + 2 * (torch.arange(vocab, device=gpu) == t[:, None])) * (4 * off + 64 * U + 4 * U * l.abs().amax())
    for rows in (slice(0, 600), slice(vocab - 9000, vocab)):
        want, bound = p[:, rows].t() @ x64, (b_p[:, rows].t() @ x64.abs()) * 1.01 + (tokens / 32 + 64) * 2 * U * (p[:, rows].abs().t() @ x64.abs())
        within(dw[rows], want.cpu(), bound.cpu(), H)
    want, bound = torch.zeros_like(x64), torch.zeros_like(x64)
    for a in range(0, vocab, 30000):
        part = w[a:a + 30000].double()
        want += p[:, a:a + 30000] @ part
        bound += b_p[:, a:a + 30000] @ part.abs() * 1.01 + (vocab / 32 + 64) * 2 * U * (p[:, a:a + 30000].abs() @ part.abs())
    within(dx, want.cpu(), bound.cpu(), H)


@pytest.mark.parametrize("tokens,hidden,vocab", [(300, 520, 10000), (1000, 1024, 8010), (24, 1472, 33651), (100, 1032, 15900), (16, 1000, 2859), (200, 328, 3000)])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_every_shape_of_tiles(gpu, tokens, hidden, vocab, smoothing):
    """128 x 128, 128 x 256, 64 x 256, 64 x 128 and, the last two, 64 x 64; the largest are above.  Each row's loss, and both gradients."""
    import hpfp8
    from hpfp8 import _lib
    cols = -(-vocab // _lib.load().hpfp8_cross_entropy_parts(tokens, hidden, vocab))
    assert (cols <= 64) == (vocab < 8000)
    x, w, t = (v.to(gpu) for v in make(tokens, hidden, vocab, 12))
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = hpfp8.linear_cross_entropy(xg, wg, t, label_smoothing=smoothing, reduction="none")
    go = torch.randn((tokens,), generator=torch.Generator().manual_seed(13)).to(gpu)
    dx, dw = torch.autograd.grad(loss, (xg, wg), go)
    rows, rdx, rdw, b_rows, b_dx, b_dw = (v.cpu() for v in reference(x, w, t, smoothing, go))
    within(loss.detach(), rows, b_rows)
    within(dx, rdx, b_dx, H)
    within(dw, rdw, b_dw, H)


def test_the_last_tokens_may_take_other_tiles(gpu, monkeypatch):
    """A forward in several launches, whose last one writes more parts for fewer rows."""
    import hpfp8
    from hpfp8 import _lib
    from hpfp8 import loss as module
    parts = _lib.load().hpfp8_cross_entropy_parts
    assert parts(512, 512, 8000) < parts(68, 512, 8000)
    x, w, t = (v.to(gpu) for v in make(580, 512, 8000, 14))
    want = hpfp8.linear_cross_entropy(x, w, t, reduction="none", label_smoothing=0.1).cpu().double()
    monkeypatch.setattr(module, "_FORWARD_ROWS", 512)
    hook = []
    monkeypatch.setattr(module.ops, "_gpu", lambda x: hook.append(x) or False)        # (the Python form, which is the one that takes several)
    got = hpfp8.linear_cross_entropy(x, w, t, reduction="none", label_smoothing=0.1)
    rows, b_rows = (v.cpu() for v in (lambda r: (r[0], r[3]))(reference(x, w, t, 0.1, torch.ones(580, device=gpu))))
    assert hook
    within(got, rows, b_rows)
    within(want, rows, b_rows)


@pytest.mark.parametrize("at", [1, 3, 4])
@pytest.mark.parametrize("tokens", [1, 70])
def test_contiguous_tensors_that_start_between_two_vectors(gpu, at, tokens):
    """Views in a flat buffer: input and weight, and what hooks on saved tensors hand back."""
    import hpfp8
    x, w, t = (v.to(gpu) for v in make(tokens, 64, 300, 15))

    def view(v):
        out = torch.empty(v.numel() + at, dtype=v.dtype, device=gpu)[at:].view(v.shape).copy_(v)
        assert out.is_contiguous() and out.data_ptr() % 16
        return out

    def step(x, w, hooks=None):
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        with hooks or torch.enable_grad():
            loss = hpfp8.linear_cross_entropy(a, b, t)
        return (loss.detach(),) + torch.autograd.grad(loss, (a, b))
    want = step(x, w)
    hooks = torch.autograd.graph.saved_tensors_hooks(lambda v: v, lambda v: view(v) if v.dtype == torch.bfloat16 else v)
    for got in (step(view(x), w), step(x, view(w)), step(view(x), view(w)), step(x, w, hooks)):
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("shape", [(300,), (3, 100), (1, 1)])
def test_a_gradient_that_all_rows_share_is_one_factor(gpu, shape, native, monkeypatch):
    """Losses one by one, summed or averaged by torch: the gradients are those of the sum with that factor, bit for bit, and the logits'
    gradient is not rounded with the factor in it."""
    import hpfp8
    from hpfp8 import ops
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    tokens = math.prod(shape)
    x, w, t = (v.to(gpu) for v in make(tokens, 256, 1100, 16))
    x, t = x.reshape(shape + (256,)), t.reshape(shape)

    def gradients(reduction, after, go):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = after(hpfp8.linear_cross_entropy(a, b, t, reduction=reduction))
        return torch.autograd.grad(loss, (a, b), go)
    go = torch.tensor(0.7, device=gpu)
    want = gradients("sum", lambda v: v, go)
    for got in (gradients("none", lambda v: v.sum(), go), gradients("none", lambda v: v, go.expand(shape))):
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    # one value for each row is another matter, also where the values agree
    rows = gradients("none", lambda v: v, go.expand(shape).clone())
    _, rdx, rdw, _, b_dx, b_dw = reference(x.reshape(tokens, 256).cpu(), w.cpu(), t.reshape(-1).cpu(), 0.0, go.cpu().expand(tokens))
    for dx, dw in (want, rows):
        within(dx.reshape(tokens, 256), rdx, b_dx, H)
        within(dw, rdw, b_dw, H)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("tokens,rows,smoothing", [(600, 256, 0.1), (513, 256, 0.0), (257, 256, 0.1), (256, 256, 0.0)])
def test_a_forward_in_several_launches_and_its_backward(gpu, tokens, rows, smoothing, reduction, monkeypatch):
    """A last launch of one row, one whose rows are all ignored: the losses are reduced once, over all of them."""
    import hpfp8
    from hpfp8 import _lib
    from hpfp8 import loss as module
    x, w, t = make(tokens, 64, 500, 17)
    t[256:512] = IGNORE
    if tokens == 513:
        t[512] = 3
    names, call = [], _lib.call
    monkeypatch.setattr(_lib, "call", lambda name, *args: names.append(name) or call(name, *args))
    monkeypatch.setattr(module, "_FORWARD_ROWS", rows)
    xg, wg = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
    loss = hpfp8.linear_cross_entropy(xg, wg, t.to(gpu), reduction=reduction, label_smoothing=smoothing)
    launches = -(-tokens // rows)
    if launches > 1:
        assert names.count("hpfp8_linear_cross_entropy_forward") == launches
        assert names.count("hpfp8_linear_cross_entropy_reduce") == (reduction != "none")
    counted = t != IGNORE
    n = counted.sum() if reduction == "mean" else 1
    go = torch.randn((tokens,), generator=torch.Generator().manual_seed(18)) if reduction == "none" else torch.tensor(0.7)
    dx, dw = torch.autograd.grad(loss, (xg, wg), go.to(gpu))
    each, rdx, rdw, b_rows, b_dx, b_dw = reference(x, w, t, smoothing, (go / n).expand(tokens))
    if reduction == "none":
        within(loss.detach(), each, b_rows)
    else:
        within(loss.detach(), each.sum() / n, (b_rows * counted).sum() / n + U * (each.sum() / n).abs())
    within(dx, rdx, b_dx, H)
    within(dw, rdw, b_dw, H)
    with torch.no_grad():
        assert torch.equal(hpfp8.linear_cross_entropy(xg, wg, t.to(gpu), reduction=reduction, label_smoothing=smoothing), loss)


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_more_tokens_than_a_forward_takes(gpu, reduction):
    import hpfp8
    from hpfp8 import loss as module
    tokens = module._FORWARD_ROWS + 3001
    x, w, t = (v.to(gpu) for v in make(tokens, 64, 300, 19))
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = hpfp8.linear_cross_entropy(xg, wg, t, reduction=reduction, label_smoothing=0.1)
    dx, dw = torch.autograd.grad(loss, (xg, wg))
    counted = t != IGNORE
    n = counted.sum() if reduction == "mean" else torch.ones((), device=gpu)
    each, rdx, rdw, b_rows, b_dx, b_dw = reference(x, w, t, 0.1, (1 / n.double()).expand(tokens))
    within(loss.detach(), (each.sum() / n).cpu(), ((b_rows * counted).sum() / n + U * (each.sum() / n).abs()).cpu())
    within(dx, rdx.cpu(), b_dx.cpu(), H)
    within(dw, rdw.cpu(), b_dw.cpu(), H)


def test_both_host_paths_cut_the_vocabulary_alike(gpu, monkeypatch):
    """By bytes and by elements: the pieces' bits in dx, which is summed over them, are those of the same pieces."""
    import hpfp8
    from hpfp8 import loss as module, ops
    x, w, t = (v.to(gpu) for v in make(90, 64, 3000, 20))

    def step():
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        return torch.autograd.grad(hpfp8.linear_cross_entropy(a, b, t), (a, b))
    whole = step()
    for name, value, pieces in (("_PIECE_BYTES", 4 * 256 * 1024, 3), ("_PIECE_ELEMENTS", 512 * 64 + 1, 6)):
        with monkeypatch.context() as m:
            m.setattr(module, name, value)
            assert len(module._pieces(90, 64, 3000, module._PIECE_BYTES)) == pieces
            native = step()
            m.setattr(ops, "_native", None)
            python = step()
        assert all(torch.equal(p, q) for p, q in zip(native, python)) and torch.equal(native[1], whole[1])
        assert not torch.equal(native[0], whole[0])


@pytest.mark.parametrize("dtype,add", [(torch.bfloat16, 0), (torch.float32, 0), (torch.float32, 1)])
def test_a_piece_of_no_tokens(gpu, dtype, add):
    """Through the C entry: its rows of the weight's gradient are zeros, or as they were if they are added onto, all others untouched."""
    from hpfp8 import _lib, ops
    dw = torch.full((2500, 72), 3.0, dtype=dtype, device=gpu)
    _lib.call("hpfp8_linear_cross_entropy_piece", None, 72, None, None, 72, None, 0, 72, 2500, 256, 2000, -100, 0.0, None, None, 0, None, None, None, None, 1, 0,
              ops._ptr(dw), _lib.OUT_F32 if dtype == torch.float32 else _lib.OUT_BF16, add, ops._stream())
    assert (dw[:256] == 3).all() and (dw[2256:] == 3).all() and (dw[256:2256] == (3 if add else 0)).all()
