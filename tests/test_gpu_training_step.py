"""The operators of a training step together: norm, FP8 linears, activations in 8 bits, the loss over the vocabulary."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def randn(shape, seed, std=1.0, device="cuda"):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(torch.bfloat16).to(device)


@pytest.mark.parametrize("tokens", [128, 77])
@pytest.mark.parametrize("trained", ["both", "down"])
def test_mlp_block_with_its_gate_up_output_in_8_bits(gpu, tokens, trained):
    """The result is that of the block as it was; the gradients are those of the steps one by one, SwiGLU's taken at the codes' values."""
    import hpfp8
    from hpfp8 import ops
    x, wgu, wd, go = randn((tokens, 256), 1), randn((512, 256), 2, 0.1), randn((384, 256), 3, 0.1), randn((tokens, 384), 4)

    def step(keep):
        leaves = [t.clone().requires_grad_(i != 1 or trained == "both") for i, t in enumerate((x, wgu, wd))]
        y = hpfp8.fp8_swiglu_mlp(*leaves, keep_8bit=keep)
        return (y.detach(),) + torch.autograd.grad(y, [t for t in leaves if t.requires_grad], go)
    plain, kept = step(False), step(True)
    assert torch.equal(plain[0], kept[0]) and torch.equal(plain[-1], kept[-1])          # (w_down's gradient does not see h)
    h = hpfp8.fp8_linear(x, wgu)
    h8 = hpfp8.quantize_activation(h).dequantize()
    gq, sg = ops.quantize_1x128(go, kmajor=True)
    wq, sw, wt = ops.quantize_128x128(wd, with_transpose=True)
    dh = ops.swiglu_backward(h8, ops.gemm_blockwise(gq, sg, wt, sw.t()))
    a, b = x.clone().requires_grad_(), wgu.clone().requires_grad_()
    dx, dw = torch.autograd.grad(hpfp8.fp8_linear(a, b), (a, b), dh)
    if trained == "both":
        assert torch.equal(kept[1], dx) and torch.equal(kept[2], dw)
    else:
        assert torch.equal(kept[1], dx)


def test_mlp_module_keeps_its_largest_activation_in_half_the_memory(gpu):
    import hpfp8
    x = randn((1024, 512), 5).requires_grad_()

    def held(keep):
        mlp = hpfp8.Fp8SwiGLUMLP(512, 2048, keep_8bit=keep, device="cuda")
        mlp(x).sum()                                    # (what the first call of all allocates for good is there)
        requested = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]     # noqa: E731
        before = requested()
        y = mlp(x)
        return requested() - before, y
    h = 1024 * 4096
    assert held(False)[0] - held(True)[0] == h * 2 - (h + h // 128 * 4)


class Block(torch.nn.Module):
    def __init__(self, hidden, inter, keep, fp8):
        super().__init__()
        import hpfp8
        self.fp8, self.keep = fp8, keep
        self.norm = hpfp8.LayerNorm(hidden, keep_8bit=keep, device="cuda") if fp8 else torch.nn.LayerNorm(hidden, device="cuda")
        self.up, self.down = (hpfp8.Fp8Linear(*s, device="cuda") if fp8 else torch.nn.Linear(*s, device="cuda")
                              for s in ((hidden, inter), (inter // 2, hidden)))

    def forward(self, x):
        import hpfp8
        h = self.up(self.norm(x))
        if self.fp8:
            return x + self.down(hpfp8.activation(h, "swiglu", keep_8bit=self.keep))
        gate, up = h.chunk(2, -1)
        return x + self.down(torch.nn.functional.silu(gate) * up)


def model(fp8, keep=False, blocks=2):
    torch.manual_seed(0)
    layers = torch.nn.ModuleList(Block(256, 512, keep, fp8) for _ in range(blocks))
    head = torch.nn.Parameter(randn((1000, 256), 7, 0.05).to(torch.bfloat16 if fp8 else torch.float32))
    return layers, head


def run(layers, head, x, target, fp8):
    import hpfp8
    for layer in layers:
        x = layer(x)
    if fp8:
        return hpfp8.linear_cross_entropy(x, head, target)
    return torch.nn.functional.cross_entropy(torch.nn.functional.linear(x, head).flatten(0, 1), target.flatten())


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("hooks", [False, True])
def test_a_step_of_a_small_model_against_torch_in_fp32(gpu, keep, hooks):
    """Each weight's and the input's gradient within what E4M3 costs: an operand's rounding is 2^-4 at most and 2^-4 / sqrt(3) = 0.036 in the
    square mean, and a gradient passes through up to three quantized operands of each of up to four linears and four kept tensors."""
    import hpfp8
    x, target = randn((3, 50, 256), 8), torch.randint(1000, (3, 50), generator=torch.Generator().manual_seed(9)).cuda()
    target[0, :7] = -100
    layers, head = model(True, keep)
    reference, rhead = model(False)
    reference.load_state_dict({k: v.float() for k, v in layers.state_dict().items()})
    xg, xr = x.clone().requires_grad_(), x.float().requires_grad_()
    if hooks:
        with hpfp8.keep_activations_8bit(min_elements=1 << 12):
            loss = run(layers, head, xg, target, True)
    else:
        loss = run(layers, head, xg, target, True)
    loss.backward()
    want = run(reference, rhead, xr, target, False)
    want.backward()
    assert abs(float(loss) - float(want)) < 0.036 * float(want)
    pairs = [(xg.grad, xr.grad), (head.grad, rhead.grad)] + [(a.grad, b.grad) for a, b in zip(layers.parameters(), reference.parameters())]
    limit = 0.036 * math.sqrt(3 * 4 + 4)
    for got, ref in pairs:
        assert got.shape == ref.shape and float((got.float() - ref).norm()) < limit * float(ref.norm())


def test_a_step_in_a_graph_has_the_eager_results_on_every_replay(gpu):
    """Forward and backward captured together; replayed with other inputs and eager work in between."""
    import hpfp8
    layers, head = model(True, keep=True)
    params = [head] + list(layers.parameters())
    batches = [(randn((2, 64, 256), 20 + i), torch.randint(1000, (2, 64), generator=torch.Generator().manual_seed(30 + i)).cuda()) for i in range(4)]

    def step(x, target):
        x = x.detach().requires_grad_()
        loss = run(layers, head, x, target, True)
        return (loss.detach(),) + torch.autograd.grad(loss, [x] + params)
    x, target = batches[0][0].clone(), batches[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, target)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = step(x, target)
    for a, b in batches + batches[:2]:
        want = [t.clone() for t in step(a, b)]
        x.copy_(a)
        target.copy_(b)
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(outputs, want))
        torch.cuda.synchronize()


def test_operators_on_another_stream_and_two_at_once(gpu):
    """Workspaces belong to a call: steps on two streams side by side have the results of steps one after the other."""
    import hpfp8
    w = randn((1500, 256), 40, 0.05)
    nw = randn((256,), 41)
    inputs = [(randn((300, 256), 42 + i), torch.randint(1500, (300,), generator=torch.Generator().manual_seed(i)).cuda()) for i in range(2)]

    def step(x, t):
        a, b, c = x.clone().requires_grad_(), w.clone().requires_grad_(), nw.clone().requires_grad_()
        y = hpfp8.activation(hpfp8.layer_norm(a, 256, c, keep_8bit=True), "gelu")
        return torch.autograd.grad(hpfp8.linear_cross_entropy(y, b, t), (a, b, c))
    want = [step(*i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    for _ in range(3):
        got = []
        for s, i in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(step(*i))
        torch.cuda.synchronize()
        for g, r in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(g, r))


def test_a_step_inside_the_context_in_a_graph(gpu):
    """What torch code saves is kept in 8 bits and read back within the capture; replayed with other inputs and eager work in between."""
    import hpfp8
    w, head, nw = randn((512, 256), 50, 0.05).requires_grad_(), randn((700, 256), 51, 0.05).requires_grad_(), randn((256,), 52).requires_grad_()
    batches = [(randn((90, 256), 53 + i), torch.randint(700, (90,), generator=torch.Generator().manual_seed(60 + i)).cuda()) for i in range(3)]

    def step(x, target):
        x = x.detach().requires_grad_()
        with hpfp8.keep_activations_8bit(min_elements=1000):
            h = torch.nn.functional.linear(hpfp8.layer_norm(x, 256, nw), w)
            gate, up = h.chunk(2, -1)
            y = torch.nn.functional.silu(gate.masked_fill(gate > 2, -math.inf).clamp(min=-9)) * up
            each = hpfp8.linear_cross_entropy(y, head, target, reduction="none")
        return (each.detach(),) + torch.autograd.grad(each.mean(), (x, w, head, nw))
    x, target = batches[0][0].clone(), batches[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, target)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = step(x, target)
    for a, b in batches + batches:
        want = [t.clone() for t in step(a, b)]
        x.copy_(a)
        target.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outputs, want)) and all(t.isfinite().all() for t in want)


def test_threads_side_by_side(gpu):
    """Each on a stream of its own, half of them inside the context, which is a thread's own: results as one after the other."""
    import contextlib
    import threading
    import hpfp8
    head, nw, w = randn((1500, 256), 70, 0.05), randn((256,), 71), randn((256, 256), 72, 0.1)
    inputs = [(randn((200 + 50 * i, 256), 73 + i), torch.randint(1500, (200 + 50 * i,), generator=torch.Generator().manual_seed(i)).cuda()) for i in range(4)]

    def step(i):
        x, t = inputs[i]
        leaves = [v.clone().requires_grad_() for v in (x, head, nw, w)]
        with hpfp8.keep_activations_8bit(min_elements=1000) if i % 2 else contextlib.nullcontext():
            y = torch.nn.functional.silu(hpfp8.fp8_linear(hpfp8.layer_norm(leaves[0], 256, leaves[2]), leaves[3]))
            loss = hpfp8.linear_cross_entropy(hpfp8.activation(y, "gelu"), leaves[1], t)
        return torch.autograd.grad(loss, leaves)
    want = [step(i) for i in range(4)]
    torch.cuda.synchronize()
    got, errors = [[None] * 5 for _ in range(4)], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for k in range(5):
                    got[i][k] = step(i)
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for i in range(4):
        assert all(torch.equal(p, q) for k in range(5) for p, q in zip(got[i][k], want[i]))
