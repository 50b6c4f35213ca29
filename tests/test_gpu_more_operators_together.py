"""Norm, linears and clipping as a program runs them: a training step of a block, a served block in 8 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def randn(shape, seed, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


class Block(torch.nn.Module):
    """A pre-norm residual block: the stream is added in the next norm."""

    def __init__(self, hidden, inner, apply_grad_on_fp32_main_grad):
        import hpfp8
        super().__init__()
        self.norm = hpfp8.RMSNorm(hidden, 1e-6, device="cuda")
        self.up = hpfp8.Fp8Linear(hidden, inner, device="cuda", apply_grad_on_fp32_main_grad=apply_grad_on_fp32_main_grad)
        self.down = hpfp8.Fp8Linear(inner, hidden, device="cuda", apply_grad_on_fp32_main_grad=apply_grad_on_fp32_main_grad)

    def forward(self, x, residual):
        import hpfp8
        y, stream = self.norm(x, residual)
        return self.down(hpfp8.activation(self.up(y), "silu")), stream


def test_a_training_step_with_main_gradients_and_clipping(gpu):
    import hpfp8
    torch.manual_seed(0)
    block = Block(256, 384, True)
    x, residual = randn((100, 256), 1).requires_grad_(), randn((100, 256), 2).requires_grad_()
    out, stream = block(x, residual)
    (out.float() ** 2).sum().add((stream.float() ** 2).sum()).backward()
    grads = {n: (p.main_grad if getattr(p, "main_grad", None) is not None else p.grad).clone() for n, p in block.named_parameters()}
    assert grads["up.weight"].dtype == torch.float32 and grads["norm.weight"].dtype == torch.bfloat16
    norm = hpfp8.clip_grad_norm_(block.parameters(), 1.0)
    exact = torch.sqrt(sum((g.double() ** 2).sum() for g in grads.values()))
    assert abs(float(norm) - float(exact)) <= 2.0 ** -23 * float(exact) and float(norm) > 1
    factor = 1.0 / (norm + 1e-6)
    for n, p in block.named_parameters():
        g = p.main_grad if getattr(p, "main_grad", None) is not None else p.grad
        assert torch.equal(g, (grads[n].float() * factor).to(g.dtype)), n
    # the norm's own part against torch in fp32: what reaches x and the residual is the same tensor's gradient
    assert torch.equal(x.grad, residual.grad)


def test_a_served_block_in_8_bits_is_its_operators_one_by_one(gpu):
    import hpfp8
    x, residual, w = randn((37, 512), 1), randn((37, 512), 2), randn((512,), 3)
    weight = randn((1024, 512), 4, 0.02)
    with torch.no_grad():
        y, stream = hpfp8.rms_norm(x, 512, w, 1e-6, residual=residual)
        # int8: from fp32 where the two steps round y to bf16 between them: off by a rounding of y (2^-8 of a value) and a step
        w8 = hpfp8.quantize_weight_int8(weight)
        codes, scale, total = hpfp8.rms_norm_quantize_int8(x, w, 1e-6, residual=residual)
        assert torch.equal(total, stream)
        fused = hpfp8.gemm_int8(codes, scale, w8.codes, w8.scale_inv)
        apart = hpfp8.int8_linear(y, w8)
        exact = y.double() @ w8.dequantize(torch.float64).t()
        reach = w8.dequantize(torch.float64).abs().sum(1)
        step = scale.double().unsqueeze(1) * 1.01 + 2.0 ** -8 * y.double().abs().amax(1, keepdim=True)
        for got in (fused, apart):
            assert ((got.double() - exact).abs() <= step * reach + 2.0 ** -7 * exact.abs()).all()
        # FP8, with both recipes
        for pow2 in (False, True):
            f8 = hpfp8.quantize_weight(weight, with_transpose=False, pow2=pow2)
            codes, scale, total = hpfp8.rms_norm_quantize_1x128(x, w, 1e-6, residual=residual, pow2=pow2)
            assert torch.equal(total, stream)
            fused = hpfp8.gemm_blockwise(codes, scale, f8.codes, f8.scale_inv, pow2_scales=pow2)
            apart = hpfp8.fp8_linear(y, weight, weight_fp8=f8, recipe="blockwise_pow2" if pow2 else "blockwise")
            rel = (fused.float() - apart.float()).norm() / apart.float().norm()
            assert rel < 2.0 ** -4                           # (each code is within half a step, 2^-4, of its value)


def test_a_step_captured_and_replayed(gpu):
    import hpfp8
    torch.manual_seed(1)
    block = Block(256, 256, False)
    x, residual = randn((64, 256), 5), randn((64, 256), 6)
    held, other = x.clone(), residual.clone()

    def run():
        out, stream = block(held, other)
        grads = torch.autograd.grad((out.float() * stream.float()).sum(), list(block.parameters()))
        for p, g in zip(block.parameters(), grads):
            p.grad = g
        norm = hpfp8.clip_grad_norm_(block.parameters(), 0.5)
        return [out.detach(), stream.detach(), norm] + [p.grad for p in block.parameters()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for k in range(4):
        held.copy_(x * (1 + k))
        other.copy_(residual - k)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, run()))


def test_two_graphs_and_eager_calls_on_streams_of_their_own(gpu):
    """No workspace is shared: two captured graphs and the eager call run at once."""
    import hpfp8
    xs = [randn((1024, 2048), i) for i in range(3)]
    w8 = hpfp8.quantize_weight_int8(randn((512, 2048), 9, 0.02))
    gs = [[randn((300000,), 20 + i, dtype=torch.float32), randn((70001,), 30 + i)] for i in range(3)]

    def run(i):
        with torch.no_grad():
            codes, scale = hpfp8.rms_norm_quantize_int8(xs[i])
            return [hpfp8.gemm_int8(codes, scale, w8.codes, w8.scale_inv), hpfp8.get_total_norm(gs[i])]
    want = [[t.clone() for t in run(i)] for i in range(3)]
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(i))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(3):
        for t in outs[0] + outs[1]:
            t.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            eager = run(2)
        torch.cuda.synchronize()
        for got, expected in zip(outs + [eager], want):
            assert all(torch.equal(a, b) for a, b in zip(got, expected))
