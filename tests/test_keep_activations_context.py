"""What `keep_activations_8bit` leaves as it is, without a GPU: tensors on the CPU are all of that kind."""
import gc
import weakref

import pytest
import torch


def test_a_graph_that_is_dropped_without_a_backward_is_freed():
    """A node that saves its own result must not hold it through what the context puts in its place."""
    import hpfp8
    x = torch.randn(100, requires_grad=True)
    with hpfp8.keep_activations_8bit(min_elements=1):
        for f in (torch.exp, torch.tanh, lambda t: torch.softmax(t * 2, 0), lambda t: (t * 1).relu()):
            y = f(x)
            result = weakref.ref(y)
            del y
            gc.collect()
            assert result() is None


def test_a_write_to_a_saved_tensor_is_noticed():
    """As outside the context; a write before it was saved, or after the backward, is none."""
    import hpfp8
    x, w = torch.randn(100, requires_grad=True), torch.nn.Parameter(torch.randn(100))
    with hpfp8.keep_activations_8bit(min_elements=1):
        y = x * 1
        y.add_(1)
        z = torch.exp(y) * w
    go = torch.ones(100)
    dx, dw = torch.autograd.grad(z, (x, w), go, retain_graph=True)
    assert torch.equal(dw, torch.exp(y.detach())) and torch.equal(dx, w.detach() * torch.exp(y.detach()))
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(z, (x, w), go)
    with hpfp8.keep_activations_8bit(min_elements=1):
        y = torch.exp(x)
    with torch.no_grad():
        y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, go)


@pytest.mark.parametrize("second", [False, True])
def test_gradients_of_what_stays_are_those_outside(second):
    """Operations in place, nodes that save their result, views; first and second derivatives."""
    import contextlib
    import hpfp8
    x, w = torch.randn(30, 40, generator=torch.Generator().manual_seed(0)), torch.randn(30, 40, generator=torch.Generator().manual_seed(1))
    for f in (lambda x, w: ((x * 1).relu_() * w).sigmoid_() * w, lambda x, w: ((x * 0.1) ** 3).cumsum(0).exp() * w, lambda x, w: torch.linalg.norm(x @ w.t(), dim=1),
              lambda x, w: x.t().contiguous().view(-1)[::3] ** 2 * w.view(-1)[::3]):
        results = []
        for context in (contextlib.nullcontext(), hpfp8.keep_activations_8bit(min_elements=1)):
            leaves = [t.clone().requires_grad_() for t in (x, w)]
            with context:
                y = f(*leaves)
                grads = torch.autograd.grad((y * y).sum(), leaves, create_graph=second)
            results.append(torch.autograd.grad(sum(g.sum() for g in grads), leaves) if second else grads)
        assert all(torch.equal(p, q) for p, q in zip(*results))
