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
