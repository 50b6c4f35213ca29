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
