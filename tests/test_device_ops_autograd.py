"""What the operators on device matrices say to torch's autograd, without a GPU."""
import pytest
import torch

import nmfx
from nmfx import device


def test_results_without_a_graph_refuse_a_backward_pass():
    W, H = torch.zeros(4, 2, requires_grad=True), torch.zeros(2, 3)
    loss, lse = device._no_graph().apply(W, H, lambda: (torch.tensor(2.0), torch.ones(3)))
    assert loss.requires_grad and lse.requires_grad and float(loss.detach()) == 2
    for part in (loss, lse.sum(), loss + W.sum()):
        with pytest.raises(nmfx.ArgumentError, match="softmax_xent_grad"):
            part.backward(retain_graph=True)
    (loss.detach() + W.sum()).backward()
    assert (W.grad == 1).all()


def test_host_tensors_are_refused_with_and_without_gradients(built):
    for grad in (False, True):
        with pytest.raises(nmfx.ArgumentError, match="no CPU path"):
            nmfx.softmax_xent(torch.zeros(4, 2, requires_grad=grad), torch.zeros(2, 3), torch.zeros(3, dtype=torch.int64))
