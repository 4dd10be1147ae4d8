"""Calls of layer norm, Newton-Schulz and the Muon step that the device cannot
serve, with tensors that are really there (those that are not:
test_device_calls_cpu.py)."""

import pytest
import torch

from stochastic_gradient_push_amd import ops

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda", 0)


@pytest.mark.filterwarnings("ignore:Accessing the data pointer")
def test_results_without_memory():
    """Real inputs under a mode in which new tensors have no memory."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    x = torch.randn(4, 8, device=dev())
    leaf = x.clone().requires_grad_(True)
    y = ops.layer_norm(leaf)
    plan = ops.MuonPlan([(0, 4, 8)], 32, "cuda")
    flat = [x.flatten().clone() for _ in range(3)]
    lr = torch.ones(1, device=dev())
    with FakeTensorMode(allow_non_fake_inputs=True):
        with pytest.raises(RuntimeError, match="no memory"):
            ops.layer_norm(x)
        with pytest.raises(RuntimeError):
            y.backward(x)
        with pytest.raises(RuntimeError):
            ops.newton_schulz(x)
        with pytest.raises(RuntimeError, match="no memory"):
            ops.muon_step_(*flat, plan, lr)
    assert all(torch.equal(t, x.flatten()) for t in flat)
    with pytest.raises(RuntimeError, match="no memory"):
        torch.func.functionalize(ops.layer_norm)(x)
    for call in (torch.func.vmap(ops.layer_norm),
                 torch.func.grad(lambda t: ops.layer_norm(t).sum())):
        with pytest.raises(RuntimeError):
            call(x)
