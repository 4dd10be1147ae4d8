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


def test_inference_mode_and_one_dimension():
    with torch.inference_mode():
        x, w = torch.randn(8, device=dev()), torch.randn(8, device=dev())
        y = ops.layer_norm(x, w, residual=x, relu=True)
        want = torch.relu(torch.nn.functional.layer_norm(x, (8,), w) + x)
        assert y.shape == (8,) and float((y - want).abs().max()) <= 1e-5
        g = torch.randn(4, 6, device=dev())
        o = ops.newton_schulz(g)
        plan = ops.MuonPlan([(0, 4, 6)], 24, "cuda")
        p, buf = (torch.zeros(24, device=dev()) for _ in range(2))
        ops.muon_step_(p, g.flatten(), buf, plan, 1.0, nesterov=False)
        # both in one block or in tiles: within the bound of five steps of
        # fp32 roundings, 5 * 485 * 8 * 2^-23, each
        assert float((p.view(4, 6) + o).norm()) <= 2 * 2.4e-3
    leaf = torch.randn(8, device=dev(), requires_grad=True)
    dx, = torch.autograd.grad(ops.layer_norm(leaf, relu=True).sum(), leaf)
    assert dx.shape == (8,)
    empty = torch.empty(0, 3, 8, device=dev(), requires_grad=True)
    dx, = torch.autograd.grad(ops.layer_norm(empty, relu=True).sum(), empty)
    assert dx.shape == (0, 3, 8)


def test_compiled_callers():
    """A compiled function calls the kernels between its graphs."""
    import torch._dynamo

    x = torch.randn(6, 8, device=dev())
    w = torch.randn(8, device=dev(), requires_grad=True)

    def f(t, w):
        return ops.layer_norm(t * 2, w).sin()

    compiled = torch.compile(f, backend="eager")
    y, ref = compiled(x, w), f(x, w)
    assert torch.equal(y, ref)
    got, = torch.autograd.grad(y.sum(), w)
    want, = torch.autograd.grad(ref.sum(), w)
    assert torch.equal(got, want)
