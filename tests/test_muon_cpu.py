"""Newton-Schulz and the Muon step on the CPU: the reference path against 64
bits, plans, refusals, the optimiser and the trainer that uses it."""

import copy

import pytest
import torch

from stochastic_gradient_push_amd import GossipDataParallel, ops
from stochastic_gradient_push_amd.models import resnet18
from stochastic_gradient_push_amd.ops.flat import FlatParams
from stochastic_gradient_push_amd.ops.fused_muon import FusedMuon

from .test_trainer import _run_trainer

COEF = (3.4445, -4.7750, 2.0315)


def factor(g, steps=5, coef=COEF, eps=1e-7):
    """The definition in 64 bits."""
    a, b, c = coef
    x = g.double()
    x = x / (x.norm() + eps)
    for _ in range(steps):
        s = x @ x.T
        x = a * x + b * s @ x + c * s @ s @ x
    return x


@pytest.mark.parametrize("shape", [(1, 1), (3, 8), (8, 3), (40, 40),
                                   (20, 70)])
def test_reference_path(shape):
    torch.manual_seed(0)
    g = torch.randn(*shape)
    out = ops.newton_schulz(g)
    ref = factor(g)
    # fp32 roundings of X (norm 1) grow by 485 in five steps
    assert float((out - ref).norm()) <= 5 * 485 * 8 * 2.0 ** -24
    # singular values are near 1 (gaussian: the smallest start at 1e-3)
    sv = torch.linalg.svdvals(out.double())
    assert float(sv.max()) < 1.21
    if shape == (20, 70):
        assert float(sv.min()) > 0.68 - 1e-3


def test_batch_and_layout():
    torch.manual_seed(1)
    g = torch.randn(2, 3, 9, 5)
    out = ops.newton_schulz(g)
    for i in range(2):
        for j in range(3):
            assert torch.allclose(out[i, j], ops.newton_schulz(g[i, j]),
                                  atol=1e-5)
    t = ops.newton_schulz(g.mT)
    assert t.is_contiguous() and torch.allclose(t, out.mT, atol=1e-5)
    assert ops.newton_schulz(g.bfloat16()).dtype == torch.bfloat16
    assert ops.newton_schulz(torch.empty(0, 4, 4)).shape == (0, 4, 4)


def test_zeros_and_bad_values():
    assert bool((ops.newton_schulz(torch.zeros(4, 6)) == 0).all())
    for bad in (float("nan"), float("inf")):
        g = torch.randn(4, 6)
        g[1, 2] = bad
        assert bool(torch.isnan(ops.newton_schulz(g)).all())


@pytest.mark.parametrize("call,error", [
    (lambda g: ops.newton_schulz(g[0]), ValueError),
    (lambda g: ops.newton_schulz(g.double()), TypeError),
    (lambda g: ops.newton_schulz(g, steps=0), ValueError),
    (lambda g: ops.newton_schulz(g, steps=101), ValueError),
    (lambda g: ops.newton_schulz(g, steps=2.0), ValueError),
    (lambda g: ops.newton_schulz(g, eps=-1.0), ValueError),
    (lambda g: ops.newton_schulz(g, eps=float("nan")), ValueError),
    (lambda g: ops.newton_schulz(g, coefficients=(1.0, 2.0)), ValueError),
    # singular values run away
    (lambda g: ops.newton_schulz(g, coefficients=(3.0, 1.0, 1.0)),
     ValueError),
    (lambda g: ops.newton_schulz(g, coefficients=(float("nan"), 0.0, 0.0)),
     ValueError),
    (lambda g: ops.newton_schulz(g, coefficients=(1.9, -80.0, 79.0)),
     ValueError),
    (lambda g: ops.newton_schulz(g.requires_grad_(True)), RuntimeError),
])
def test_refusals(call, error):
    with pytest.raises(error, match="newton_schulz"):
        call(torch.randn(4, 6))


def test_other_coefficients():
    # the cubic that converges to 1
    g = torch.randn(6, 10)
    out = ops.newton_schulz(g, steps=30, coefficients=(1.5, -0.5, 0.0))
    sv = torch.linalg.svdvals(out.double())
    assert float((sv - 1).abs().max()) < 1e-4


@pytest.mark.parametrize("coef", [COEF, (1.5, -0.5, 0.0),
                                  (1.875, -1.25, 0.375), (2.0, -1.5, 0.5)])
@pytest.mark.parametrize("steps", [1, 2, 5, 10, 100])
def test_steps_in_one_number(coef, steps):
    """As many last steps as let their roundings grow to 16 in all."""
    from stochastic_gradient_push_amd.ops import muon

    growth = muon._growth(coef, steps)
    for dtype in (torch.float32, torch.float16):
        assert muon._split_steps(steps, growth, dtype) == steps
    single = steps - muon._split_steps(steps, growth, torch.bfloat16)
    assert 0 <= single <= steps
    assert sum(growth ** k for k in range(1, single + 1)) <= 16
    assert single == steps or sum(
        growth ** k for k in range(1, single + 2)) > 16


def test_plan_refusals():
    with pytest.raises(ValueError, match="overlaps"):
        ops.MuonPlan([(0, 2, 3), (5, 1, 1)], 10, "cpu")
    with pytest.raises(ValueError, match="overlaps|before"):
        ops.MuonPlan([(-1, 2, 3)], 10, "cpu")
    with pytest.raises(ValueError, match="behind"):
        ops.MuonPlan([(6, 2, 3)], 10, "cpu")
    with pytest.raises(ValueError, match="rows"):
        ops.MuonPlan([(0, 0, 3)], 10, "cpu")
    plan = ops.MuonPlan([(0, 2, 3)], 10, "cpu")
    p = torch.zeros(10)
    with pytest.raises(ValueError, match="grads"):
        ops.muon_step_(p, torch.zeros(9), p.clone(), plan, 0.1)
    with pytest.raises(ValueError, match="params"):
        ops.muon_step_(p[:9], p, p.clone(), plan, 0.1)
    with pytest.raises(ValueError, match="plan is for"):
        ops.muon_step_(p.to("meta"), p, p.clone(), plan, 0.1)
    with pytest.raises(ValueError, match="share memory"):
        ops.muon_step_(p, torch.zeros(10), p, plan, 0.1)
    both = torch.zeros(15)
    with pytest.raises(ValueError, match="share memory"):
        ops.muon_step_(p, both[:10], both[5:], plan, 0.1)


def step_oracle(p, g, buf, matrices, lr, mu, wd, nesterov, rest_lr):
    p, g, buf = p.double(), g.double(), buf.double()
    inside = torch.zeros(p.numel(), dtype=torch.bool)
    for start, rows, cols in matrices:
        inside[start:start + rows * cols] = True
    g = g + wd * p * ~inside
    buf = mu * buf + g
    u = g + mu * buf if nesterov else buf
    new = torch.where(inside, p * (1 - lr * wd), p - lr * rest_lr * u)
    for start, rows, cols in matrices:
        part = slice(start, start + rows * cols)
        scale = max(1.0, rows / cols) ** 0.5
        new[part] -= lr * scale * factor(u[part].view(rows, cols)).reshape(-1)
    return new, buf


@pytest.mark.parametrize("nesterov", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step(nesterov, dtype):
    torch.manual_seed(2)
    matrices = [(3, 8, 5), (60, 4, 9), (43, 1, 6)]
    plan = ops.MuonPlan(matrices, 110, "cpu")
    p, buf = torch.randn(110), torch.randn(110)
    g = torch.randn(110).to(dtype)
    shadow = torch.empty(110, dtype=torch.bfloat16)
    want, wbuf = step_oracle(p, g, buf, matrices, 0.05, 0.9, 0.1, nesterov,
                             0.3)
    ops.muon_step_(p, g, buf, plan, 0.05, momentum=0.9, weight_decay=0.1,
                   nesterov=nesterov, rest_lr=0.3, shadow=shadow)
    assert torch.allclose(p.double(), want, atol=1e-4)
    assert torch.allclose(buf.double(), wbuf, atol=1e-6)
    assert torch.equal(shadow, p.bfloat16())


class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.conv = torch.nn.Conv2d(3, 6, 3)
        self.norm = torch.nn.BatchNorm1d(6)
        self.fc = torch.nn.Linear(6, 4)

    def forward(self, x):
        return self.fc(self.norm(self.conv(x).mean((2, 3))))


def test_optimizer_splits_matrices_and_vectors():
    torch.manual_seed(3)
    net = Net()
    start = {k: v.detach().clone() for k, v in net.named_parameters()}
    flatp = FlatParams(net, flatten_grads=True)
    opt = FusedMuon(flatp, lr=0.1, momentum=0.9, nesterov=False,
                    rest_lr=0.5, sgd_params=[net.fc.weight])
    net(torch.randn(5, 3, 6, 6)).square().mean().backward()
    grads = {k: v.grad.detach().clone() for k, v in net.named_parameters()}
    opt.step()
    for name, p in net.named_parameters():
        if name == "conv.weight":
            step = factor(grads[name].reshape(6, 27)).view_as(p)
            want = start[name] - 0.1 * step
        else:
            want = start[name] - 0.05 * grads[name]
        assert torch.allclose(p.double(), want.double(), atol=1e-5), name
    opt.zero_grad()
    assert bool((flatp.flat_grad == 0).all())
    with pytest.raises(ValueError, match="sgd_params"):
        FusedMuon(flatp, lr=0.1, sgd_params=[torch.nn.Parameter(
            torch.zeros(2, 2))])


def test_optimizer_state_round_trip():
    torch.manual_seed(4)
    net = Net()
    flatp = FlatParams(net, flatten_grads=True)
    opt = FusedMuon(flatp, lr=0.1)
    flatp.flat_grad.normal_()
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    other = FusedMuon(FlatParams(copy.deepcopy(net), flatten_grads=True),
                      lr=0.7, momentum=0.5)
    other.load_state_dict(saved)
    assert torch.equal(other.momentum_buf, opt.momentum_buf)
    assert other.param_groups[0]["lr"] == 0.1
    flatp.flat_grad.normal_()
    other.flatp.flat_grad.copy_(flatp.flat_grad)
    other.flatp.flat.copy_(flatp.flat)
    opt.step()
    other.step()
    assert torch.equal(opt.flatp.flat, other.flatp.flat)


def test_working_weights_follow():
    torch.manual_seed(5)
    net = resnet18(num_classes=5, norm="layer")
    gdp = GossipDataParallel(net, rank=0, world_size=1,
                             working_dtype=torch.bfloat16)
    opt = FusedMuon(gdp.flatp, lr=0.02, steal_grads=True)
    before = gdp.flatp.flat.clone()
    for p in net.parameters():
        p.grad = torch.randn_like(p)
    opt.step()
    flatp = gdp.flatp
    assert torch.equal(flatp.shadow, flatp.flat[:flatp.n_cast].bfloat16())
    assert bool((flatp.flat != before).float().mean() > 0.99)
    gdp.shutdown()


def test_trainer_with_layer_norm_and_muon(tmp_path):
    _run_trainer(tmp_path, ["--norm", "layer", "--optimizer", "muon",
                            "--lr", "0.02", "--rest_lr", "0.1"])


def test_trainer_refuses_muon_without_flat_parameters(tmp_path):
    import subprocess

    with pytest.raises(subprocess.CalledProcessError):
        _run_trainer(tmp_path, ["--optimizer", "muon", "--fused_sgd",
                                "False"])


def test_reduced_is_for_the_device():
    g = torch.randn(6, 10)
    for dtype in (torch.float32, torch.bfloat16):
        assert torch.equal(ops.newton_schulz(g.to(dtype), reduced=True),
                           ops.newton_schulz(g.to(dtype)))


def test_plan_refuses_more_than_a_launch_holds():
    # 2^24 chunks of 2048 values, a block of 256 threads each
    ext = ops._load_extension()
    if ext is None:
        pytest.skip("extension not built")
    with pytest.raises(RuntimeError, match="too many"):
        ext.muon_plan([], 2048 << 24)
    tables, layout = ext.muon_plan([(0, 4, 6, 1.0)], 1 << 20)
    assert layout[1] == 1 + 512 and tables.numel() > 0
