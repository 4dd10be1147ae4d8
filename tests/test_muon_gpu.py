"""Newton-Schulz and Muon kernels against the definition in 64 bits.

Bounds are in the Frobenius norm.  X starts with norm 1; a rounding of size
d relative to X, A or B in any step grows by at most a = 3.4445 in each step
up to the result, so by a^5 = 485 in all.  A step rounds X, A and B to 22
bits (2^-23) and accumulates three products in fp32; eight such roundings a
step are allowed: 5 * 485 * 8 * 2^-23 = 2.3e-3 for a result whose norm is
about sqrt(n), against 0.12 per rounding for values of 11 bits.  Sharper,
where the input is noise: at most four times the error of the same formulas
in fp32, two bits for 22-bit values instead of 24.
"""

import copy

import pytest
import torch

from stochastic_gradient_push_amd import GossipDataParallel, ops
from stochastic_gradient_push_amd.models import resnet18
from stochastic_gradient_push_amd.ops.flat import FlatParams
from stochastic_gradient_push_amd.ops.fused_muon import FusedMuon

from .test_muon_cpu import COEF, Net

pytestmark = pytest.mark.gpu

BOUND = 5 * 485 * 8 * 2.0 ** -23


def dev():
    return torch.device("cuda", 0)


def factor(g, steps=5, coef=COEF, eps=1e-7):
    """The definition, in 64 bits on the CPU."""
    a, b, c = coef
    x = g.detach().double().cpu()
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + eps)
    for _ in range(steps):
        s = x @ x.mT if x.shape[-2] <= x.shape[-1] else x.mT @ x
        eye = torch.eye(s.shape[-1], dtype=s.dtype)
        p = a * eye + s @ (b * eye + c * s)
        x = p @ x if x.shape[-2] <= x.shape[-1] else x @ p
    return x.to(g.device)


def rounding(ref, dtype):
    """Norm of one rounding to the type."""
    return torch.finfo(dtype).eps / 2 * float(ref.norm())


def strong(rows, cols, seed=0, batch=()):
    """A few strong directions over noise."""
    g = torch.Generator(device=dev()).manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device=dev())

    k = min(rows, cols, 3)
    return randn(*batch, rows, cols) + torch.matmul(
        randn(*batch, rows, k), randn(*batch, k, cols))


# one block's, both tiles, their borders, both orientations
SHAPES = [(1, 1), (1, 9), (7, 1), (3, 2), (16, 16), (63, 65), (64, 64),
          (65, 64), (65, 65), (64, 192), (64, 193), (192, 33), (193, 33),
          (20, 129), (64, 576), (640, 40), (129, 257), (256, 256), (257, 300),
          (300, 1000), (1000, 260), (512, 512), (385, 385)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
def test_shapes(shape, dtype):
    g = strong(*shape, seed=sum(shape)).to(dtype)
    out = ops.newton_schulz(g)
    assert out.dtype == dtype and out.shape == g.shape
    assert out.is_contiguous()
    ref = factor(g)
    # bf16: the last two steps round to 11 bits, which grows by a^2 = 12,
    # in each of X, A and B
    single = 6 * 12 * 2.0 ** -12 * float(ref.norm()) \
        if dtype == torch.bfloat16 else 0.0
    err = float((out.double() - ref).norm())
    assert err <= BOUND + rounding(ref, dtype) + single, (
        err, float(ref.norm()))


# at 1e-3 the norm is not so far above eps that |G| / (|G| + eps) is 1
@pytest.mark.parametrize("scale", [1.0, 1e-3, 3e-6])
@pytest.mark.parametrize("shape", [(64, 64), (64, 190), (200, 300),
                                   (128, 1152), (512, 512), (700, 300)])
def test_noise_against_fp32(shape, scale):
    g = scale * torch.randn(*shape, device=dev())
    ref = factor(g)
    x = g.clone()
    tall = shape[0] > shape[1]
    x = x.T.contiguous() if tall else x
    x = x / (x.norm() + 1e-7)
    a, b, c = COEF
    for _ in range(5):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    plain = float(((x.T if tall else x).double() - ref).norm())
    err = float((ops.newton_schulz(g).double() - ref).norm())
    assert err <= 4 * plain + 4 * 2.0 ** -24 * float(ref.norm()), (err, plain)
    # bf16: no further off than twice its own rounding
    g = g.bfloat16()
    ref = factor(g)
    err = float((ops.newton_schulz(g).double() - ref).norm())
    own = float((ref.bfloat16().double() - ref).norm())
    assert err <= 2 * own, (err, own)


def test_noise_in_groups_of_large_matrices():
    # steps in groups from m = 2 n on, at four times the error of the same
    # formulas in fp32 like smaller ones
    g = torch.randn(800, 1700, device=dev())
    ref = factor(g)
    x = g / (g.norm() + 1e-7)
    a, b, c = COEF
    for _ in range(5):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    plain = float((x.double() - ref).norm())
    for h in (g, g.T):
        out = ops.newton_schulz(h)
        out = out if h is g else out.T
        err = float((out.double() - ref).norm())
        assert err <= 4 * plain + 4 * 2.0 ** -24 * float(ref.norm())


@pytest.mark.parametrize("batch,rows,cols", [
    ((5,), 48, 80), ((2, 3), 100, 70), ((3,), 300, 270), ((17,), 16, 5)])
def test_batches(batch, rows, cols):
    g = strong(rows, cols, batch=batch)
    out = ops.newton_schulz(g)
    flat, each = g.view(-1, rows, cols), out.view(-1, rows, cols)
    for i in range(flat.shape[0]):
        # a matrix's result does not depend on what lies beside it (nor, at
        # these sizes, on how many there are)
        assert torch.equal(each[i], ops.newton_schulz(flat[i])), i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tiles_of_both_sizes(dtype):
    # 20 of 9 x 11 tiles of 64: X X^T in tiles of 128 and a row of 64s, B X
    # in a round of 128s and the rest in 64s
    g = strong(560, 700, batch=(20,)).to(dtype)
    ref = factor(g)
    out = ops.newton_schulz(g)
    single = 6 * 12 * 2.0 ** -12 if dtype == torch.bfloat16 else 0.0
    for i in range(20):
        err = float((out[i].double() - ref[i]).norm())
        assert err <= BOUND + rounding(ref[i], dtype) + single * float(
            ref[i].norm()), i


def test_strides():
    g = strong(70, 90, batch=(4,))
    want = ops.newton_schulz(g)
    wide = torch.randn(4, 71, 97, device=dev())
    wide[:, 1:, 7:] = g
    assert torch.equal(ops.newton_schulz(wide[:, 1:, 7:]), want)
    assert torch.equal(ops.newton_schulz(g.mT.contiguous().mT), want)
    assert torch.equal(ops.newton_schulz(g[::2]), want[::2])
    same = ops.newton_schulz(g[:1].expand(3, 70, 90))
    assert torch.equal(same, want[:1].expand(3, 70, 90))
    # the transpose of the input gives the transpose of the result
    assert torch.equal(ops.newton_schulz(g.mT), want.mT)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e-8, 1e-3, 1e15, 1e30])
def test_scales(scale):
    # far below eps the result is 485 g / eps, not 0; far above, squares
    # leave fp32's range
    g = strong(60, 100) * scale
    ref = factor(g)
    out = ops.newton_schulz(g)
    r = float(g.double().norm() / (g.double().norm() + 1e-7))
    assert float((out.double() - ref).norm()) <= BOUND * r + \
        2.0 ** -149 * 100
    assert float(out.double().norm()) >= 0.9 * float(ref.norm())


def test_one_strong_entry():
    # all of the norm in one value: the largest that X can hold
    g = 1e-3 * torch.randn(512, 2048, device=dev())
    g[100, 1000] = 1e6
    for scale in (1.0, 1e-16):
        ref = factor(g * scale)
        out = ops.newton_schulz(g * scale)
        assert bool(torch.isfinite(out).all())
        assert float((out.double() - ref).norm()) <= BOUND


def test_zeros_and_bad_values():
    g = strong(70, 300, batch=(4,))
    clean = ops.newton_schulz(g)
    g[0] = 0
    g[1, 3, 5] = float("nan")
    g[2, 69, 299] = -float("inf")
    out = ops.newton_schulz(g)
    assert bool((out[0] == 0).all())
    assert bool(torch.isnan(out[1:3]).all())
    assert torch.equal(out[3], clean[3])
    for eps in (0.0, 1e-7):
        assert bool((ops.newton_schulz(torch.zeros_like(g[0]), eps=eps)
                     == 0).all())


@pytest.mark.parametrize("steps,coef", [
    (1, COEF), (2, COEF), (3, COEF), (4, COEF), (10, COEF), (25, (1.5, -0.5, 0.0)),
    (12, (1.875, -1.25, 0.375))])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [130, 400])  # steps one by one, in groups
def test_steps_and_coefficients(steps, coef, dtype, cols):
    g = torch.randn(90, cols, device=dev()).to(dtype)
    ref = factor(g, steps, coef)
    out = ops.newton_schulz(g, steps=steps, coefficients=coef)
    # growth up to the result is at most that from the start to size 1: a
    # singular value of noise starts above 1e-4 here
    growth = min(coef[0] ** steps, 1e4)
    bound = steps * growth * 8 * 2.0 ** -23
    single = 6 * 16 * 2.0 ** -12 * float(ref.norm()) \
        if dtype == torch.bfloat16 else 0.0
    err = float((out.double() - ref).norm())
    assert err <= bound + rounding(ref, dtype) + single


@pytest.mark.parametrize("steps,coef", [
    (8, (1.5, -0.5, 0.0)), (6, (1.875, -1.25, 0.375)), (8, (2.0, -1.5, 0.5))])
@pytest.mark.parametrize("shape", [(64, 100), (90, 400), (300, 200)])
def test_bf16_with_slow_coefficients(steps, coef, shape):
    # the steps in 11 bits add what 16 roundings of 2^-11 do if all of them
    # are the largest, twice the 2^-8 of the result's own; noise, half of it
    g = torch.randn(*shape, device=dev()).bfloat16()
    ref = factor(g, steps, coef)
    own = float((ref.bfloat16().double() - ref).norm())
    out = ops.newton_schulz(g, steps=steps, coefficients=coef)
    assert float((out.double() - ref).norm()) <= 2 * own


def test_same_call_same_bits():
    g = strong(300, 500, batch=(2,))
    first = ops.newton_schulz(g)
    assert all(torch.equal(ops.newton_schulz(g), first) for _ in range(3))


@pytest.mark.parametrize("rows,cols,batch", [(64, 64, 530_000),
                                             (256, 256, 33_000)])
def test_batch_beyond_32_bits(rows, cols, batch):
    g = torch.zeros(batch, rows, cols, device=dev(), dtype=torch.bfloat16)
    assert g.numel() > 1 << 31
    g[-2:] = strong(rows, cols, batch=(2,)).bfloat16()
    out = ops.newton_schulz(g)
    # against the definition, as in test_shapes: other tiles than for two
    # matrices, so other last bits
    for i in (-2, -1):
        ref = factor(g[i])
        err = float((out[i].double() - ref).norm())
        assert err <= BOUND + rounding(ref, torch.bfloat16) \
            + 6 * 12 * 2.0 ** -12 * float(ref.norm())
    assert bool((out[:2] == 0).all()) and bool((out[-3] == 0).all())


def test_step_beyond_32_bits():
    total = (1 << 31) + 40_000
    start = total - 20_001
    plan = ops.MuonPlan([(start, 100, 200)], total, "cuda")
    p, g, buf = (torch.zeros(total, device=dev()) for _ in range(3))
    g[start:start + 20_000] = strong(100, 200).flatten()
    g[-1] = 2.0
    ops.muon_step_(p, g, buf, plan, 0.5, momentum=0.9, nesterov=False)
    want = -0.5 * factor(g[start:start + 20_000].view(100, 200)).flatten()
    got = p[start:start + 20_000].double()
    assert float((got - want).norm()) <= 0.5 * BOUND
    assert float(p[-1]) == -1.0 and float(buf[-1]) == 2.0
    assert bool((p[:start] == 0).all())


def test_refusals():
    g = torch.randn(4, 6, device=dev())
    ext = ops._ext_for(g)
    with pytest.raises(RuntimeError, match="not differentiable"):
        ops.newton_schulz(g.clone().requires_grad_(True))
    with torch.no_grad():
        ops.newton_schulz(g.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="contiguous"):
        ext.newton_schulz(g, 5, 5, 1, *COEF, 4.0, 1e-7)
    with pytest.raises(RuntimeError, match="2\\^20"):
        ops.newton_schulz(torch.empty(1, (1 << 20) + 1, device=dev()))
    plan = ops.MuonPlan([(0, 4, 6)], 24, "cuda")
    flat = g.flatten().clone()
    with pytest.raises(RuntimeError, match="momentum_buf"):
        ops.muon_step_(flat, flat.clone(), flat.double(), plan, 0.1)
    with pytest.raises(RuntimeError, match="grads"):
        ops.muon_step_(flat, flat.half(), flat.clone(), plan, 0.1)
    with pytest.raises(RuntimeError, match="shadow"):
        ops.muon_step_(flat, flat.clone(), flat.clone(), plan, 0.1,
                       shadow=flat.clone())
    with pytest.raises(ValueError, match="plan is for"):
        ops.muon_step_(flat, flat.clone(), flat.clone(),
                       ops.MuonPlan([(0, 4, 6)], 24, "cpu"), 0.1)
    with pytest.raises(RuntimeError, match="overlap"):
        ext.muon_plan([(0, 4, 6, 1.0), (5, 2, 2, 1.0)], 24)
    with pytest.raises(RuntimeError, match="outside"):
        ext.muon_plan([(4, 4, 6, 1.0)], 24)


# ------------------------------------------------------------------- step

def oracle(p, g, buf, matrices, lr, mu, wd, nesterov, rest_lr):
    p, g, buf = p.double(), g.double(), buf.double()
    inside = torch.zeros(p.numel(), dtype=torch.bool, device=p.device)
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


LAYOUTS = {
    # odd places, gaps before, between and behind
    "mixed": ([(5, 64, 147), (20000, 256, 64), (9500, 30, 300),
               (40000, 1, 77), (40100, 77, 1), (50001, 300, 270)], 140007),
    "one": ([(0, 40, 30)], 1200),
    "none": ([], 20001),
    "small": ([(i * 50, 5 + i % 3, 6) for i in range(40)], 2000),
}


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [False, True])
def test_step(layout, dtype, nesterov):
    matrices, total = LAYOUTS[layout]
    torch.manual_seed(total)
    plan = ops.MuonPlan(matrices, total, "cuda")
    p, buf = (torch.randn(total, device=dev()) for _ in range(2))
    g = torch.randn(total, device=dev()).to(dtype)
    shadow = torch.empty(total, device=dev(), dtype=torch.bfloat16)
    lr, mu, wd, rest_lr = 0.05, 0.9, 0.1, 0.3
    for _ in range(2):
        want, wbuf = oracle(p, g, buf, matrices, lr, mu, wd, nesterov,
                            rest_lr)
        ops.muon_step_(p, g, buf, plan, lr, momentum=mu, weight_decay=wd,
                       nesterov=nesterov, rest_lr=rest_lr, shadow=shadow)
        # a few roundings of values of at most about 10
        assert float((buf.double() - wbuf).abs().max()) <= 64 * 2.0 ** -24
        tol = 64 * 2.0 ** -24 * torch.ones_like(want)
        for start, rows, cols in matrices:
            tol[start:start + rows * cols] += \
                lr * max(1.0, rows / cols) ** 0.5 * BOUND
        assert bool(((p.double() - want).abs() <= tol).all())
        for start, rows, cols in matrices:
            part = slice(start, start + rows * cols)
            scale = lr * max(1.0, rows / cols) ** 0.5
            assert float((p[part].double() - want[part]).norm()) <= \
                scale * BOUND + 8 * 2.0 ** -24 * float(want[part].norm())
        assert torch.equal(shadow, p.bfloat16())


def test_step_agrees_with_newton_schulz():
    torch.manual_seed(0)
    matrices = [(0, 100, 64), (6400, 64, 300)]
    plan = ops.MuonPlan(matrices, 25600, "cuda")
    g = torch.randn(25600, device=dev())
    p, buf = torch.zeros_like(g), torch.zeros_like(g)
    ops.muon_step_(p, g, buf, plan, 1.0, momentum=0.5, nesterov=False)
    assert torch.equal(buf, g)
    for start, rows, cols in matrices:
        part = slice(start, start + rows * cols)
        o = ops.newton_schulz(g[part].view(rows, cols)).reshape(-1)
        scale = max(1.0, rows / cols) ** 0.5
        # the two may group their steps differently; each is within BOUND of
        # the definition in the norm, so they are within twice that
        assert float((p[part] + scale * o).norm()) <= 2 * BOUND * scale


def test_step_with_tiles_of_both_sizes():
    # 66 of 512 x 512: more than a round of tiles of 128 of each product
    n, side = 66, 512
    plan = ops.MuonPlan([(i * side * side, side, side) for i in range(n)],
                        n * side * side)
    p, buf = (torch.zeros(plan.total, device=dev()) for _ in range(2))
    g = torch.randn(plan.total, device=dev())
    ops.muon_step_(p, g, buf, plan, 1.0, nesterov=False)
    o = ops.newton_schulz(g.view(n, side, side))
    for i in range(n):
        # both are within BOUND of the definition
        assert float((p.view_as(o)[i] + o[i]).norm()) <= 2 * BOUND, i


def test_optimizer_against_cpu():
    torch.manual_seed(1)
    cpu = Net()
    gpu = Net()
    gpu.load_state_dict(cpu.state_dict())
    gpu.to(dev())
    opts = []
    for net in (cpu, gpu):
        flatp = FlatParams(net, flatten_grads=True)
        opts.append(FusedMuon(flatp, lr=0.1, weight_decay=0.01,
                              sgd_params=[net.fc.weight], rest_lr=0.5))
    for _ in range(3):
        opts[0].flatp.flat_grad.normal_()
        opts[1].flatp.flat_grad.copy_(opts[0].flatp.flat_grad)
        for opt in opts:
            opt.step()
        # each within BOUND times lr of the definition, and so is the CPU
        assert float((opts[0].flatp.flat - opts[1].flatp.flat.cpu())
                     .abs().max()) <= 3 * 2 * 0.1 * BOUND


def test_working_weights_and_sgd_params():
    """bf16 working weights with a matrix among the SGD parameters: the
    cast section has matrices and plain values, the rest none."""
    torch.manual_seed(2)
    nets = [resnet18(num_classes=10, norm="layer")]
    nets.append(copy.deepcopy(nets[0]).to(dev()))
    opts = []
    for net in nets:
        gdp = GossipDataParallel(net, rank=0, world_size=1,
                                 working_dtype=torch.bfloat16)
        opts.append(FusedMuon(
            gdp.flatp, lr=0.1, weight_decay=0.01, rest_lr=0.5,
            sgd_params=[net.fc.weight, net.conv1.weight], steal_grads=True))
    for _ in range(2):
        for p, q in zip(nets[0].parameters(), nets[1].parameters()):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.to(dev())
        for opt in opts:
            opt.step()
    flat = opts[1].flatp
    # in two steps each matrix stays within BOUND times lr and its scale (at
    # most sqrt(2): the downsampling ones) of the definition, and so the CPU
    assert float((opts[0].flatp.flat - flat.flat.cpu()).abs().max()) <= (
        2 * 2 * 0.1 * 2 ** 0.5 * BOUND)
    assert torch.equal(flat.shadow, flat.flat[:flat.n_cast].bfloat16())


def _training(steps, capture):
    """A ResNet-18 with layer norm in the gossip wrapper: bf16 working
    weights, stolen gradients, layer norm and Muon together."""
    torch.manual_seed(7)
    net = resnet18(num_classes=10, norm="layer").to(dev()).to(
        memory_format=torch.channels_last)
    gdp = GossipDataParallel(net, rank=0, world_size=1,
                             working_dtype=torch.bfloat16)
    opt = FusedMuon(gdp.flatp, lr=0.02, rest_lr=0.1, weight_decay=0.01,
                    steal_grads=True)
    x = torch.randn(4, 3, 64, 64, device=dev()).to(
        memory_format=torch.channels_last)
    y = torch.randint(0, 10, (4,), device=dev())

    def step():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = torch.nn.functional.cross_entropy(net(x), y)
        loss.backward()
        opt.step()
        opt.zero_grad()
        return loss.detach()

    if not capture:
        for _ in range(steps):
            loss = step()
        return gdp, opt, loss
    for _ in range(2):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    for _ in range(steps - 2):
        graph.replay()
        torch.cuda.synchronize()
    return gdp, opt, loss


def test_layer_norm_and_muon_train_together():
    gdp, opt, loss = _training(3, capture=False)
    assert bool(torch.isfinite(loss)) and bool(
        torch.isfinite(gdp.flatp.flat).all())
    flatp = gdp.flatp
    assert torch.equal(flatp.shadow, flatp.flat[:flatp.n_cast].bfloat16())
    # every matrix moved by a full-rank step: its norm says so
    assert float(opt.momentum_buf.norm()) > 0
    gdp.shutdown()


def test_captured_training():
    # (convolutions may sum in another order from run to run, so that whole
    # trainings are not compared bit by bit; the step itself is, below)
    gdp, _, loss = _training(5, capture=True)
    assert bool(torch.isfinite(loss)) and bool(
        torch.isfinite(gdp.flatp.flat).all())
    gdp.shutdown()


def test_captured_step():
    matrices, total = LAYOUTS["mixed"]
    torch.manual_seed(3)
    plan = ops.MuonPlan(matrices, total, "cuda")
    state = [torch.randn(total, device=dev()) for _ in range(3)]
    lr = torch.tensor([0.05], device=dev())
    eager = [t.clone() for t in state]
    p, g, buf = state
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up on copies
        ops.muon_step_(p.clone(), g, buf.clone(), plan, lr)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.muon_step_(p, g, buf, plan, lr)
        o = ops.newton_schulz(g[:1000 * 9].view(100, 90))
    for k in range(4):
        g.normal_()
        eager[1].copy_(g)
        lr.fill_(0.05 / (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        ops.muon_step_(eager[0], eager[1], eager[2], plan, lr)
        want = ops.newton_schulz(eager[1][:1000 * 9].view(100, 90))
        for a, b in zip(state, eager):
            assert torch.equal(a, b), k
        assert torch.equal(o, want), k


def test_two_streams_at_once():
    g = [strong(200, 300, seed=i) for i in range(2)]
    want = [ops.newton_schulz(t) for t in g]
    streams = [torch.cuda.Stream() for _ in g]
    torch.cuda.synchronize()
    out = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                out[i].append(ops.newton_schulz(g[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in out[i])


def plain_error(g):
    """How far the formulas in fp32 are from the definition, and that."""
    ref = factor(g)
    x = g.float()
    x = x.mT.contiguous() if g.shape[0] > g.shape[1] else x
    x = x / (x.norm() + 1e-7)
    a, b, c = COEF
    for _ in range(5):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    x = x.mT if g.shape[0] > g.shape[1] else x
    return float((x.double() - ref).norm()), ref


# one block, tiles of 64, steps in groups, tiles of 128
@pytest.mark.parametrize("shape", [(60, 90), (300, 700), (90, 400),
                                   (1100, 257), (2100, 2200)])
def test_bf16_results_are_rounded_once(shape):
    """A result that is fp32's and then rounded is the rounded definition but
    where the border between two values lies in between.  A value off by d is
    on the wrong side with probability d / step, and then off by a step (at
    most 2^-7 of it), so the sum of the squares is about sum(d step), at most
    the product of the norms.  d as for fp32 results: four times that of
    fp32's formulas; twice all that for chance."""
    torch.manual_seed(sum(shape))
    g = torch.randn(*shape, device=dev()).bfloat16()
    plain, ref = plain_error(g)
    d = 4 * plain + 4 * 2.0 ** -24 * float(ref.norm())
    off = float((ops.newton_schulz(g).double()
                 - ref.bfloat16().double()).norm())
    assert off ** 2 <= 2 * d * 2.0 ** -7 * float(ref.norm()), (
        off / float(ref.norm()), plain)


@pytest.mark.parametrize("shape", [(60, 90), (300, 700)])
def test_reduced_steps_are_a_choice(shape):
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        g = strong(*shape, seed=sum(shape)).to(dtype)
        full, reduced = (ops.newton_schulz(g, reduced=r)
                         for r in (False, True))
        # only bf16 results can do with fewer bits
        assert torch.equal(full, reduced) == (dtype != torch.bfloat16)
        ref = factor(g)
        err = float((reduced.double() - ref).norm())
        assert err <= BOUND + rounding(ref, dtype) + (
            6 * 12 * 2.0 ** -12 * float(ref.norm())
            if dtype == torch.bfloat16 else 0.0)


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd

    g = torch.randn(4, 6, device=dev())
    plan = ops.MuonPlan([(0, 4, 6)], 24, "cuda")
    with fwd.dual_level():
        dual = fwd.make_dual(g, torch.ones_like(g))
        for grad in (False, True):
            with torch.set_grad_enabled(grad), \
                    pytest.raises(RuntimeError, match="forward-mode"):
                ops.newton_schulz(dual)
        ops.newton_schulz(dual.detach())
        flat = [g.flatten().clone() for _ in range(3)]
        for i in range(3):
            some = list(flat)
            some[i] = dual.flatten()
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops.muon_step_(*some, plan, 0.1)
        assert all(torch.equal(t, g.flatten()) for t in flat)


@pytest.mark.filterwarnings("ignore")
def test_tracing_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx

    g = torch.randn(4, 6, device=dev())
    plan = ops.MuonPlan([(0, 4, 6)], 24, "cuda")
    flat = [g.flatten().clone() for _ in range(3)]

    def step(p, grads, buf):
        ops.muon_step_(p, grads, buf, plan, torch.ones(1, device=dev()))
        return p

    for trace in (lambda f, a: torch.jit.trace(f, a),
                  lambda f, a: make_fx(f)(*a)):
        with pytest.raises(RuntimeError, match="traced"):
            trace(lambda t: ops.newton_schulz(t), (g,))
        with pytest.raises(RuntimeError, match="traced"):
            trace(step, tuple(flat))
    assert all(torch.equal(t, g.flatten()) for t in flat)


@pytest.mark.parametrize("shape", [(8, 24), (300, 100), (128, 640),
                                   (700, 800)])
def test_far_below_eps_with_many_steps(shape):
    # r = |G| / (|G| + eps) = 1e-23, whose square fp32 does not hold: values
    # that have grown to 1 after 85 steps still have to stop there
    steps, coef = 100, (1.875, -1.25, 0.375)
    torch.manual_seed(sum(shape))
    g = torch.randn(*shape, device=dev())
    g = g * (1e-30 / float(g.norm()))
    ref = factor(g, steps, coef)
    out = ops.newton_schulz(g, steps=steps, coefficients=coef)
    assert bool(torch.isfinite(out).all())
    # a step's eight roundings are relative to the norm, and grow as the
    # smallest singular value does
    s = torch.linalg.svdvals(g.double())
    bound = steps * 8 * 2.0 ** -23 * float(s.norm() / s.min())
    assert float((out.double() - ref).norm()) <= bound


def test_more_matrices_than_a_launch_has_threads():
    # a block of 256 threads a matrix: 2^32 from 2^24 on
    batch = (1 << 24) + 5
    g = torch.zeros(batch, 2, 3, device=dev(), dtype=torch.bfloat16)
    some = [0, 1, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, batch - 1]
    for i in some:
        g[i] = strong(2, 3, seed=i % 97).bfloat16()
    out = ops.newton_schulz(g)
    for i in some:
        assert torch.equal(out[i], ops.newton_schulz(g[i])), i
    assert int((out != 0).any(-1).any(-1).sum()) == len(some)


def input_roundings(g):
    """What roundings of the input do to the result: noise of size d |g|
    comes out as d |g| f(s) / s for each singular value s, where f(s) <=
    1.21; four roundings."""
    s = torch.linalg.svdvals(g.double())
    return 4 * 1.21 * 2.0 ** -24 * float(
        s.norm() * s.reciprocal().square().mean().sqrt())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_on_noise(dtype):
    """Steps on noise, as sharp as test_noise_against_fp32: four times the
    error of the same formulas in fp32, and the roundings of p."""
    matrices = [(3, 64, 147), (10_000, 256, 64), (30_001, 300, 270),
                (120_000, 128, 576), (200_003, 512, 640)]
    total = 600_001
    torch.manual_seed(4)
    plan = ops.MuonPlan(matrices, total, "cuda")
    p, buf = (torch.randn(total, device=dev()) for _ in range(2))
    g = torch.randn(total, device=dev()).to(dtype)
    lr, mu, wd = 0.5, 0.9, 0.1
    for nesterov in (False, True):
        before, was = p.double(), buf.clone()
        ops.muon_step_(p, g, buf, plan, lr, momentum=mu, weight_decay=wd,
                       nesterov=nesterov)
        # u as the kernel has it: a rounding or two of u are noise too
        u = mu * was + g.float()
        u = g.float() + mu * u if nesterov else u
        for start, rows, cols in matrices:
            part = slice(start, start + rows * cols)
            scale = lr * max(1.0, rows / cols) ** 0.5
            ref_u = u[part].view(rows, cols)
            plain, ref = plain_error(ref_u)
            want = before[part] * (1 - lr * wd) - scale * ref.reshape(-1)
            bound = scale * (4 * plain + input_roundings(ref_u)) \
                + 8 * 2.0 ** -24 * float(want.norm())
            assert float((p[part].double() - want).norm()) <= bound, (
                rows, cols)


def check_moves(opt, before):
    """Every matrix of the plan has made the step that the definition makes
    of the momentum and gradients that lie in the buffers."""
    group = opt.param_groups[0]
    _, plan, grads, _ = opt._plans[0]
    u = grads.double() + group["momentum"] * opt.momentum_buf[
        :plan.total].double()
    keep = 1 - group["lr"] * group["weight_decay"]
    assert plan.matrices
    for (start, rows, cols), scale in zip(plan.matrices, plan.scales):
        part = slice(start, start + rows * cols)
        was, now = before[part].double(), opt.flatp.flat[part].double()
        step = (was * keep - now) / (group["lr"] * scale)
        want = factor(u[part].view(rows, cols)).reshape(-1)
        # four roundings of parameters, seen through lr
        bound = BOUND + 4 * 2.0 ** -24 * float(was.norm() + now.norm()) / (
            group["lr"] * scale)
        assert float((step - want).norm()) <= bound, (rows, cols)
        # and that is a step of all directions the gradient has
        assert float(want.norm()) >= 0.5


@pytest.mark.parametrize("capture", [False, True])
def test_training_moves_every_matrix(capture):
    torch.manual_seed(8)
    net = resnet18(num_classes=10, norm="layer").to(dev()).to(
        memory_format=torch.channels_last)
    gdp = GossipDataParallel(net, rank=0, world_size=1,
                             working_dtype=torch.bfloat16)
    opt = FusedMuon(gdp.flatp, lr=0.02, rest_lr=0.1, weight_decay=0.01,
                    steal_grads=True)
    x = torch.randn(4, 3, 64, 64, device=dev()).to(
        memory_format=torch.channels_last)
    y = torch.randint(0, 10, (4,), device=dev())

    def step():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = torch.nn.functional.cross_entropy(net(x), y)
        loss.backward()
        opt.step()
        opt.zero_grad()
        return loss.detach()

    # the last norm of a residual branch starts at 0: no gradient before it
    for _ in range(2):
        step()
    once = step
    if capture:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        once = graph.replay
    for _ in range(3):
        torch.cuda.synchronize()
        before = opt.flatp.flat.clone()
        x.normal_()
        once()
        torch.cuda.synchronize()
        check_moves(opt, before)
        n = gdp.flatp.n_cast
        assert torch.equal(gdp.flatp.shadow, gdp.flatp.flat[:n].bfloat16())
        # and the vectors
        assert bool((opt.flatp.flat[n:] != before[n:]).float().mean() > 0.9)
    gdp.shutdown()


def test_channels_last_weights_move_alike():
    """A convolution's matrix in another order of its columns: the same
    step, in that order."""
    torch.manual_seed(9)
    nets = [torch.nn.Sequential(torch.nn.Conv2d(24, 70, 3, bias=False),
                                torch.nn.Conv2d(70, 130, 5, bias=False))
            for _ in range(2)]
    nets[1].load_state_dict(nets[0].state_dict())
    nets[1].to(memory_format=torch.channels_last)
    opts = [FusedMuon(FlatParams(net.to(dev()), flatten_grads=True), lr=0.1)
            for net in nets]
    start = [p.detach().clone() for p in nets[0].parameters()]
    for p, q in zip(nets[0].parameters(), nets[1].parameters()):
        assert p.stride() != q.stride() and torch.equal(p, q)
        p.grad.normal_()
        q.grad.copy_(p.grad)
    # with a momentum of 0 before, u = (1 + mu) g, whose size does not count
    grads = [p.grad.detach().clone() for p in nets[0].parameters()]
    for opt in opts:
        opt.step()
    for p, q, s, g in zip(nets[0].parameters(), nets[1].parameters(), start,
                          grads):
        plain, ref = plain_error(g.flatten(1))
        scale = 0.1 * max(1.0, ref.shape[0] / ref.shape[1]) ** 0.5
        want = s.double() - scale * ref.view_as(s)
        bound = scale * (4 * plain + input_roundings(g.flatten(1))) \
            + 8 * 2.0 ** -24 * float(want.norm())
        for t in (p, q):
            assert float((t.detach().double() - want).norm()) <= bound
