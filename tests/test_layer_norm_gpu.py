"""Layer norm kernels against the formulas in 64 bits.

Bounds count roundings.  Let u = 2^-24.  A row's sums are trees over at most
32 values per thread and ten levels, so a mean is off by at most 48 u times
the mean of |x|, and likewise the other sums; the rest is a handful of
operations on values of the sizes that appear in each bound.  Every output
is rounded once to its type: eps / 2 of its value.
"""

import pytest
import torch

from stochastic_gradient_push_amd import ops
from stochastic_gradient_push_amd.models.layers import (
    FusedLayerNorm,
    FusedLayerNorm2d,
)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def dev():
    return torch.device("cuda", 0)


def half_step(t, dtype):
    # half a step of the type; below its normal numbers half the smallest
    fi = torch.finfo(dtype)
    return fi.eps / 2 * t.abs() + fi.smallest_normal * fi.eps / 2


def formulas(x, w, b, eps, res, relu, dy):
    """All outputs and gradients in 64 bits, with a bound for each."""
    # the vectors' gradients have the vectors' type (fp16: half a step of a
    # db of 8 is 2^-11 * 8 = 4e-3)
    dtype = x.dtype
    wtype = next((t.dtype for t in (w, b) if t is not None), torch.float32)
    x = x.double()
    cols = x.shape[-1]
    w = torch.ones(cols, device=x.device).double() if w is None \
        else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    hat = (x - mean) * rstd
    # the centred value: the mean's error and its own rounding
    dhat = 64 * U * (x.abs().mean(-1, keepdim=True) + x.abs()) * rstd \
        + 64 * U * hat.abs()
    z = hat * w + b
    tz = dhat * w.abs() + 8 * U * ((hat * w).abs() + b.abs())
    if res is not None:
        z = z + res.double()
        tz = tz + 4 * U * res.double().abs()
    y = torch.relu(z) if relu else z
    out = {"y": (y, tz + half_step(y, dtype))}
    if dy is None:
        return out
    g = dy.double()
    if relu:
        g = torch.where(z > 0, g, torch.zeros_like(g))
    gw = g * w
    m0 = gw.mean(-1, keepdim=True)
    m1 = (gw * hat).mean(-1, keepdim=True)
    dx = rstd * (gw - m0 - hat * m1)
    a0 = gw.abs().mean(-1, keepdim=True)
    a1 = (gw * hat).abs().mean(-1, keepdim=True)
    e1 = 64 * U * a1 + (gw.abs() * dhat).mean(-1, keepdim=True)
    tdx = rstd * (64 * U * (gw.abs() + a0) + hat.abs() * e1 + dhat * m1.abs()
                  + 16 * U * (hat * m1).abs()) + 8 * U * dx.abs()
    out["dx"] = (dx, tdx + half_step(dx, dtype))
    # a column's sum: at most `chain` additions after one another
    chain = min(x.shape[0], 512) + 64
    dw, db = (g * hat).sum(0), g.sum(0)
    out["dw"] = (dw, chain * U * (g * hat).abs().sum(0)
                 + (g.abs() * dhat).sum(0) + half_step(dw, wtype))
    out["db"] = (db, chain * U * g.abs().sum(0) + half_step(db, wtype))
    out["dres"] = (g, torch.zeros_like(g))
    return out


def check(got, want, name):
    ref, bound = want
    assert got.shape == ref.shape, name
    err = (got.double() - ref).abs()
    bad = err > bound
    assert not bool(bad.any()), (
        f"{name}: {int(bad.sum())} of {bad.numel()} off, worst "
        f"{float(err.max()):.3e}, at most {float((err / bound).max()):.2f} "
        "times its bound"
    )


def inputs(rows, cols, dtype, wtype, residual, relu, seed=0, offset=0.0):
    g = torch.Generator(device=dev()).manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device=dev())

    x = (randn(rows, cols) * (0.25 + randn(rows, 1).abs()) + offset).to(dtype)
    w, b = (1 + 0.5 * randn(cols)).to(wtype), randn(cols).to(wtype)
    res = randn(rows, cols).to(dtype) if residual else None
    dy = randn(rows, cols).to(dtype)
    if relu:
        # no gradient where rounding decides the side of the border
        z = formulas(x, w, b, 1e-5, res, False, None)["y"][0]
        dy = torch.where(z.abs() < 1e-2, torch.zeros_like(dy), dy)
    return x, w, b, res, dy


def run(x, w, b, res, relu, dy, eps=1e-5):
    leaves = {"dx": x, "dw": w, "db": b, "dres": res}
    leaves = {k: v.detach().clone().requires_grad_(True)
              for k, v in leaves.items() if v is not None}
    y = ops.layer_norm(leaves["dx"], leaves.get("dw"), leaves.get("db"), eps,
                       leaves.get("dres"), relu)
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    out = dict(zip(leaves, grads))
    out["y"] = y.detach()
    return out


# every row group and its borders, in 16-byte vectors of 8 (and 4) values
COLS = [1, 2, 7, 8, 9, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513,
        1000, 1024, 1025, 2047, 2048, 2049, 4097, 8192, 8200, 16384, 16391]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_widths(cols, dtype):
    rows = 67
    x, w, b, res, dy = inputs(rows, cols, dtype, torch.float32, True, True,
                              seed=cols)
    got = run(x, w, b, res, True, dy)
    want = formulas(x, w, b, 1e-5, res, True, dy)
    for name in want:
        check(got[name], want[name], name)


@pytest.mark.parametrize("cols", [16392, 32768, 32776, 50001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_beyond_registers(cols, dtype):
    x, w, b, res, dy = inputs(5, cols, dtype, torch.float32, True, True)
    got = run(x, w, b, res, True, dy)
    want = formulas(x, w, b, 1e-5, res, True, dy)
    for name in want:
        check(got[name], want[name], name)


@pytest.mark.parametrize("rows", [1, 2, 3, 31, 33, 2049, 20000])
@pytest.mark.parametrize("cols", [24, 256, 768])
def test_row_counts(rows, cols):
    x, w, b, res, dy = inputs(rows, cols, torch.bfloat16, torch.float32,
                              False, False, seed=rows)
    got = run(x, w, b, res, False, dy)
    want = formulas(x, w, b, 1e-5, res, False, dy)
    for name in got:
        check(got[name], want[name], name)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("wtype", ["own", "fp32"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_forms(dtype, wtype, relu, residual):
    wtype = dtype if wtype == "own" else torch.float32
    x, w, b, res, dy = inputs(130, 300, dtype, wtype, residual, relu)
    got = run(x, w, b, res, relu, dy)
    want = formulas(x, w, b, 1e-5, res, relu, dy)
    for name in got:
        check(got[name], want[name], name)
    assert got["dw"].dtype == wtype and got["db"].dtype == wtype


@pytest.mark.parametrize("with_w", [False, True])
@pytest.mark.parametrize("with_b", [False, True])
def test_weight_and_bias_are_optional(with_w, with_b):
    x, w, b, _, dy = inputs(50, 100, torch.float16, torch.float16, False,
                            False)
    w, b = w if with_w else None, b if with_b else None
    got = run(x, w, b, None, False, dy)
    want = formulas(x, w, b, 1e-5, None, False, dy)
    for name in got:
        check(got[name], want[name], name)


def test_mean_far_from_zero():
    # the variance is that of the centred values, not a difference of
    # squares (which would lose all of it here: 1e4^2 * 2^-24 = 6)
    x, w, b, _, dy = inputs(64, 1024, torch.float32, torch.float32, False,
                            False, offset=1e4)
    got = run(x, w, b, None, False, dy)
    want = formulas(x, w, b, 1e-5, None, False, dy)
    for name in got:
        check(got[name], want[name], name)


def test_constant_rows():
    # variance 0: hat = 0, y = b, and rstd = 1 / sqrt(eps)
    x = torch.full((9, 96), 3.0, device=dev())
    w, b = torch.randn(96, device=dev()), torch.randn(96, device=dev())
    got = run(x, w, b, None, False, torch.randn(9, 96, device=dev()))
    assert torch.equal(got["y"], b.expand(9, 96))
    assert bool((got["dw"] == 0).all())
    assert bool(torch.isfinite(got["dx"]).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("cols", [100, 3000, 40000])
def test_a_bad_row_stays_alone(bad, cols):
    x = torch.randn(6, cols, device=dev())
    clean = ops.layer_norm(x)
    x[2, cols // 2] = bad
    y = ops.layer_norm(x)
    assert bool(torch.isnan(y[2]).all())
    keep = torch.arange(6, device=dev()) != 2
    assert torch.equal(y[keep], clean[keep])
    # a ReLU keeps the NaN
    assert bool(torch.isnan(ops.layer_norm(x, relu=True)[2]).all())


def test_strides():
    base = torch.randn(40, 6, 80, device=dev()).to(torch.bfloat16)
    w, b = torch.randn(64, device=dev()), torch.randn(64, device=dev())
    views = [
        base[:, 0, 3:67],               # rows far apart, off by 3 elements
        base[:, :, 1:65],               # rows of two distances
        base[::3, 2, :64],
        base.permute(2, 1, 0)[:64].permute(2, 1, 0),
        base[0, 0, :64].expand(7, 64),  # one row, repeated
        base[:, :, :64].transpose(0, 1),
    ]
    for i, v in enumerate(views):
        plain = v.contiguous().requires_grad_(True)
        view = v.detach().requires_grad_(True)
        dy = torch.randn_like(plain)
        y, ref = (ops.layer_norm(t, w, b, residual=t) for t in (view, plain))
        assert torch.equal(y, ref), i
        got, = torch.autograd.grad(y, view, dy)
        want, = torch.autograd.grad(ref, plain, dy)
        assert torch.equal(got, want), i
        # a gradient of any strides
        y = ops.layer_norm(view, w, b)
        got, = torch.autograd.grad(y.sum(), view)
        want, = torch.autograd.grad(
            ops.layer_norm(plain, w, b), plain, torch.ones_like(plain))
        assert torch.equal(got, want), i


def test_shared_leaves():
    # the same tensor as rows and residual, the same weight twice
    x, w, b, _, dy = inputs(33, 72, torch.float32, torch.float32, False,
                            False)
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = ops.layer_norm(ops.layer_norm(xs, ws, b, residual=xs), ws, b)
    got = torch.autograd.grad(y, (xs, ws), dy)
    xd, wd = x.double().requires_grad_(True), w.double().requires_grad_(True)
    ln = torch.nn.functional.layer_norm
    t = ln(xd, (72,), wd, b.double()) + xd
    want = torch.autograd.grad(ln(t, (72,), wd, b.double()), (xd, wd),
                               dy.double())
    for a, r in zip(got, want):
        assert float((a.double() - r).abs().max()) <= \
            1024 * U * float(r.abs().max())


def test_gradient_against_differences():
    # along a direction v: (f(x + h v) - f(x - h v)) / 2h, off by O(h^2)
    # (1e-4 of unit-sized values) and by rounding u / h (6e-6)
    x, w, b, res, dy = inputs(16, 200, torch.float32, torch.float32, True,
                              False)
    got = run(x, w, b, res, False, dy)
    h = 1e-2
    for name, i in (("dx", 0), ("dw", 1), ("db", 2), ("dres", 3)):
        args = [x, w, b, res]
        v = torch.randn_like(args[i])
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[i] = args[i] + sign * h * v
            y = ops.layer_norm(moved[0], moved[1], moved[2], 1e-5, moved[3])
            ends.append(y.double())
        diff = float(((ends[0] - ends[1]) / (2 * h) * dy).sum())
        want = float((got[name].double() * v).sum())
        scale = float((got[name].double() * v).norm()) + 1
        assert abs(diff - want) <= 1e-2 * scale, name


def test_only_what_is_asked_for():
    x, w, b, res, dy = inputs(64, 96, torch.bfloat16, torch.float32, True,
                              True)
    full = run(x, w, b, res, True, dy)
    names = ["dx", "dw", "db", "dres"]
    for name in names:
        args = [t.detach().clone() for t in (x, w, b, res)]
        args[names.index(name)].requires_grad_(True)
        y = ops.layer_norm(args[0], args[1], args[2], 1e-5, args[3], True)
        got, = torch.autograd.grad(y, args[names.index(name)], dy)
        assert torch.equal(got, full[name]), name
    with torch.no_grad():
        y = ops.layer_norm(x, w, b, 1e-5, res, True)
    assert torch.equal(y, full["y"]) and not y.requires_grad


def test_same_call_same_bits():
    x, w, b, res, dy = inputs(5000, 192, torch.bfloat16, torch.float32, True,
                              True)
    first = run(x, w, b, res, True, dy)
    for _ in range(3):
        again = run(x, w, b, res, True, dy)
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_rows_beyond_32_bits():
    rows, cols = (1 << 21) + 5, 1032
    x = torch.zeros(rows, cols, device=dev(), dtype=torch.bfloat16)
    assert x.numel() > 1 << 31
    some, w, b, _, dy = inputs(4, cols, torch.bfloat16, torch.float32, False,
                               False)
    x[-4:] = some
    leaf = x.requires_grad_(True)
    g = torch.zeros_like(x)
    g[-4:] = dy
    y = ops.layer_norm(leaf, w, b)
    dx, = torch.autograd.grad(y, leaf, g)
    want = run(some, w, b, None, False, dy)
    assert torch.equal(y[-4:], want["y"])
    assert torch.equal(dx[-4:], want["dx"])
    assert bool((dx[:-4] == 0).all())
    assert torch.equal(y[0], b.to(torch.bfloat16))


def test_no_rows():
    x = torch.empty(0, 64, device=dev(), requires_grad=True)
    w = torch.ones(64, device=dev(), requires_grad=True)
    y = ops.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == dx.shape == (0, 64) and bool((dw == 0).all())


def test_refusals():
    x = torch.randn(4, 8, device=dev())
    with pytest.raises(ValueError, match="layer_norm"):
        ops.layer_norm(x, torch.ones(8))  # on the host
    with pytest.raises(ValueError, match="layer_norm"):
        ops.layer_norm(x, residual=torch.ones(4, 8))
    ext = ops._ext_for(x)
    with pytest.raises(RuntimeError, match="contiguous rows"):
        ext.layer_norm_fwd(x.t(), None, None, None, 1e-5, False, False)
    with pytest.raises(RuntimeError, match="shape"):
        ext.layer_norm_fwd(x, None, None, x[:2], 1e-5, False, False)
    with pytest.raises(RuntimeError, match="statistics"):
        ext.layer_norm_bwd(x, x, None, None, x[0], x[0], True, True, False,
                           False, False)
    # differentiable once
    z = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(ops.layer_norm(z).square().sum(), z,
                             create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_side_stream():
    x, w, b, res, dy = inputs(3000, 512, torch.bfloat16, torch.float32, True,
                              True)
    want = run(x, w, b, res, True, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, w, b, res, True, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[k], want[k]) for k in want)


def test_captured_and_replayed():
    x, w, b, res, dy = inputs(700, 256, torch.bfloat16, torch.float32, True,
                              True)
    sx, sdy = x.clone().requires_grad_(True), dy.clone()
    sw = w.clone().requires_grad_(True)

    def step():
        y = ops.layer_norm(sx, sw, b, 1e-5, res, True)
        dx, dw = torch.autograd.grad(y, (sx, sw), sdy)
        return y.detach(), dx, dw

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        nx = x + 0.5 * k
        ndy = dy * (1 + k)
        with torch.no_grad():
            sx.copy_(nx)
            sdy.copy_(ndy)
        graph.replay()
        torch.cuda.synchronize()
        want = run(nx, w, b, res, True, ndy)
        for a, name in zip(out, ("y", "dx", "dw")):
            assert torch.equal(a, want[name]), (k, name)


def test_module_2d_under_autocast():
    torch.manual_seed(0)
    norm = FusedLayerNorm2d(48, relu=True).to(dev())
    x = torch.randn(2, 48, 7, 5, device=dev()).to(torch.bfloat16)
    res = torch.randn_like(x)
    for layout in (torch.channels_last, torch.contiguous_format):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = norm(x.contiguous(memory_format=layout), res)
        assert y.dtype == torch.bfloat16
        assert y.is_contiguous(memory_format=torch.channels_last)
        flat = x.permute(0, 2, 3, 1).reshape(-1, 48)
        want = formulas(flat, norm.weight.detach(), norm.bias.detach(), 1e-5,
                        res.permute(0, 2, 3, 1).reshape(-1, 48), True, None)
        check(y.detach().permute(0, 2, 3, 1).reshape(-1, 48), want["y"], "y")


def test_module_over_two_dimensions():
    norm = FusedLayerNorm((6, 10)).to(dev())
    x = torch.randn(3, 4, 6, 10, device=dev(), requires_grad=True)
    y = norm(x)
    ref = torch.nn.functional.layer_norm(x.double(), (6, 10))
    assert float((y.double() - ref).abs().max()) <= 256 * U * 4
    y.sum().backward()
    assert norm.weight.grad.shape == (6, 10)


@pytest.mark.parametrize("rows,cols", [(100352, 256), (300_000, 24),
                                       (40_000, 1000)])
def test_fp16_rows_fill_the_card(rows, cols):
    # as many blocks as the card holds of this very kernel, each with a row
    # of partial sums
    x, w, b, res, dy = inputs(rows, cols, torch.float16, torch.float32, True,
                              True)
    got = run(x, w, b, res, True, dy)
    want = formulas(x, w, b, 1e-5, res, True, dy)
    for name in want:
        check(got[name], want[name], name)


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd

    x, res = torch.randn(4, 8, device=dev()), torch.randn(4, 8, device=dev())
    w, b = torch.randn(8, device=dev()), torch.randn(8, device=dev())
    args = [x, w, b, res]
    with fwd.dual_level():
        for i in range(4):
            some = list(args)
            some[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            for grad in (False, True):
                some[0] = some[0] if i == 0 else x.clone().requires_grad_(grad)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    ops.layer_norm(some[0], some[1], some[2],
                                   residual=some[3])
        # a tangent that comes with the output's gradient
        leaf = x.clone().requires_grad_(True)
        y = ops.layer_norm(leaf, w, b)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, leaf, fwd.make_dual(res, x))
        # one that was left behind is no hindrance
        dual = fwd.make_dual(x, res)
        assert torch.equal(ops.layer_norm(dual.detach(), w, b),
                           ops.layer_norm(x, w, b))
    for call in (
        lambda: torch.func.jvp(lambda t: ops.layer_norm(t, w, b), (x,),
                               (res,)),
        lambda: torch.func.vmap(lambda t: ops.layer_norm(t, w, b))(x),
        lambda: torch.func.grad(lambda t: ops.layer_norm(t, w, b).sum())(x),
    ):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.filterwarnings("ignore")
def test_tracing_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.randn(4, 8, device=dev())
    for grad in (False, True):
        leaf = x.clone().requires_grad_(grad)
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(lambda t: ops.layer_norm(t), (leaf,))
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda t: ops.layer_norm(t))(x)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(FusedLayerNorm2d(6).to(dev()),
                        (torch.randn(2, 6, 3, 3, device=dev()),))


@pytest.mark.parametrize("shape", [(6, 40), (3, 5, 40)])
def test_output_changed_in_place(shape):
    torch.manual_seed(0)
    x = torch.randn(*shape, device=dev())
    w = torch.randn(40, device=dev())
    dy = torch.randn_like(x)

    def grads(change):
        xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = change(ops.layer_norm(xs, ws, residual=x))
        return [y.detach(), *torch.autograd.grad(y, (xs, ws), dy)]

    for inplace, other in (
        (lambda y: y.mul_(2.0), lambda y: y * 2.0),
        (lambda y: torch.relu_(y), torch.relu),
        (lambda y: y.add_(x), lambda y: y + x),
    ):
        assert all(torch.equal(a, b)
                   for a, b in zip(grads(inplace), grads(other)))
    # the ReLU's output is needed for its gradient
    xs = x.clone().requires_grad_(True)
    y = ops.layer_norm(xs, relu=True).mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_modules_outputs_changed_in_place():
    torch.manual_seed(1)
    relu = torch.nn.ReLU(inplace=True)
    for norm, x in ((FusedLayerNorm(24), torch.randn(5, 24)),
                    (FusedLayerNorm((4, 6)), torch.randn(5, 4, 6)),
                    (FusedLayerNorm2d(24), torch.randn(2, 24, 3, 5))):
        norm, x = norm.to(dev()), x.to(dev()).requires_grad_(True)
        y = relu(norm(x))
        want = torch.relu(norm(x))
        assert torch.equal(y, want)
        got, = torch.autograd.grad(y.sum(), x)
        ref, = torch.autograd.grad(want.sum(), x)
        assert torch.equal(got, ref)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [24, 600, 3000, 16500])
def test_constant_long_rows_and_short_ones(cols, dtype):
    # a mean that is off shows undiminished where the variance is 0
    x = torch.full((2, cols), 0.1, device=dev()).to(dtype)
    y = ops.layer_norm(x)
    assert float(y.abs().max()) <= 48 * U * 0.1 / 1e-5 ** 0.5


def test_a_constant_row_of_millions():
    # 2^16 values a thread: added one after another in 32 bits the mean was
    # off by up to 2^16 * 2^-25 of itself
    cols = (1 << 26) + 5
    x = torch.full((1, cols), 0.1, device=dev())
    bound = 48 * U * 0.1 / 1e-5 ** 0.5
    y = ops.layer_norm(x)
    assert float(y.abs().max()) <= bound
    # the gradient's sums likewise: of equal values nothing is left
    leaf = x.requires_grad_(True)
    w = torch.full((cols,), 0.1, device=dev())
    dx, = torch.autograd.grad(ops.layer_norm(leaf, w), leaf,
                              torch.ones_like(x))
    assert float(dx.abs().max()) <= bound


def test_more_columns_than_a_launch_has_threads():
    # 16 threads a column of dw and of db in the sum over the blocks: 2^32
    cols = (1 << 27) + 3
    g = torch.Generator(device=dev()).manual_seed(0)
    x = torch.randn(1, cols, generator=g, device=dev())
    dy = torch.randn(1, cols, generator=g, device=dev())
    w, b = (torch.ones(cols, device=dev(), requires_grad=True)
            for _ in range(2))
    dw, db = torch.autograd.grad(ops.layer_norm(x, w, b), (w, b), dy)
    assert torch.equal(db, dy[0])
    mean = float(x.mean(dtype=torch.float64))
    var = float(((x.double() - mean) ** 2).mean())
    hat = (x[0].double() - mean) / (var + 1e-5) ** 0.5
    want = dy[0].double() * hat
    # the mean and the deviation: 24 roundings of values of size 1, as above
    bound = 8 * U * want.abs() + 64 * U * dy[0].double().abs()
    assert bool(((dw.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype,tiny", [(torch.float16, 2.0 ** -26),
                                        (torch.float16, 2.0 ** -25),
                                        (torch.bfloat16, 2.0 ** -135)])
@pytest.mark.parametrize("cols", [24, 600, 3000, 16500])
def test_relu_of_sums_that_round_to_zero(dtype, tiny, cols):
    # hat is 0, so a column's sum is its bias: positive and too small for
    # the type, negative likewise, zero
    x = torch.ones(3, cols, device=dev()).to(dtype)
    b = torch.tensor([tiny, -tiny, 0.0], device=dev()).repeat(cols // 3 + 1)
    b = b[:cols].contiguous()
    res = torch.zeros_like(x).requires_grad_(True)
    b.requires_grad_(True)
    y = ops.layer_norm(x, None, b, residual=res, relu=True)
    assert bool((y == 0).all())
    dy = torch.ones_like(y)
    dres, db = torch.autograd.grad(y, (res, b), dy)
    want = (b.detach() > 0).to(dtype)
    assert torch.equal(dres, want.expand(3, cols))
    assert torch.equal(db, 3.0 * want.float())
