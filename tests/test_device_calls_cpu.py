"""What layer norm, Newton-Schulz and the Muon step refuse before they touch
the device: calls that kernels past PyTorch's dispatcher cannot serve.  The
refusals come first, so that no device is needed to see them."""

import pytest
import torch

from stochastic_gradient_push_amd import ops

ext = ops._load_extension()
needs_ext = pytest.mark.skipif(ext is None, reason="extension not built")

COEF = (3.4445, -4.7750, 2.0315)


class Wrapper(torch.Tensor):
    """Says that it is on the device, and has no memory."""

    @staticmethod
    def __new__(cls, *shape, dtype=torch.float32):
        return torch.Tensor._make_wrapper_subclass(
            cls, shape, dtype=dtype, device="cuda:0")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        if func is torch.ops.aten.detach.default:
            return args[0]
        raise NotImplementedError(func)


def fake(*shape):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        return torch.empty(*shape, device="cuda:0")


@needs_ext
@pytest.mark.filterwarnings("ignore:Accessing the data pointer")
@pytest.mark.parametrize("make", [Wrapper, fake])
def test_tensors_without_memory(make):
    none = "no memory"
    x, v = make(4, 8), make(8)
    for args in ((x, None, None, 1e-5, None, False),
                 (x, v, v, 1e-5, x, True)):
        with pytest.raises(RuntimeError, match=none):
            ext.layer_norm(*args)
    with pytest.raises(RuntimeError, match=none):
        ext.layer_norm_fwd(x, v, None, None, 1e-5, False, True)
    with pytest.raises(RuntimeError, match=none):
        ext.layer_norm_bwd(x, x, None, v, make(4), make(4), True, True,
                           False, True, False)
    with pytest.raises(RuntimeError, match=none):
        ext.newton_schulz(make(1, 4, 6), 5, 5, 1, *COEF, 4.0, 1e-7)
    tables, layout = ext.muon_plan([(0, 4, 6, 1.0)], 24)
    with pytest.raises(RuntimeError, match=none):
        ext.muon_step_(make(24), make(24), make(24), None, tables, layout,
                       24, make(1), 0.9, 0.0, 1.0, True, 5, 1, *COEF, 4.0,
                       1e-7)


@needs_ext
def test_public_entry_points_refuse_them_too():
    with pytest.raises(RuntimeError, match="no memory"):
        ops.layer_norm(Wrapper(4, 8))


@needs_ext
@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_tangents():
    """A dual tensor is refused for its tangent before it is refused for
    where it lies."""
    import torch.autograd.forward_ad as fwd

    none = "forward-mode"
    x, v = torch.randn(4, 8), torch.randn(8)
    tables, layout = ext.muon_plan([(0, 4, 6, 1.0)], 24)
    with fwd.dual_level():
        for i in range(4):
            args = [x, v, v, x.clone()]
            args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError, match=none):
                ext.layer_norm(*args[:3], 1e-5, args[3], False)
        with pytest.raises(RuntimeError, match=none):
            ext.newton_schulz(fwd.make_dual(torch.ones(1, 4, 6),
                                            torch.ones(1, 4, 6)),
                              5, 5, 1, *COEF, 4.0, 1e-7)
        for i in range(5):
            args = [torch.ones(24) for _ in range(4)] + [torch.ones(1)]
            args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            p, g, buf, shadow, lr = args
            with pytest.raises(RuntimeError, match=none):
                ext.muon_step_(p, g, buf, shadow, tables, layout, 24, lr,
                               0.9, 0.0, 1.0, True, 5, 1, *COEF, 4.0, 1e-7)
        # the host's path differentiates
        y = ops.layer_norm(fwd.make_dual(x, torch.ones_like(x) * x), v)
        assert fwd.unpack_dual(y).tangent is not None


@needs_ext
@pytest.mark.filterwarnings("ignore")
def test_tracing():
    from torch.fx.experimental.proxy_tensor import make_fx

    tables, layout = ext.muon_plan([(0, 4, 6, 1.0)], 24)

    def norm(t):
        return ext.layer_norm(t, None, None, 1e-5, None, False)

    def orthogonal(t):
        return ext.newton_schulz(t[None], 5, 5, 1, *COEF, 4.0, 1e-7)

    def step(t):
        t = t.flatten()
        ext.muon_step_(t, t, t, None, tables, layout, 24, t[:1], 0.9, 0.0,
                       1.0, True, 5, 1, *COEF, 4.0, 1e-7)
        return t

    x = torch.randn(4, 6)
    for f in (norm, orthogonal, step):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, (x,))
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(f)(x)
    # the host's path can be
    traced = torch.jit.trace(ops.layer_norm, (x,))
    y = torch.randn(4, 6)
    assert torch.allclose(traced(y), ops.layer_norm(y), atol=1e-6)
