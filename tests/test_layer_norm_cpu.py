"""Layer norm on the CPU: the reference path against 64 bits, refusals, and
the modules and models that use it."""

import pytest
import torch

from stochastic_gradient_push_amd import ops
from stochastic_gradient_push_amd.models import resnet18
from stochastic_gradient_push_amd.models.layers import (
    FusedBatchNorm2d,
    FusedLayerNorm,
    FusedLayerNorm2d,
)


def oracle(x, w, b, eps, res=None, relu=False):
    x = x.double()
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(var + eps)
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    if res is not None:
        y = y + res.double()
    return torch.relu(y) if relu else y


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("relu", [False, True])
def test_reference_path(dtype, residual, relu):
    torch.manual_seed(0)
    x = torch.randn(3, 5, 37).to(dtype)
    w, b = torch.randn(37), torch.randn(37)
    res = torch.randn(3, 5, 37).to(dtype) if residual else None
    y = ops.layer_norm(x, w, b, 1e-5, res, relu)
    assert y.dtype == dtype and y.shape == x.shape
    ref = oracle(x, w, b, 1e-5, res, relu)
    # fp32 arithmetic over 37 values, one rounding to the type at the end
    tol = 64 * 2.0 ** -24 * 8 + torch.finfo(dtype).eps / 2 * ref.abs()
    assert bool(((y.double() - ref).abs() <= tol).all())


def test_weight_and_bias_are_optional():
    x = torch.randn(4, 16)
    for w in (None, torch.randn(16)):
        for b in (None, torch.randn(16)):
            y = ops.layer_norm(x, w, b)
            assert torch.allclose(y.double(), oracle(x, w, b, 1e-5),
                                  atol=1e-5)


def test_no_rows():
    assert ops.layer_norm(torch.empty(0, 8)).shape == (0, 8)


@pytest.mark.parametrize("call,error", [
    (lambda x: ops.layer_norm(x.double()), TypeError),
    (lambda x: ops.layer_norm(x.long()), TypeError),
    (lambda x: ops.layer_norm(torch.tensor(1.0)), ValueError),
    (lambda x: ops.layer_norm(x[:, :0]), ValueError),
    (lambda x: ops.layer_norm(x, eps=-1e-5), ValueError),
    (lambda x: ops.layer_norm(x, eps=float("nan")), ValueError),
    (lambda x: ops.layer_norm(x, torch.ones(7)), ValueError),
    (lambda x: ops.layer_norm(x, torch.ones(1, 8)), ValueError),
    (lambda x: ops.layer_norm(x, bias=torch.ones(9)), ValueError),
    (lambda x: ops.layer_norm(x, torch.ones(8).half()), TypeError),
    (lambda x: ops.layer_norm(x, torch.ones(8).double()), TypeError),
    (lambda x: ops.layer_norm(x.half(), torch.ones(8),
                              torch.ones(8).half()), TypeError),
    (lambda x: ops.layer_norm(x, residual=torch.ones(8)), ValueError),
    (lambda x: ops.layer_norm(x, residual=torch.ones(4, 8).half()),
     ValueError),
    (lambda x: ops.layer_norm(x, torch.ones(8, device="meta")), ValueError),
])
def test_refusals(call, error):
    with pytest.raises(error, match="layer_norm"):
        call(torch.randn(4, 8))


def test_module_matches_stock():
    torch.manual_seed(1)
    for shape in (24, (6, 4)):
        ours, stock = FusedLayerNorm(shape), torch.nn.LayerNorm(shape)
        stock.load_state_dict(ours.state_dict())
        x = torch.randn(2, 3, 6, 4).flatten(-2) if shape == 24 \
            else torch.randn(2, 3, 6, 4)
        assert torch.allclose(ours(x), stock(x), atol=1e-6)
    bare = FusedLayerNorm(24, elementwise_affine=False)
    assert not list(bare.parameters())
    assert bare(torch.randn(2, 24)).shape == (2, 24)
    with pytest.raises(ValueError, match="FusedLayerNorm"):
        bare(torch.randn(2, 23))


def test_module_refuses_another_residual():
    # as many values in a row, but not the input's
    with pytest.raises(ValueError, match="residual"):
        FusedLayerNorm((4, 6))(torch.randn(3, 4, 6), torch.randn(3, 6, 4))


@pytest.mark.parametrize("channels_last", [False, True])
def test_module_2d(channels_last):
    torch.manual_seed(2)
    norm = FusedLayerNorm2d(12, relu=True)
    torch.nn.init.normal_(norm.weight)
    torch.nn.init.normal_(norm.bias)
    x, res = torch.randn(2, 12, 5, 3), torch.randn(2, 12, 5, 3)
    if channels_last:
        x = x.contiguous(memory_format=torch.channels_last)
    ref = oracle(x.permute(0, 2, 3, 1), norm.weight, norm.bias, 1e-5,
                 res.permute(0, 2, 3, 1), True).permute(0, 3, 1, 2)
    y = norm(x, res)
    assert y.is_contiguous(memory_format=torch.channels_last)
    assert torch.allclose(y.double(), ref, atol=1e-5)
    with pytest.raises(ValueError, match="FusedLayerNorm2d"):
        norm(x[:, :11])
    with pytest.raises(ValueError, match="FusedLayerNorm2d"):
        norm(x[0])


def test_resnet_with_layer_norm():
    torch.manual_seed(3)
    net = resnet18(num_classes=7, norm="layer")
    kinds = {type(m) for m in net.modules()}
    assert FusedLayerNorm2d in kinds and FusedBatchNorm2d not in kinds
    assert not list(net.buffers())  # nothing that gossip does not mix
    # zero-init of each residual branch's last norm, as for batch norm
    assert bool((net.layer1[0].bn2.weight == 0).all())
    x = torch.randn(2, 3, 32, 32)
    net.eval()
    y = net(x)
    assert y.shape == (2, 7)
    # a sample's output does not depend on its batch
    assert torch.allclose(net(x[:1]), y[:1], atol=1e-5)
    y.sum().backward()
    assert all(p.grad is not None for p in net.parameters())


def test_resnet_norms_that_were_there():
    assert any(isinstance(m, FusedBatchNorm2d)
               for m in resnet18(norm="fused").modules())
    with pytest.raises(ValueError):
        resnet18(norm="nosuch")
