"""Layer norm over the last dimension, fused with a residual and a ReLU.

``layer_norm`` is one kernel forward and, for the gradients of the rows and
of the weight and bias, two backward (``csrc/layer_norm_kernels.hip``).  It
has no running statistics: unlike a batch norm's, there is nothing in it
that gossip leaves different from rank to rank.
"""

from typing import Optional

import torch

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def layer_norm(
    x: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    eps: float = 1e-5,
    residual: Optional[torch.Tensor] = None,
    relu: bool = False,
) -> torch.Tensor:
    """``y = (x - mean) / sqrt(var + eps) * weight + bias``, mean and
    (biased) variance over the last dimension of ``x``; then
    ``+ residual``, then ``max(y, 0)`` if ``relu``.

    ``x`` is fp32, bf16 or fp16 of any shape and strides; ``y`` has its
    shape and dtype and is contiguous.  ``weight`` and ``bias`` are vectors
    over the last dimension, both fp32 or both of ``x``'s dtype, and may be
    left out; ``residual`` has ``x``'s shape and dtype.  Arithmetic is fp32
    throughout, rounded once.  Differentiable once in ``x``, ``weight``,
    ``bias`` and ``residual``, on the device in reverse mode only (a dual
    tensor is refused, and so is a call under ``torch.jit.trace`` or
    ``make_fx``); the vectors' gradients are summed in a fixed order.  A row
    with a NaN or an infinity gives a row of NaN.  With ``relu`` a positive
    sum that the type rounds to zero is -0 on the device: its gradient passes.
    """
    if x.dtype not in _DTYPES:
        raise TypeError(f"layer_norm: x must be fp32, bf16 or fp16, got "
                        f"{x.dtype}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 1 << 30:
        raise ValueError("layer_norm: x needs a last dimension of 1 to 2^30, "
                         f"got shape {tuple(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps must not be negative, got {eps}")
    cols = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dtype != torch.float32 and t.dtype != x.dtype:
            raise TypeError(f"layer_norm: {name} must be fp32 or {x.dtype}, "
                            f"got {t.dtype}")
        if t.shape != (cols,):
            raise ValueError(f"layer_norm: {name} must have shape ({cols},), "
                             f"got {tuple(t.shape)}")
        if t.device != x.device:
            raise ValueError(f"layer_norm: {name} is on {t.device}, x on "
                             f"{x.device}")
    if weight is not None and bias is not None and \
            weight.dtype != bias.dtype:
        raise TypeError("layer_norm: weight and bias must have one dtype, "
                        f"got {weight.dtype} and {bias.dtype}")
    if residual is not None and (
        residual.shape != x.shape or residual.dtype != x.dtype
        or residual.device != x.device
    ):
        raise ValueError("layer_norm: the residual must have x's shape, "
                         "dtype and device")

    if not x.is_cuda:
        # PyTorch reference (also the numerics oracle in tests)
        y = torch.nn.functional.layer_norm(
            x.float(), (cols,), None if weight is None else weight.float(),
            None if bias is None else bias.float(), eps,
        )
        if residual is not None:
            y = y + residual.float()
        return (torch.relu(y) if relu else y).to(x.dtype)

    from . import _ext_for

    return _ext_for(x).layer_norm(
        x, weight if weight is None else weight.contiguous(),
        bias if bias is None else bias.contiguous(), eps, residual, relu,
    )
