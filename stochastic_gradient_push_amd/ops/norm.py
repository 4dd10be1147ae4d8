"""Layer norm over the last dimension, fused with a residual and a ReLU.

``layer_norm`` is one kernel forward and, for the gradients of the rows and
of the weight and bias, two backward (``csrc/layer_norm_kernels.hip``).  It
has no running statistics: unlike a batch norm's, there is nothing in it
that gossip leaves different from rank to rank.
"""

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as a matrix of its last dimension's rows.  A view where the
    rows are contiguous and evenly spaced, a copy elsewhere."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.shape[1] == 1 or t.stride(1) == 1 else t.contiguous()


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, relu):
        from . import _ext_for

        x2d = _rows(x)
        y, mean, rstd = _ext_for(x).layer_norm_fwd(
            x2d, weight, bias, None if residual is None else _rows(residual),
            eps, relu, True,
        )
        y = y.view(x.shape)
        ctx.save_for_backward(x, weight, mean, rstd, y if relu else None)
        vector = weight if weight is not None else bias
        ctx.vectors_fp32 = (
            vector is not None and vector.dtype == torch.float32
        )
        ctx.relu = relu
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        from . import _ext_for

        x, weight, mean, rstd, y = ctx.saved_tensors
        need_dx, need_dw, need_db, need_dres = ctx.needs_input_grad[:4]
        dx = dw = db = dres = None
        # without a ReLU the residual's gradient is dy itself
        masked = need_dres and ctx.relu
        if need_dx or need_dw or need_db or masked:
            dx, dres, dw, db = _ext_for(x).layer_norm_bwd(
                _rows(dy), _rows(x), None if y is None else _rows(y), weight,
                mean, rstd, ctx.vectors_fp32, need_dx, masked, need_dw,
                need_db,
            )
            dx = dx.view(x.shape) if need_dx else None
            dres = dres.view(x.shape) if masked else None
        if need_dres and not masked:
            dres = dy
        return dx, dw, db, dres, None, None


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
    ``bias`` and ``residual``; the vectors' gradients are summed in a fixed
    order.  A row with a NaN or an infinity gives a row of NaN.
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

    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and any(
        t is not None and t.requires_grad
        for t in (x, weight, bias, residual)
    ):
        return _LayerNormFn.apply(x, weight, bias, residual, float(eps),
                                  bool(relu))
    from . import _ext_for

    y, _, _ = _ext_for(x).layer_norm_fwd(
        _rows(x), weight, bias, None if residual is None else _rows(residual),
        eps, relu, False,
    )
    return y.view(x.shape)
