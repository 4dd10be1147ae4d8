"""Orthogonalised updates: Newton-Schulz products, and the Muon step over a
flat parameter buffer (``csrc/muon_kernels.hip``).

``newton_schulz`` maps a matrix ``G = U S V^T`` to about ``U V^T`` by

    X = G / (|G|_F + eps);   steps times:  X = (a I + b A + c A^2) X,
                                           A = X X^T

(the Newton-Schulz iteration for a polar factor with a quintic instead of the
classic cubic).

``muon_step_`` is one optimiser step of every matrix in a flat buffer (the
layout of :class:`~stochastic_gradient_push_amd.ops.flat.FlatParams`), all
shapes together in one launch per product; what lies between the matrices
gets plain momentum SGD.
"""

import math
from functools import lru_cache
from typing import Optional, Sequence, Tuple

import torch

#: slope at zero as large as convergence into [0.68, 1.21] allows; from the
#: publication of the method: K. Jordan et al., "Muon: An optimizer for hidden
#: layers in neural networks", 2024, like the update's scale in a step
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


@lru_cache(maxsize=64)
def _growth(coefficients: Tuple[float, float, float], steps: int) -> float:
    """The most that one step multiplies a singular value with.  Raises
    where values of at most 1 do not stay below 2, or the polynomial leaves
    the range that the kernels hold it in."""
    a, b, c = coefficients
    if not all(math.isfinite(v) for v in coefficients):
        raise ValueError(f"newton_schulz: coefficients {coefficients} are "
                         "not finite")
    values, most, widest = [i / 1000 for i in range(1001)], 0.0, 1.0
    for _ in range(steps):
        factors = [a + b * s * s + c * s ** 4 for s in values]
        most = max(most, *(abs(f) for f in factors))
        values = [abs(s * f) for s, f in zip(values, factors)]
        widest = max(widest, *values)
        if not widest < 2.0:
            raise ValueError(
                f"newton_schulz: {steps} steps with coefficients "
                f"{coefficients} do not keep singular values below 2"
            )
    if abs(a) + abs(b) * widest ** 2 + abs(c) * widest ** 4 >= 60.0:
        raise ValueError(f"newton_schulz: coefficients {coefficients} are "
                         "too large")
    return max(most, 1.0)


def _split_steps(steps: int, growth: float, dtype: torch.dtype) -> int:
    """How many steps need two fp16 numbers for a value where a caller asks
    for reduced ones.  A rounding to one (2^-11) grows by at most ``growth``
    in its own step and in every one that follows.  16 of them together, all
    at their largest, are twice the rounding of a bf16 result (2^-8); in norm
    they stay below it (measured 0.6 of it for noise, 0.95 for a few strong
    directions).  fp16 and fp32 results need every step."""
    if dtype != torch.bfloat16:
        return steps
    single, total = 0, growth
    while single < steps and total <= 16.0:
        single += 1
        total += growth ** (single + 1)
    return steps - single


def _group(growth: float, most: int) -> int:
    """How many steps may share one product with the whole matrix: up to
    ``most``, while their common factor stays in the range that the kernels
    hold such a matrix in."""
    group = 1
    while group < most and growth ** (group + 1) < 60.0:
        group += 1
    return group


def _check_numbers(name, steps, coefficients, eps):
    if not isinstance(steps, int) or not 1 <= steps <= 100:
        raise ValueError(f"{name}: steps must be 1 to 100, got {steps}")
    if len(coefficients) != 3:
        raise ValueError(f"{name}: three coefficients, got {coefficients}")
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"{name}: eps must not be negative, got {eps}")
    return tuple(float(v) for v in coefficients)


def _reference(g, steps, coefficients, eps):
    """The formulas in fp32 (the CPU path and the tests' oracle)."""
    a, b, c = coefficients
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    norm = torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True,
                                    dtype=torch.float64)
    x = (x / (norm + eps)).float()
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def newton_schulz(
    g: torch.Tensor,
    steps: int = 5,
    coefficients: Sequence[float] = COEFFICIENTS,
    eps: float = 1e-7,
    reduced: bool = False,
) -> torch.Tensor:
    """``U V^T``, approximately, of a matrix ``[rows, cols]`` or a batch
    ``[..., rows, cols]`` in fp32, bf16 or fp16; contiguous, of ``g``'s
    shape and dtype.

    With the usual coefficients five steps bring every singular value above
    about 1e-3 of the matrix's norm into [0.68, 1.21].  Results have fp32's
    accuracy and are rounded once.  ``reduced`` lets the last steps of a bf16
    result keep 11 bits on the device, which adds an error of up to its
    rounding's size (0.6 of it for noise) and takes a quarter off the time of
    large matrices; it does nothing elsewhere.  A matrix of zeros stays one;
    one with a NaN or an infinity becomes NaN as a whole.  Not differentiable:
    a ``g`` that requires a gradient is refused, on the device a dual one and
    a call under ``torch.jit.trace`` or ``make_fx`` too.

    Workspace on the device: 16 bytes a value and 20 bytes a value of a square
    of the smaller side, both sides padded to multiples of 64, for the whole
    batch; none up to 64 x 192 (or 192 x 64).
    """
    if g.dim() < 2:
        raise ValueError("newton_schulz: g must be a matrix or a batch of "
                         f"them, got shape {tuple(g.shape)}")
    if g.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("newton_schulz: g must be fp32, bf16 or fp16, got "
                        f"{g.dtype}")
    if g.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("newton_schulz is not differentiable: call it "
                           "under torch.no_grad() or on g.detach()")
    coefficients = _check_numbers("newton_schulz", steps, coefficients, eps)
    growth = _growth(coefficients, steps)
    if not g.is_cuda:
        return _reference(g, steps, coefficients, eps).to(g.dtype) \
            .contiguous()
    from . import _ext_for

    rows, cols = g.shape[-2:]
    out = _ext_for(g).newton_schulz(
        g.contiguous().view(g.shape[:-2].numel(), rows, cols), steps,
        _split_steps(steps, growth, g.dtype) if reduced else steps,
        _group(growth, 2 if g.dtype == torch.float32 else 3), *coefficients,
        growth, eps,
    )
    return out.view(g.shape)


class MuonPlan:
    """Where the matrices of a flat buffer lie, laid out for the kernels.

    ``matrices``: ``(start, rows, cols)`` of each, ``rows * cols`` values
    from ``start`` on in row order, none overlapping; ``total``: the
    buffer's length.  A matrix's update is scaled by
    ``sqrt(max(1, rows / cols))``.  Built once; holds no state of a step, so
    any number of buffers, streams and captured graphs may share it.
    """

    def __init__(self, matrices, total: int, device="cuda"):
        self.matrices = [tuple(int(v) for v in m) for m in matrices]
        self.total = int(total)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        end = 0
        for m in sorted(self.matrices):
            if len(m) != 3 or m[1] < 1 or m[2] < 1:
                raise ValueError("MuonPlan: a matrix is (start, rows, cols), "
                                 f"got {m}")
            if m[0] < end:
                raise ValueError(f"MuonPlan: the matrix {m} overlaps "
                                 "another or starts before the buffer")
            end = m[0] + m[1] * m[2]
        if end > self.total:
            raise ValueError(f"MuonPlan: matrices end at {end}, behind the "
                             f"buffer's {self.total} values")
        self.scales = [math.sqrt(max(1.0, r / c))
                       for _, r, c in self.matrices]
        self.tables = self.layout = None
        if self.device.type == "cuda":
            from . import _ext_for

            tables, self.layout = _ext_for(self).muon_plan(
                [(*m, s) for m, s in zip(self.matrices, self.scales)],
                self.total,
            )
            self.tables = tables.to(self.device)


def muon_step_(
    params: torch.Tensor,
    grads: torch.Tensor,
    momentum_buf: torch.Tensor,
    plan: MuonPlan,
    lr,
    momentum: float = 0.95,
    weight_decay: float = 0.0,
    nesterov: bool = True,
    steps: int = 5,
    coefficients: Sequence[float] = COEFFICIENTS,
    eps: float = 1e-7,
    rest_lr: float = 1.0,
    shadow: Optional[torch.Tensor] = None,
) -> None:
    """One Muon step over flat fp32 ``params`` with fp32 or bf16 ``grads``.

    In each matrix of ``plan``:
      buf = momentum * buf + g
      u = g + momentum * buf  (nesterov)  |  u = buf
      p = p * (1 - lr * weight_decay) - lr * scale * newton_schulz(u)
    and elsewhere, with ``lr * rest_lr``:
      g = g + weight_decay * p;  buf, u as above;  p = p - lr * u
    ``shadow``, where given, receives the new parameters in bf16.  ``lr`` is
    a float, or one value on the device that a captured step reads anew.
    Not recorded by autograd; the device refuses dual tensors and tracing.
    Its workspace is that of ``newton_schulz`` for all matrices at once (16
    bytes a value and 20 a value of the smaller sides' squares, padded).
    """
    coefficients = _check_numbers("muon_step_", steps, coefficients, eps)
    growth = _growth(coefficients, steps)
    if params.device != plan.device:
        raise ValueError(f"muon_step_: the plan is for {plan.device}, params "
                         f"are on {params.device}")
    for name, t in (("params", params), ("grads", grads),
                    ("momentum_buf", momentum_buf), ("shadow", shadow)):
        if t is not None and t.shape != (plan.total,):
            raise ValueError(f"muon_step_: {name} must have the plan's "
                             f"{plan.total} values, got shape "
                             f"{tuple(t.shape)}")
    ends = sorted(
        (t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
        for t in (params, grads, momentum_buf, shadow)
        if t is not None and t.numel()
    )
    if any(a[1] > b[0] for a, b in zip(ends, ends[1:])):
        raise ValueError("muon_step_: params, grads, momentum_buf and shadow "
                         "must not share memory")
    if params.is_cuda:
        from . import _as_scalar_tensor, _ext_for

        _ext_for(params).muon_step_(
            params, grads, momentum_buf, shadow, plan.tables, plan.layout,
            plan.total, _as_scalar_tensor(lr, params), float(momentum),
            float(weight_decay), float(rest_lr), bool(nesterov), steps,
            _group(growth, 3), *coefficients, growth, eps,
        )
        return
    lr = float(lr)
    g = grads.float()
    inside = torch.zeros(plan.total, dtype=torch.bool)
    for start, rows, cols in plan.matrices:
        inside[start:start + rows * cols] = True
    g = torch.where(inside, g, g + weight_decay * params)
    momentum_buf.mul_(momentum).add_(g)
    u = g + momentum * momentum_buf if nesterov else momentum_buf
    new = torch.where(inside, params * (1.0 - lr * weight_decay),
                      params - lr * rest_lr * u)
    for (start, rows, cols), scale in zip(plan.matrices, plan.scales):
        part = slice(start, start + rows * cols)
        o = _reference(u[part].view(rows, cols), steps, coefficients, eps)
        new[part] -= lr * scale * o.reshape(-1)
    params.copy_(new)
    if shadow is not None:
        shadow.copy_(params)
