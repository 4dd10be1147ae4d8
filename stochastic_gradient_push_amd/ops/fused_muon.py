"""FusedMuon — orthogonalised momentum updates over a flat parameter buffer.

The counterpart of :class:`~stochastic_gradient_push_amd.ops.fused_sgd.FusedSGD`
for networks whose matrices should move by the orthogonal factor of their
momentum rather than by the momentum itself.  Matrices of all shapes go
through every Newton-Schulz product in one launch
(:func:`~stochastic_gradient_push_amd.ops.muon_step_`); vectors — norm
weights, biases — and parameters named in ``sgd_params`` get momentum SGD in
the same pass.  State, gradient and checkpoint handling are FusedSGD's.
"""

import torch

from .flat import FlatParams
from .fused_sgd import FusedSGD
from .muon import COEFFICIENTS, MuonPlan, muon_step_
from ..utils.roctx import trace as _roctx


class FusedMuon(FusedSGD):
    """``lr``: of the orthogonalised updates, whose entries are around
    ``1 / sqrt(cols)`` whatever the gradient's size; ``rest_lr``: what ``lr``
    is multiplied with for all other parameters; ``weight_decay``: taken off
    the matrices directly, added to the gradient elsewhere.

    A parameter of two or more dimensions is a matrix of ``shape[0]`` rows
    (a convolution: one row per output channel) unless it is in
    ``sgd_params``, an iterable of parameters.
    """

    def __init__(
        self,
        flatp: FlatParams,
        lr: float,
        momentum: float = 0.95,
        weight_decay: float = 0.0,
        nesterov: bool = True,
        ns_steps: int = 5,
        ns_coefficients=COEFFICIENTS,
        eps: float = 1e-7,
        rest_lr: float = 1.0,
        sgd_params=(),
        steal_grads: bool = False,
    ):
        if flatp.flat.dtype != torch.float32:
            raise TypeError("FusedMuon needs fp32 parameters, got "
                            f"{flatp.flat.dtype}")
        super().__init__(flatp, lr, momentum=momentum,
                         weight_decay=weight_decay, nesterov=nesterov,
                         steal_grads=steal_grads)
        self.momentum_buf = torch.zeros_like(flatp.flat)
        self.param_groups[0].update(
            ns_steps=ns_steps, ns_coefficients=tuple(ns_coefficients),
            eps=eps, rest_lr=rest_lr,
        )
        known = {id(p) for p in flatp.params}
        skip = {id(p) for p in sgd_params}
        if not skip <= known:
            raise ValueError("FusedMuon: sgd_params has a parameter that is "
                             "not in the flat buffer")
        matrices, at = [], 0
        for p in flatp.params:
            if p.dim() >= 2 and p.numel() and id(p) not in skip:
                matrices.append((at, p.shape[0], p.numel() // p.shape[0]))
            at += p.numel()
        # with bf16 working weights: the section that has them, whose
        # gradients are bf16, and the fp32 rest behind it
        n_cast, total = flatp.n_cast, flatp.flat.numel()
        device = flatp.flat.device
        if self._mixed:
            # (a matrix has two dimensions and so lies in the first)
            self._plans = [
                (0, MuonPlan(matrices, n_cast, device), flatp.flat_grad_w,
                 flatp.shadow),
                (n_cast, MuonPlan([], total - n_cast, device),
                 flatp.flat_grad, None),
            ]
        else:
            self._plans = [
                (0, MuonPlan(matrices, total, device), flatp.flat_grad, None),
            ]

    @torch.no_grad()
    def step(self, closure=None):
        g = self.param_groups[0]
        if self._steal:
            self.flatp.gather_grads()
        elif not self.flatp.grads_wired():
            self.flatp.rewire_grads()
        self.sync_lr()
        lr = self._lr_dev if self._lr_dev is not None else g["lr"]
        with _roctx("sgp:fused_muon_step"):
            for start, plan, grads, shadow in self._plans:
                if plan.total == 0:
                    continue
                muon_step_(
                    self.flatp.flat.narrow(0, start, plan.total), grads,
                    self.momentum_buf.narrow(0, start, plan.total), plan, lr,
                    momentum=g["momentum"], weight_decay=g["weight_decay"],
                    nesterov=g["nesterov"], steps=g["ns_steps"],
                    coefficients=g["ns_coefficients"], eps=g["eps"],
                    rest_lr=g["rest_lr"], shadow=shadow,
                )
        self._first_step = False
