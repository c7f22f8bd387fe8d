"""Applies the SGD rules to a network's flat vectors.

On CUDA this is the fused one-pass kernel (csrc/sgd_fused.cu), launched once for the regularised range and
once for the unregularised tail; on CPU it is ``reference_step``. ``phase`` lets the training loop split
"accumulate into the momentum buffer" from "apply to the parameters" when a parameter exchange sits between
the two (the reference's SyncParamsThenStep order, src/opt/sgd/new.rs:408-431).

With `clip_norm` the gradients of all parameters are measured first (csrc/grad_clip.cu) and the sweep multiplies them by the
coefficient, which it reads on the device: a captured step clips as an eager one does. What is measured is the gradient buffer:
with the rule that keeps its momentum there (GRAD_DECAY), the momentum is part of the norm and is clipped with the rest.
"""
from __future__ import annotations

import math

import torch

from ..ops import native_ops as K
from .sgd import Momentum, clip_coefficient, reference_step


class SgdStepper:
    def __init__(self, net, momentum: Momentum, mu: float, l2: float, clip_norm: float = 0.0):
        if not (clip_norm == 0.0 or 2.0 ** -149 <= clip_norm < math.inf):
            raise ValueError(f"gradients are clipped to a norm that is a float32 above 0 (0: not at all), not {clip_norm}")
        self.net = net
        self.mode = int(momentum)
        self.mu = float(mu) if momentum != Momentum.ZERO else 0.0
        self.l2 = float(l2)
        self.clip_norm = float(clip_norm)
        # norm and coefficient of the present iteration: on the device, or as numbers
        self.clip = torch.zeros(2, dtype=torch.float32, device=net.device) if net.is_cuda and self.clip_norm else None
        self._clip_host = (0.0, 1.0)
        self._clip_ws = K.grad_norm_scratch(net.device) if self.clip is not None else None
        self._clip_list = self._clip_of = None

    def _measure(self, grad_scale):
        """Norm and coefficient of all gradients, as they are now."""
        net = self.net
        if net.is_cuda:
            if self._clip_of is not net.grads:
                self._clip_list, self._clip_of = K.grad_list([net.grads]), net.grads
            K.grad_norm(self._clip_list, self.clip_norm, self.clip, self._clip_ws, scale=grad_scale)
        else:
            norm = float((grad_scale * torch.linalg.vector_norm(net.grads.detach(), dtype=torch.float64)).float())
            self._clip_host = (norm, clip_coefficient(norm, self.clip_norm))

    def grad_norm(self):
        """Global norm of the gradients of the last iteration, before clipping; None where they are not clipped. Waits for the
        device."""
        if not self.clip_norm:
            return None
        return float(self.clip[0]) if self.clip is not None else self._clip_host[0]

    def _ranges(self, lo, hi):
        """Split [lo, hi) at the boundary between regularised and unregularised parameters."""
        d = self.net.decay_len
        out = []
        if lo < min(hi, d):
            out.append((lo, min(hi, d), self.l2))
        if max(lo, d) < hi:
            out.append((max(lo, d), hi, 0.0))
        return out

    def step(self, lr: float, grad_scale: float = 1.0, phase: int = 7, lo: int = 0, hi: int = None, grid=None):
        """`lr`: a number, or one float on the device that the sweep reads when it runs. `grid` = (blocks, threads) launches
        the sweep with small blocks (used when it runs beside backward)."""
        net = self.net
        hi = net.flat_len if hi is None else hi
        clip = {}
        if self.clip_norm:
            if (lo, hi) != (0, net.flat_len) or grid is not None:
                raise ValueError("gradients are clipped by the norm of all of them: the sweep can neither take a part nor run beside "
                                 "backward")
            if phase & 1:        # a later phase of the iteration goes by the norm that this one has found
                self._measure(grad_scale)
            if net.is_cuda:
                clip["clip"] = self.clip
        for a, b, l2 in self._ranges(lo, hi):
            n = b - a
            if net.is_cuda and grid is not None:
                K.sgd_fused_grid(net.params[a:b], net.grads[a:b], net.mom[a:b], net.params16[a:b], n, lr, self.mu,
                                 l2, grad_scale, self.mode, phase, grid[0], grid[1])
            elif net.is_cuda:
                K.sgd_fused(net.params[a:b], net.grads[a:b], net.mom[a:b], net.params16[a:b], n, lr, self.mu, l2,
                            grad_scale, self.mode, phase, **clip)
            else:
                coef = self._clip_host[1] if self.clip_norm else 1.0
                with torch.no_grad():
                    if coef == 0.0:
                        net.grads[a:b].zero_()
                    reference_step(net.params[a:b], net.grads[a:b], net.mom[a:b], lr, self.mu, l2, grad_scale * coef,
                                   self.mode, phase)

    def nesterov_lookahead(self, sign: float = 1.0):
        """w += sign * mu * v: the reference keeps Nesterov parameters at the look-ahead point and applies this
        once before training (src/opt/sgd/new.rs:257-262)."""
        net = self.net
        if net.is_cuda:
            K.axpy_shadow(net.params, net.mom, net.params16, net.flat_len, sign * self.mu)
        else:
            with torch.no_grad():
                net.params.add_(net.mom, alpha=sign * self.mu)
