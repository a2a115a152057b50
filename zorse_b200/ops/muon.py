"""Muon: momentum whose matrices are orthogonalised by Newton-Schulz products before they step the weights (csrc/optim/newton_schulz.cu)."""
from __future__ import annotations

import math

import torch

COEFFICIENTS = 3.4445, -4.7750, 2.0315      # of X, X X^T X and X X^T X X^T X in an iteration
# An orthogonalised n x m matrix has entries of 1 / sqrt(max(n, m)) in root mean square: times SCALE sqrt(max(n, m)) they are of the size of
# an AdamW step's, so that one learning rate (and decay) serves both.
SCALE = 0.2


def orthogonalize(u: torch.Tensor, iterations: int = 5) -> torch.Tensor:
    """U / ||U|| with its singular values driven to about 1; zeros stay zeros.  At least fp32 inside and as the result's type."""
    u = u.to(torch.promote_types(u.dtype, torch.float32))
    norm = u.double().square().sum().sqrt()
    x = u / torch.where(norm > 0, norm, 1.0).to(u.dtype)
    turned = u.shape[0] > u.shape[1]
    x = x.t() if turned else x
    a, b, c = COEFFICIENTS
    for _ in range(iterations):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if turned else x


def muon_step(p, m, g, *, lr, momentum, weight_decay, nesterov, iterations, grad_scale) -> None:
    """In place on one weight matrix and its momentum."""
    g = g.to(m.dtype) * grad_scale
    m.mul_(momentum).add_(g)
    x = orthogonalize(g + momentum * m if nesterov else m, iterations)
    p.mul_(1 - lr * weight_decay).sub_(x * (lr * SCALE * math.sqrt(max(p.shape))))
