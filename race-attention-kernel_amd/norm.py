"""Norms of whole rows around a recurrent layer: on the way in with the residual's
addition, and of its heads on the way out.

    s = x + residual,  y = s / sqrt(mean(s^2) + eps) * weight
    y = x / sqrt(mean(x^2) + eps) * weight * silu(gate)

race_norm_rope takes a projection's heads to the streams the recurrences read;
race_gate_norm takes their output streams back to rows.  The reference has no
counterpart.
"""
from __future__ import annotations

import torch

from . import _lib


def race_add_norm(x: torch.Tensor, residual: torch.Tensor | None = None, weight: torch.Tensor | None = None, *,
                  eps: float = 1e-6):
    """(y, sum): rows normed by their root mean square, behind the residual's addition.

    Args:
        x: [..., D] float32 or bfloat16, D up to 16384, of any strides.
        residual: of x's shape and dtype; None: x itself is normed.
        weight: [D] in x's dtype or float32; None is ones.
        eps: of the root mean square.

    Returns y and sum = x + residual, both of x's shape and dtype (sum None without
    a residual).  y is the norm of sum as it is stored.  Differentiable once,
    w.r.t. x, residual and weight, through both.  A backward is captured into a
    graph together with its forward, and not while an eager graph of the same
    leaves is alive."""
    return _lib.ext().add_norm(x, residual, weight, eps)


def race_add_norm_e4m3(x: torch.Tensor, residual: torch.Tensor | None = None, weight: torch.Tensor | None = None, *,
                       eps: float = 1e-6, group: int = 0):
    """(y8, scales, sum): race_add_norm with y in 8 bits, for an 8-bit projection.
    Gradients pass through sum, the residual stream, alone: y8 and scales have none,
    so the weight and what lies behind them get none.

    y8 is float8_e4m3fn and y8 * scale stands for y: one float32 scale for each
    row (group 0, scales [..., 1]) or for each `group` of 32, 64 or 128 columns
    (scales [..., ceil(D / group)]; D a multiple of 8), the largest magnitude
    over 448.  Rows or groups of zeros have the scale 0."""
    return _lib.ext().add_norm_e4m3(x, residual, weight, eps, group)


def race_gate_norm(x: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor | None = None, *,
                   eps: float = 1e-6) -> torch.Tensor:
    """A recurrence's output streams as rows, normed per head and gated.

    Args:
        x: [B * H, T, d] float32 or bfloat16, d up to 256 (race_delta_rule's out).
        gate: [B, T, H, d] of the same dtype, of any batch, token and head strides.
        weight: [d] in x's dtype or float32; None is ones.
        eps: of the root mean square.

    Returns [B, T, H, d].  Differentiable once, w.r.t. x, gate and weight.  A
    backward is captured into a graph together with its forward, and not while an
    eager graph of the same leaves is alive."""
    return _lib.ext().gate_norm(x, gate, weight, eps)
