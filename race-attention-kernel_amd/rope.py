"""Norm and rotation of query and key heads, on the way to the op's streams.

The rows of every head are divided by their root mean square and multiplied by a
weight per column, and pairs of their values are turned by the token's position,
in the pass that takes a projection's [B, T, H, d] rows to the streams
[B * H, T, d] the op and the hashing read (the permutes of
src/race_baseline.py:35-40).  The norm and the rotation have no counterpart in
the reference.
"""
from __future__ import annotations

import torch

from . import _lib


def race_norm_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor | None = None,
                   inv_freq: torch.Tensor | None = None, *, q_weight: torch.Tensor | None = None,
                   k_weight: torch.Tensor | None = None, eps: float | None = 1e-6, sections=None,
                   interleaved: bool = False):
    """(q, k) as streams: the heads' rows normed and rotated, in one launch.

    Args:
        q: [B, T, Hq, d], k: [B, T, Hk, d] or None; float32 or bfloat16, d up to
            256, of any batch, token and head strides (a slice of a joint
            projection as it is).
        positions: int32 or int64 [T] or [B, T], or [axes, B, T] with sections.
        inv_freq: float32 [P], 2 P <= d: pair p turns by position * inv_freq[p],
            formed in 64 bits.  None: no rotation.
        q_weight, k_weight: [d] each, in q's dtype or float32; None is ones.
        eps: of the root mean square; None: no norm.
        sections: pairs per position axis, in order (they sum to P; at most 4
            axes); None: one axis.
        interleaved: the pairs are values (2p, 2p + 1), else (p, p + P).  Values
            from 2 P on are only normed.

    Returns streams [B * Hq, T, d] and [B * Hk, T, d] (or None) in q's dtype.
    Differentiable once, w.r.t. q, k and the weights.  A backward is captured into
    a graph together with its forward, and not while an eager graph of the same
    leaves is alive."""
    return _lib.ext().norm_rope(q, k, positions, inv_freq, q_weight, k_weight, eps,
                                [] if sections is None else list(sections), interleaved)
