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
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _dense


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as the kernels read it, by strides: a copy only where the values of a
    row are apart or the first is not 16-byte aligned."""
    if t.numel() and ((t.size(-1) > 1 and t.stride(-1) != 1) or t.data_ptr() % 16):
        return t.clone(memory_format=torch.contiguous_format)
    return t


class NormRopeFunction(torch.autograd.Function):
    """(q, k) streams = race_norm_rope(q, k, ..), differentiable w.r.t. the rows
    and the weights; saves the inputs."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, inv_freq, eps, norm, sections, interleaved):
        _lib.ext().check_capture("race_norm_rope", [q, k, q_weight, k_weight])
        out_q, out_k = _lib.ext().norm_rope_forward(q, k, positions, inv_freq, q_weight, k_weight, eps, norm, sections,
                                                    interleaved)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, inv_freq)
        ctx.args = (eps, norm, sections, interleaved)
        return out_q, out_k

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        grads = (None, None, None, None)
        if dq is not None or dk is not None:
            q, k, qw, kw, positions, inv_freq = ctx.saved_tensors
            _lib.ext().check_capture("race_norm_rope backward", [q, k, qw, kw])
            dq, dk = (None if g is None else _dense(g.to(q.dtype)) for g in (dq, dk))
            grads = _lib.ext().norm_rope_backward(q, k, positions, inv_freq, qw, kw, dq, dk, *ctx.args,
                                                  *ctx.needs_input_grad[:4])
        return (*grads, None, None, None, None, None, None)


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
    Differentiable w.r.t. q, k and the weights."""
    q, k = _rows(q), None if k is None else _rows(k)
    options = (0.0 if eps is None else float(eps), eps is not None, list(sections) if sections is not None else [],
               bool(interleaved))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return NormRopeFunction.apply(q, k, q_weight, k_weight, positions, inv_freq, *options)
    return _lib.ext().norm_rope_forward(q, k, positions, inv_freq, q_weight, k_weight, *options)
