"""The gated delta rule: a recurrence whose state is a matrix per stream, which every
token corrects by what it answers wrongly to the token's key.

    S_t = a_t S_{t-1} + beta_t k_t (v_t - a_t S_{t-1}^T k_t)^T,   out_t = scale S_t^T q_t

The per-bucket op's running sums B (S_t = S_{t-1} + k_t v_t^T) with a decay and
without what the state already holds.  It takes the same streams of tokens
(race_norm_rope's rows, or bucket probabilities) and hands its state on the same
way: a prompt, then a call per token (race_delta_rule_carry).  The reference has
no counterpart.
"""
from __future__ import annotations

import torch

from . import _lib
from .recurrence import _form_id


def race_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, gate: torch.Tensor | None, beta: torch.Tensor,
                    state: torch.Tensor | None = None, *, gate_form: str = "log", scale: float = 1.0,
                    lengths: torch.Tensor | None = None):
    """(out, final): the gated delta rule over the tokens of every stream.

    Args:
        q, k: [Nk, T, dk] (or [Nk, T, L, R], dk = L R) float32 or bfloat16, dk up to
            128, of any stream and token strides.  Keys are used as they are: with
            |k| <= 1 and beta <= 1 (2) the state does not grow.
        v: [N, T, dv] of the same dtype, dv up to 256.  N = g Nk: value streams g n ..
            g n + g - 1 share key stream n (value heads that share a key head).
        gate: [N, T] in q's dtype or float32, or None (a = 1).
        beta: [N, T] of gate's dtype: how much of its error a token corrects.
        state: [N, dk, dv] float32, the state before the first token; None is zero.
        gate_form: "log" (gate holds log a, at most 0; -inf, and all below -200, forgets
            everything before the token) or "sigmoid" (gate holds logits).
        scale: of the outputs.
        lengths: int32 (or int64) [N] or [N / h] (entry i for the value streams h i ..
            h i + h - 1): tokens from lengths on are not read, their rows of out are
            zero and the state passes them unchanged.

    Returns out [N, T, dv] in v's dtype and the float32 state [N, dk, dv] after the
    last token.  Sums, states and computed factors are in float32: bfloat16 rows give
    what the same values in float32 do, rounded once.  Differentiable once, w.r.t. q, k,
    v, gate, beta and state, through out and final; until its backward a call keeps
    about 4 (dk + 64) dv + 37000 bytes for each value stream and 64 tokens (8 times its
    bfloat16 values at 128 x 128; dk counts as 64 or 128, dv in multiples of 16).  A backward is captured into a
    graph together with its forward, and not while an eager graph of the same
    leaves is alive."""
    return _lib.ext().delta_rule(q, k, v, gate, beta, state, lengths, _form_id(gate_form), scale)


def race_delta_rule_carry(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, gate: torch.Tensor | None, beta: torch.Tensor,
                          state: torch.Tensor, *, gate_form: str = "log", scale: float = 1.0,
                          lengths: torch.Tensor | None = None, inplace: bool = False):
    """(out, new_state): race_delta_rule continued from a carried state, without
    autograd (its outputs require no gradients, whatever its inputs do); with inplace=True the state tensor itself is advanced and returned.
    Calls of at most 16 tokens (decode) run one small launch."""
    return _lib.ext().delta_rule_carry(q, k, v, gate, beta, state, lengths, _form_id(gate_form), scale, inplace)
