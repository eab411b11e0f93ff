"""The gated linear recurrence: h_t = a_t h_{t-1} + u_t per stream and channel.

    a = sigmoid(gate) or exp(gate),   u = (1 - a) x or x

The recurrent layer of a stack that mixes layers of the per-bucket op with
recurrent ones.  It takes the same streams of tokens and hands its state on the
same way: a prompt, then a call per token (race_gated_scan_carry).  The
reference has no counterpart.
"""
from __future__ import annotations

import torch

from . import _lib

GATE_FORMS = {"sigmoid": 0, "log": 1}


def _form_id(gate_form: str) -> int:
    try:
        return GATE_FORMS[gate_form]
    except KeyError:
        raise ValueError(f"gate_form must be one of {sorted(GATE_FORMS)}, got {gate_form!r}") from None


def race_gated_scan(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor | None = None, *,
                    gate_form: str = "sigmoid", complement: bool = True, lengths: torch.Tensor | None = None):
    """(out, final): the gated linear recurrence over the tokens of every stream.

    Args:
        x, gate: [N, T, D] float32 or bfloat16, of any stream and token strides.
        state: [N, D] float32, the state before the first token; None is zero.
        gate_form: "sigmoid" (gate holds logits) or "log" (gate holds log a, 0 at
            most: products of larger ones may overflow; -inf forgets everything
            before the token).
        complement: u = (1 - a) x, else u = x.
        lengths: int32 (or int64) [N] or [N / g] (entry i for the streams g i .. g i + g - 1):
            tokens from lengths on are not read, their rows of out are zero and
            the state passes them unchanged.

    Returns out [N, T, D] in x's dtype and the float32 state [N, D] after the
    last token.  Sums are in float32.  Differentiable once, w.r.t. x, gate and
    state, through out and final: the forward keeps the state every tile of tokens
    starts from and the backward recomputes h from those, not from the rounded
    output.  A backward is captured into a graph together with its forward, and
    not while an eager graph of the same leaves is alive."""
    return _lib.ext().gated_scan(x, gate, state, lengths, _form_id(gate_form), complement)


def race_gated_scan_carry(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, *, gate_form: str = "sigmoid",
                          complement: bool = True, lengths: torch.Tensor | None = None, inplace: bool = False):
    """(out, new_state): race_gated_scan continued from a carried state, without
    autograd; with inplace=True the state tensor itself is advanced and
    returned.  Calls of at most 16 tokens (decode) run one small launch."""
    return _lib.ext().gated_scan_carry(x, gate, state, lengths, _form_id(gate_form), complement, inplace)
