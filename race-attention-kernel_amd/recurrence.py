"""The gated linear recurrence: h_t = a_t h_{t-1} + u_t per stream and channel.

    a = sigmoid(gate) or exp(gate),   u = (1 - a) x or x

The recurrent layer of a stack that mixes layers of the per-bucket op with
recurrent ones.  It takes the same streams of tokens and hands its state on the
same way: a prompt, then a call per token (race_gated_scan_carry).  The
reference has no counterpart.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _dense

GATE_FORMS = {"sigmoid": 0, "log": 1}


def _form_id(gate_form: str) -> int:
    try:
        return GATE_FORMS[gate_form]
    except KeyError:
        raise ValueError(f"gate_form must be one of {sorted(GATE_FORMS)}, got {gate_form!r}") from None


MAX_TOKEN_STRIDE = 1 << 20  # elements; RACE_SCAN_MAX_TOKEN_STRIDE


def _channel_rows(t: torch.Tensor) -> torch.Tensor:
    """t as the kernels read it, by strides: a copy only where the channels of a
    token are apart, the first is not 16-byte aligned, or tokens lie very far apart."""
    if t.dim() == 3 and t.numel() and ((t.size(2) > 1 and t.stride(2) != 1) or t.data_ptr() % 16 or
                                       (t.size(1) > 1 and t.stride(1) > MAX_TOKEN_STRIDE)):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _lengths(lengths):
    if lengths is not None and lengths.dtype == torch.int64:
        lengths = lengths.to(torch.int32)
    return lengths


class GatedScanFunction(torch.autograd.Function):
    """(out, final) = race_gated_scan(x, gate, state).  The forward keeps the
    state every tile of tokens starts from, in 32 bits, and the backward
    recomputes h from those: the rounded output is not read."""

    @staticmethod
    def forward(ctx, x, gate, state, lengths, form, complement):
        _lib.ext().check_capture("race_gated_scan", [x, gate, state])
        out, final, records = _lib.ext().gated_scan_forward(x, gate, state, lengths, form, complement, True, False)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, gate, lengths, records)
        ctx.args = (form, complement)
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dfinal):
        if dout is None and dfinal is None:
            return None, None, None, None, None, None
        x, gate, lengths, records = ctx.saved_tensors
        _lib.ext().check_capture("race_gated_scan backward", [x, gate])
        dout = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dout is None else _dense(dout.to(x.dtype))
        if dfinal is not None:
            dfinal = _dense(dfinal.float())
        grads = _lib.ext().gated_scan_backward(x, gate, lengths, dout, dfinal, records, *ctx.args,
                                               *ctx.needs_input_grad[:3])
        return (*grads, None, None, None)


def race_gated_scan(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor | None = None, *,
                    gate_form: str = "sigmoid", complement: bool = True, lengths: torch.Tensor | None = None):
    """(out, final): the gated linear recurrence over the tokens of every stream.

    Args:
        x, gate: [N, T, D] float32 or bfloat16, of any stream and token strides.
        state: [N, D] float32, the state before the first token; None is zero.
        gate_form: "sigmoid" (gate holds logits) or "log" (gate holds log a;
            -inf forgets everything before the token).
        complement: u = (1 - a) x, else u = x.
        lengths: int32 [N] or [N / g] (entry i for the streams g i .. g i + g - 1):
            tokens from lengths on are not read, their rows of out are zero and
            the state passes them unchanged.

    Returns out [N, T, D] in x's dtype and the float32 state [N, D] after the
    last token.  Sums are in float32.  Differentiable w.r.t. x, gate and state,
    through out and final."""
    x, gate, lengths, form = _channel_rows(x), _channel_rows(gate), _lengths(lengths), _form_id(gate_form)
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (state is not None and state.requires_grad)):
        return GatedScanFunction.apply(x, gate, state, lengths, form, bool(complement))
    return _lib.ext().gated_scan_forward(x, gate, state, lengths, form, bool(complement), False, False)[:2]


def race_gated_scan_carry(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, *, gate_form: str = "sigmoid",
                          complement: bool = True, lengths: torch.Tensor | None = None, inplace: bool = False):
    """(out, new_state): race_gated_scan continued from a carried state, without
    autograd; with inplace=True the state tensor itself is advanced and
    returned.  Calls of at most 16 tokens (decode) run one small launch."""
    out, new_state, _ = _lib.ext().gated_scan_forward(_channel_rows(x), _channel_rows(gate), state, _lengths(lengths),
                                                      _form_id(gate_form), bool(complement), False, bool(inplace))
    return out, new_state
