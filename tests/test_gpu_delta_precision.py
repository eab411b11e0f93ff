"""bf16 rows of the gated delta rule: what is computed in 32 bits, rounded once.

Tolerances.  bf16 values are fp32 values, so the recurrence of bf16 rows owes what
fp32 rows owe: 384 * 2^-24 of the terms (test_gpu_delta_rule).  Results in 32 bits are
held to that as they are.  Results in bf16 are off by the rounding of a value, at most
half of its step, and by no more than that tolerance beyond it: what lies beyond a value's
half step counts, in 2-norm over a stream and over its rows (8 times, as there).  Where
only bf16 comes of a product, its computed factors are taken in two parts of bf16, each
within 2^-16: two of them in outputs, four in the gradients of calls with bf16 gates (the
pairs of tokens take two rows' and then their own matrix's)."""
from __future__ import annotations

import pytest
import torch

from gpu_util import say
from test_gpu_delta_rule import BF16, F32, NAMES, close, make, reference, tolerance

pytestmark = pytest.mark.gpu


def half_step(x):
    """Half of the distance between the bf16 values around x (float64)."""
    return torch.ldexp(torch.ones_like(x), torch.frexp(x)[1] - 9)


def rounded_once(name, got, want, what="", pairs=0):
    value, square = want
    assert got.dtype == BF16 and got.shape == value.shape and torch.isfinite(got).all(), name
    tol = tolerance(name, F32) + pairs * 2.0 ** -16
    N, D = value.shape[0], 1 if name in ("dgate", "dbeta") else value.shape[-1]
    beyond = ((got.detach().double() - value).abs() - half_step(value)).clamp(min=0).reshape(N, -1, D).norm(dim=2)
    ref = (value.reshape(N, -1, D).pow(2).sum(2) + square.expand(N, beyond.shape[1])).sqrt()
    stream = float((beyond.norm(dim=1) / ref.norm(dim=1).clamp(min=1e-30)).max())
    row = float((beyond / torch.maximum(ref, ref.pow(2).mean(1, keepdim=True).sqrt()).clamp(min=1e-30)).max())
    say(what, name, f"beyond a rounding: stream {stream:.1e} row {row:.1e} of {tol:.1e}")
    assert stream <= tol and row <= 8 * tol, f"{name}: stream {stream}, row {row}, tolerance {tol}"


# A walk in one piece and in segments, whole rows and odd ones, shared key heads.
SHAPES = [(2, 1, 130, 64, 64), (2, 2, 200, 128, 128), (6, 2, 100, 33, 17), (3, 1, 1537, 128, 72), (2, 2, 1600, 64, 50)]


@pytest.mark.parametrize("N, Nk, T, dk, dv", SHAPES)
def test_outputs_and_states(race, cuda, N, Nk, T, dk, dv):
    *args, _, _ = make(N, Nk, T, dk, dv, BF16, seed=31, gate_dtype=F32)
    want = reference(*(t.float() for t in args), scale=dk ** -0.5)
    for records in (False, True):
        some = [t.clone().requires_grad_(records) for t in args]
        out, state = race.race_delta_rule(*some, scale=dk ** -0.5)
        rounded_once("out", out, want["out"], f"T={T}", pairs=2)
        close("state", state, want["state"], F32, f"T={T}")


@pytest.mark.parametrize("T", [64, 128, 1600])
def test_small_values_overwrite_a_large_state(race, cuda, T):
    # One key of length 1, strength 1 and no decay: the state is the last value.  Within the first chunk what was there, up
    # to 1024, goes by sums of 32 bits: a few roundings of 2^-24 each; behind it the state holds values of 2^-10, with theirs.
    N, dv = 8, 40
    g = torch.Generator(device=cuda).manual_seed(32)
    one = torch.ones(N, T, 1, dtype=BF16, device=cuda)
    v = (torch.randn(N, T, dv, generator=g, device=cuda) * 2.0 ** -10).to(BF16)
    state = (torch.rand(N, 1, dv, generator=g, device=cuda) + 1) * 512.0
    beta = torch.ones(N, T, dtype=BF16, device=cuda)
    for grad in (False, True):
        out, final = race.race_delta_rule(one, one, v, None, beta, state.clone().requires_grad_(grad))
        largest = 1024.0 if T == 64 else float(v.float().abs().max()) + 1024.0 * 2.0 ** -22
        err = float((final[:, 0] - v[:, -1].float()).abs().max())
        say(T, f"{err:.1e} of {8 * 2.0 ** -24 * largest:.1e}")
        assert err <= 8 * 2.0 ** -24 * largest


@pytest.mark.parametrize("gate_dtype", [F32, BF16])
@pytest.mark.parametrize("N, Nk, T, dk, dv", SHAPES)
def test_gradients(race, cuda, N, Nk, T, dk, dv, gate_dtype):
    *args, dout, dfinal = make(N, Nk, T, dk, dv, BF16, seed=33, gate_dtype=gate_dtype)
    leaves = [t.clone().requires_grad_(True) for t in args]
    outs = race.race_delta_rule(*leaves, scale=dk ** -0.5)
    grads = torch.autograd.grad(outs, leaves, (dout, dfinal))
    want = reference(*(t.float() for t in args), scale=dk ** -0.5, dout=dout, dfinal=dfinal)
    for name, t, d in zip(NAMES, args, grads):
        assert d.dtype == t.dtype
        if t.dtype == BF16:
            rounded_once("d" + name, d, want["d" + name], f"T={T}", pairs=0 if gate_dtype == F32 else 4)
        else:
            close("d" + name, d, want["d" + name], F32, f"T={T}")
