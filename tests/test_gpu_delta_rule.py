"""race_delta_rule and race_delta_rule_carry against the recurrence token by token in
64 bits, the gradients against its derivative by autograd.

Tolerances.  Keys have |k| <= 1 and beta <= 1, so a token's map of the state is a
contraction: an error made at a token is not amplified behind it, and errors add as
the terms do that they are relative to.  terms() squares and sums those of the
chunks of 64 tokens that the sums are taken in, with T = (I + N)^-1 what the
tokens of a chunk do to each other: where the tokens' corrections of the state
cancel, results are smaller than their terms.  Relative to them, in 2-norm over a
stream and over its rows:
  fp32 rows: a sum of up to 128 + 64 products, each off by 2^-24, is taken in runs
    whose rounding adds as many again: 384 * 2^-24 = 2.3e-5.
  bf16 rows: a result is rounded once, by at most 2^-8, and so are up to three factors
    of a term; the four are independent: 2 * 2^-8.  The state takes four factors in
    pairs of bf16, each within 2^-16: as independent ones, 2 * 2^-16.
A row has fewer terms than a stream to even them out: 8 times the stream's
tolerance, relative to the row's terms or to the mean row's, whichever are larger.
"""
from __future__ import annotations

import math

import pytest
import torch

from gpu_util import say

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
NAMES = ("q", "k", "v", "gate", "beta", "state")


def tolerance(name, dtype):
    if dtype == F32:
        return 384 * 2.0 ** -24
    return 2.0 ** -15 if name == "state" else 2.0 ** -7


def close(name, got, want, dtype, what=""):
    """Streams, and rows of a stream, within the tolerance; want: (values, a row's squared terms)."""
    value, square = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.isfinite(got).all(), name
    if value.numel() == 0:
        return
    N, D, tol = value.shape[0], value.shape[-1], tolerance(name, dtype)
    if name in ("dgate", "dbeta"):
        D = 1
    err = (got.detach().double() - value).reshape(N, -1, D).norm(dim=2)
    ref = (value.reshape(N, -1, D).pow(2).sum(2) + square.expand(N, err.shape[1])).sqrt()
    stream = float((err.norm(dim=1) / ref.norm(dim=1).clamp(min=1e-30)).max())
    row = float((err / torch.maximum(ref, ref.pow(2).mean(1, keepdim=True).sqrt()).clamp(min=1e-30)).max())
    say(what, name, f"stream {stream:.1e} row {row:.1e} of {tol:.1e}")
    assert stream <= tol and row <= 8 * tol, f"{name}: stream {stream}, row {row}, tolerance {tol}"


def make(N, Nk, T, dk, dv, dtype, form="log", seed=0, gate_dtype=None, device="cuda"):
    """q, k, v, gate, beta, state, dout, dfinal."""
    g = torch.Generator(device=device).manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g, device=device)
    unit = lambda x: 0.99 * x / x.norm(dim=-1, keepdim=True)  # below 1 as bf16 too
    gate = n(N, T) + torch.linspace(0.0, 6.0, N, device=device)[:, None]
    if form == "log":
        gate = torch.nn.functional.logsigmoid(gate)
    small = gate_dtype or dtype
    return (unit(n(Nk, T, dk)).to(dtype), unit(n(Nk, T, dk)).to(dtype), n(N, T, dv).to(dtype), gate.to(small),
            torch.sigmoid(n(N, T)).to(small), n(N, dk, dv) / dk ** 0.5, n(N, T, dv).to(dtype), n(N, dk, dv) / dk ** 0.5)


def reference(q, k, v, gate, beta, state, form="log", scale=1.0, lengths=None, dout=None, dfinal=None):
    """out, final ("state") and with an upstream gradient those of NAMES, in 64 bits, all token by token, each
    with its rows' squared terms."""
    dtype = v.dtype
    N, T, dv = v.shape
    leaves = [None if t is None else t.detach().double().requires_grad_(True) for t in (q, k, v, gate, beta, state)]
    q, k, v, gate, beta, state = leaves
    g = N // q.shape[0]
    q, k = (t.flatten(2).repeat_interleave(g, 0) for t in (q, k))
    live = torch.ones(N, T, dtype=torch.bool, device=v.device)
    if lengths is not None:
        live = torch.arange(T, device=v.device) < lengths.repeat_interleave(N // len(lengths))[:, None]
    drop = lambda t: torch.where(live.view(N, T, *[1] * (t.dim() - 2)), t, torch.zeros((), dtype=t.dtype, device=t.device))
    q, k, v, b = drop(q), drop(k), drop(v), drop(beta)
    a = torch.ones(N, T, dtype=torch.float64, device=v.device)
    if gate is not None:
        a = torch.where(live, torch.exp(drop(gate)) if form == "log" else torch.sigmoid(drop(gate)), a)
    S = state if state is not None else torch.zeros(N, q.shape[2], dv, dtype=torch.float64, device=v.device)
    out, errors, states = [], [], [S]
    for t in range(T):
        aS = a[:, t, None, None] * S
        e = v[:, t] - (k[:, t, :, None] * aS).sum(1)
        S = aS + k[:, t, :, None] * (b[:, t, None] * e)[:, None]
        out.append(scale * (q[:, t, :, None] * S).sum(1))
        errors.append(e)
        if t % 64 == 63 or t == T - 1:
            states.append(S)
    out, y = torch.stack(out, 1), torch.stack(errors, 1)
    r = dict(out=out.detach(), state=S.detach())
    up, dS = torch.zeros_like(v), [torch.zeros_like(s) for s in states]
    if dout is not None or dfinal is not None:
        loss = 0.0
        if dout is not None:
            up = drop(dout.double())  # rows behind the end have no gradient
            loss = loss + (out * up).sum()
        if dfinal is not None:
            loss = loss + (S * dfinal.double()).sum()
        want = [t for t in leaves if t is not None]
        inner = [s for s in states if s.requires_grad]
        grads = torch.autograd.grad(loss, want + inner, allow_unused=True)
        grads, ends = iter(grads[:len(want)]), grads[len(want):]
        for i, d in zip(range(len(states) - len(inner), len(states)), ends):
            dS[i] = dS[i] if d is None else d
        for name, t in zip(NAMES, leaves):
            if t is not None:
                d = next(grads)
                r["d" + name] = torch.zeros_like(t) if d is None else d
    with torch.no_grad():
        squares = terms(q, k, v, a, b, y, states, up, r["dv"] if "dv" in r else up, dS, scale, g, dtype)
        if form == "sigmoid" and gate is not None:
            squares["dgate"] = squares["dgate"] * torch.sigmoid(-gate).pow(2)
    return {name: (x, squares[name]) for name, x in r.items()}


def terms(q, k, v, a, b, y, states, up, dD, dS, scale, g, dtype):
    """Squares of the terms that a row of each result is the sum of, by name: [N, rows], or broadcast to it.  w
    weighs the errors that were there before y and S are rounded to the rows' type, against that rounding."""
    w = 1.0 if dtype != BF16 else 2.0 ** -16
    N, T, dv = v.shape
    C = -(-T // 64)
    sq, tr = (lambda x: x * x), (lambda x: x.transpose(-1, -2).contiguous())
    cut = lambda t: torch.nn.functional.pad(t, (0, 0) * (t.dim() - 2) + (0, C * 64 - T)).view(N, C, 64, *t.shape[2:])
    q, k, v, b, y, up, dD = (cut(t) for t in (q, k, v, b, y, up, dD))
    G = cut(a.clamp(min=1e-87).log()).cumsum(-1)
    i = torch.arange(64, device=v.device)
    gam = torch.exp(torch.where(i[:, None] >= i, G[..., :, None] - G[..., None, :], -math.inf))
    E, Z, last = sq(torch.exp(G)), sq(torch.exp(G[..., -1:] - G)), sq(torch.exp(G[..., -1]))
    qk, kk, b2 = torch.matmul(q, tr(k)), torch.matmul(k, tr(k)), sq(b)
    strict = torch.where(i[:, None] > i, gam, 0.0)
    mix = sq(torch.linalg.inv(torch.eye(64, device=v.device, dtype=v.dtype) + strict * kk * b[..., None, :]))
    M = sq(scale * gam * qk) * b2[..., None, :]
    q2, k2, up2, dD2, norm = sq(q), sq(k), sq(up), sq(dD), (lambda x: x.sum(-1))
    times = lambda m, x: torch.matmul(m, x[..., None])[..., 0]
    S2, dS2 = sq(torch.stack(states[:C], 1)), sq(torch.stack(dS[1:C + 1], 1))
    # Forward: D, Y = T D, the states.
    d = norm(sq(v)) + E * times(k2, norm(S2))
    y_before = times(mix, d)
    y2 = sq(y) + w * (y_before / dv)[..., None]
    s = torch.zeros(N, device=v.device, dtype=v.dtype)
    S_before = []
    for c in range(C):
        S_before.append(s)
        s = last[:, c] * s + (Z * b2 * norm(k2) * y_before)[:, c].sum(-1) + sq(states[c + 1]).sum((1, 2))
    S2 = S2 + w * (torch.stack(S_before, 1) / S2[0, 0].numel())[..., None, None]
    out = times(M, norm(y2)) + scale ** 2 * E * times(q2, norm(S2))
    # Backward: dY, dD = T^T dY, the states' gradients; then the chunks'.
    dD_before = times(tr(mix), times(tr(M), norm(up2)) + Z * b2 * times(k2, norm(dS2)) * w)
    part = (scale ** 2 * E * norm(q2) * norm(up2) + E * norm(k2) * (dD_before + norm(dD2))).sum(-1)
    ds, before = torch.zeros_like(s), [None] * C
    for c in range(C - 1, -1, -1):
        before[c] = ds
        ds = last[:, c] * ds + part[:, c]
    dS2 = dS2 + (torch.stack(before, 1) / dS2[0, 0].numel())[..., None, None]
    dD2 = dD2 + (dD_before / dv)[..., None]
    P, H = sq(scale * gam) * torch.matmul(up2, tr(y2)), sq(strict) * torch.matmul(dD2, tr(y2))
    L, X = P * b2[..., None, :], H * b2[..., None, :]
    of_up, of_dD, of_y = (torch.matmul(x, tr(m)) for x, m in ((up2, S2), (dD2, S2), (y2, dS2)))
    dq = scale ** 2 * E * norm(of_up) + times(L, norm(k2))
    dk = times(tr(L), norm(q2)) + times(X + tr(X), norm(k2)) + Z * b2 * norm(of_y) + E * norm(of_dD)
    from_state = Z * norm(k2 * of_y)
    db = (sq(qk) * P + sq(kk) * H).sum(-2) + from_state
    pairs = L * sq(qk) + X * sq(kk)
    dG = E * (scale ** 2 * norm(q2 * of_up) + norm(k2 * of_dD)) + pairs.sum(-1) + pairs.sum(-2) + b2 * from_state
    dG[..., -1] += (b2 * from_state).sum(-1) + last * (S2 * dS2).sum((-1, -2))
    dG = dG.flip(-1).cumsum(-1).flip(-1)
    rows = lambda x: x.reshape(N, C * 64)[:, :T]
    shared = lambda x: rows(x).reshape(N // g, g, T).sum(1)
    per_row = lambda x: (x / S2.shape[-2])[:, None]  # a state's rows share its terms
    return dict(out=rows(out), state=per_row(s), dq=shared(dq), dk=shared(dk), dv=rows(norm(dD2)), dgate=rows(dG), dbeta=rows(db),
                dstate=per_row(ds))


def check(race, args, dout, dfinal, dtype, what, **kw):
    """Forward, carry and gradients of one call; (outs, grads)."""
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in args]
    outs = race.race_delta_rule(*leaves, **{"gate_form" if n == "form" else n: x for n, x in kw.items()})
    want = reference(*args, **kw, dout=dout, dfinal=dfinal)
    close("out", outs[0], want["out"], dtype, what)
    close("state", outs[1], want["state"], dtype, what)
    some = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(outs, some, (dout, dfinal))
    for (name, t), d in zip([p for p in zip(NAMES, leaves) if p[1] is not None], grads):
        close("d" + name, d, want["d" + name], dtype, what)
        assert d.dtype == t.dtype
    return outs, grads


# Key and value widths around the tiles' (16, 32, 64, 128 columns), odd ones, and shared key heads; lengths around
# a chunk of 64 and the 16 tokens of the small launch.
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N, Nk, dk, dv", [(2, 2, 64, 64), (4, 2, 128, 128), (3, 1, 33, 17), (2, 2, 96, 50), (3, 3, 16, 256),
                                           (2, 1, 128, 100), (2, 2, 4, 12), (2, 2, 8, 8), (2, 2, 1, 1), (6, 2, 65, 129),
                                           (2, 2, 100, 72), (1, 1, 127, 255)])
def test_forward_and_gradients(race, cuda, N, Nk, dk, dv, dtype):
    for T in (1, 2, 16, 17, 63, 64, 65, 200):
        form, times = "sigmoid" if T % 2 else "log", -(-64 // T)
        *args, dout, dfinal = make(N * times, Nk * times, T, dk, dv, dtype, form, seed=T)
        if T == 65:
            args[5] = None
        what = f"T={T}"
        check(race, args, dout, dfinal, dtype, what, form=form, scale=dk ** -0.5)
        if args[5] is not None:
            out, state = race.race_delta_rule_carry(*args, gate_form=form, scale=dk ** -0.5)
            want = reference(*args, form=form, scale=dk ** -0.5)
            close("out", out, want["out"], dtype, what + " carry"), close("state", state, want["state"], dtype, what + " carry")


# Few streams: their tokens are walked in segments, forward and backward; ends within a segment and at its edges.
@pytest.mark.parametrize("N, Nk, T, dk, dv, dtype", [(1, 1, 2048, 64, 64, F32), (3, 1, 1537, 128, 72, BF16), (2, 2, 1600, 40, 20, BF16),
                                                     (2, 2, 1700, 128, 128, F32)])
def test_tokens_in_segments(race, cuda, N, Nk, T, dk, dv, dtype):
    *args, dout, dfinal = make(N, Nk, T, dk, dv, dtype, seed=3)
    args[3].clamp_(min=-0.5)
    lengths = torch.tensor([T, 511, 1025][:N], dtype=torch.int32, device=cuda)
    check(race, args, dout, dfinal, dtype, "segments", scale=dk ** -0.5, lengths=lengths)
    carried = args[5].clone()
    a = race.race_delta_rule_carry(*args, scale=dk ** -0.5, lengths=lengths)
    b = race.race_delta_rule_carry(*args[:5], carried, scale=dk ** -0.5, lengths=lengths, inplace=True)
    assert b[1] is carried or b[1].data_ptr() == carried.data_ptr()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths, T", [((0, 70, 200, 1), 200), ((64, 65, 63, 128), 129), ((0, 0, 0, 0), 90), ((3, 0, 16, 9), 16)])
def test_padded_batches(race, cuda, lengths, T, dtype):
    N, Nk, dk, dv = 8, 4, 48, 40
    *args, dout, dfinal = make(N, Nk, T, dk, dv, dtype, seed=5)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    dead = torch.arange(T, device=cuda) >= n.repeat_interleave(2)[:, None]
    clean = check(race, args, dout, dfinal, dtype, "padded", scale=0.25, lengths=n)
    # What stands behind the ends is not read, and has no gradient.
    q, k, v, gate, beta, state = (t.clone() for t in args)
    v[dead], gate[dead], beta[dead] = math.nan, math.nan, math.inf
    q[dead[::2]], k[dead[::2]] = math.nan, math.inf
    bad = dout.clone()
    bad[dead] = math.nan
    leaves = [t.requires_grad_(True) for t in (q, k, v, gate, beta, state)]
    outs = race.race_delta_rule(*leaves, scale=0.25, lengths=n.long())
    grads = torch.autograd.grad(outs, leaves, (bad, dfinal))
    for a, b in zip((*clean[0], *clean[1]), (*outs, *grads)):
        assert torch.equal(a, b)
    assert (outs[0][dead] == 0).all()
    for d, mask in zip(grads, (dead[::2], dead[::2], dead, dead, dead)):
        assert (d[mask] == 0).all()
    empty = n.repeat_interleave(2) == 0
    assert torch.equal(outs[1][empty], state[empty]) and torch.equal(grads[5][empty], dfinal[empty])
    # Lengths out of range count as the ends.  (The carry of a few tokens takes another launch.)
    far = torch.where(n == T, n + 1000, torch.where(n == 0, n - 7, n))
    again = race.race_delta_rule_carry(*args, scale=0.25, lengths=far)
    exact = race.race_delta_rule_carry(*args, scale=0.25, lengths=n)
    assert torch.equal(again[0], exact[0]) and torch.equal(again[1], exact[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [7, 150, 1600])
def test_gates_at_their_ends(race, cuda, T, dtype):
    # Gates that forget everything (-inf, and the type's lowest value), that keep everything, or that barely do.
    *args, dout, dfinal = make(2, 2, T, 64, 64, dtype, seed=6)
    lowest = torch.finfo(dtype).min
    args[3][0, 3], args[3][0, T // 2], args[3][1, 0], args[3][1, T - 1] = -math.inf, lowest, 0.0, -0.0
    args[3][1, T // 3] = -199.0
    args[4][1, T // 2], args[4][0, 1], args[4][0, 5] = 0.0, 1.0, 0.0
    leaves = [t.detach().requires_grad_(True) for t in args]
    outs = race.race_delta_rule(*leaves, scale=0.125)
    assert all(torch.isfinite(t).all() for t in outs)
    safe = args[3].double().clamp(min=-1e4)  # e^-1e4 is zero in 64 bits too, without 0 * inf in the derivative
    want = reference(args[0], args[1], args[2], safe, *args[4:], scale=0.125, dout=dout, dfinal=dfinal)
    close("out", outs[0], want["out"], dtype), close("state", outs[1], want["state"], dtype)
    grads = torch.autograd.grad(outs, leaves, (dout, dfinal))
    for name, d in zip(NAMES, grads):
        close("d" + name, d, want["d" + name], dtype)
    # Nothing before a reset reaches what follows it.
    other = [t.clone() for t in args]
    other[0][0, :T // 2], other[2][0, :T // 2], other[5][0] = 3.0, -5.0, 9.0
    other[1][0, :T // 2] = args[1][0, :T // 2].roll(1, -1)
    a, b = race.race_delta_rule_carry(*args, scale=0.125), race.race_delta_rule_carry(*other, scale=0.125)
    # (chunks share sums, whose rounding may differ; what the tokens write does not)
    out_terms, state_terms = want["out"][1], want["state"][1]
    close("out", b[0][:1, T // 2:], (a[0][:1, T // 2:].double(), out_terms[:1, T // 2:]), dtype)
    close("state", b[1][:1], (a[1][:1].double(), state_terms[:1]), dtype)
    # Logits of +-inf and the lowest value: keep and forget.
    logit = torch.full_like(args[3], math.inf)
    kept = race.race_delta_rule_carry(*args[:3], None, *args[4:], scale=0.125)
    sure = race.race_delta_rule_carry(*args[:3], logit, *args[4:], gate_form="sigmoid", scale=0.125)
    assert torch.equal(kept[0], sure[0]) and torch.equal(kept[1], sure[1])
    for x in (-math.inf, lowest):
        gone = race.race_delta_rule_carry(*args[:3], logit.fill_(x), *args[4:], gate_form="sigmoid", scale=0.125)
        want = reference(*args[:3], torch.full_like(safe, -1e4), *args[4:], scale=0.125)
        close("out", gone[0], want["out"], dtype), close("state", gone[1], want["state"], dtype)


@pytest.mark.parametrize("dtype, gate_dtype", [(F32, F32), (BF16, F32)])
def test_without_gates_and_with_gates_in_32_bits(race, cuda, dtype, gate_dtype):
    for T in (9, 130):
        *args, dout, dfinal = make(4, 2, T, 64, 32, dtype, seed=7, gate_dtype=gate_dtype)
        check(race, args, dout, dfinal, dtype, f"T={T}", scale=0.125)
        args[3] = None
        check(race, args, dout, dfinal, dtype, f"T={T} no gate", scale=0.125)


def test_a_nan_stays_in_its_stream_and_after_its_token(race, cuda):
    for T, at in ((12, 5), (300, 130), (1600, 700)):
        for which in range(5):
            *args, _, _ = make(4, 4, T, 32, 32, F32, seed=8)
            clean = race.race_delta_rule_carry(*args)
            args[which][1, at] = math.nan
            out, state = race.race_delta_rule_carry(*args)
            others = [0, 2, 3]
            assert torch.equal(out[others], clean[0][others]) and torch.equal(state[others], clean[1][others])
            # Whole chunks before it are as they were, and it is seen where it belongs.
            start = at // 64 * 64 if T > 16 else at
            assert torch.equal(out[1, :start], clean[0][1, :start]), (T, which)
            assert out[1, at].isnan().all(), (T, which)
            assert which == 0 or (out[1, at + 1:].isnan().all() and state[1].isnan().all()), (T, which)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_inputs_equal_dense_ones(race, cuda, dtype):
    for T, dk, dv in ((1, 64, 64), (100, 64, 64), (100, 40, 24), (1600, 64, 64)):
        *args, dout, dfinal = make(4, 2, T, dk, dv, dtype, seed=9)
        dense = [t.requires_grad_(True) for t in args]
        want = race.race_delta_rule(*dense, scale=0.125)
        want_grads = torch.autograd.grad(want, dense, (dout, dfinal))

        def wide(t, pad):  # rows of a wider tensor
            x = torch.full((*t.shape[:-1], t.shape[-1] + pad), math.nan, dtype=t.dtype, device=cuda)
            x[..., 8:8 + t.shape[-1]] = t
            return x[..., 8:8 + t.shape[-1]]

        def tokens_first(t):  # [T, N, d] in memory
            return t.transpose(0, 1).contiguous().transpose(0, 1)

        def odd(t):  # no piece of a row is aligned
            x = torch.full((t.numel() + 1,), math.nan, dtype=t.dtype, device=cuda)
            x[1:] = t.reshape(-1)
            return x[1:].view(t.shape)

        for how in (lambda t: wide(t, 16), lambda t: wide(t, 13), tokens_first, odd):
            got_in = [how(t.detach()).requires_grad_(True) for t in dense[:3]] + [odd(t.detach()).requires_grad_(True) for t in dense[3:5]]
            got = race.race_delta_rule(*got_in, dense[5], scale=0.125)
            grads = torch.autograd.grad(got, (*got_in, dense[5]), (odd(dout), dfinal))
            for name, a, b in zip(("out", "state", *("d" + n for n in NAMES)), (*got, *grads), (*want, *want_grads)):
                # The loads' widths do not change the sums.
                assert torch.equal(a, b), (T, dk, name)


def test_bucket_probabilities_as_keys_and_broadcast_inputs(race, cuda):
    N, T, L, R, dv = 2, 90, 2, 16, 32
    *args, dout, dfinal = make(N, N, T, L * R, dv, F32, seed=10)
    probs = [torch.softmax(t.view(N, T, L, R), -1) / 2 ** 0.5 for t in args[:2]]  # |k| <= 1
    flat = [t.flatten(2) for t in probs]
    outs, grads = check(race, [*flat, *args[2:]], dout, dfinal, F32, "probabilities")
    leaves = [t.requires_grad_(True) for t in probs] + args[2:]
    got = race.race_delta_rule(*leaves)
    more = torch.autograd.grad(got, leaves[:2], (dout, dfinal))
    assert torch.equal(got[0], outs[0]) and torch.equal(more[1].flatten(2), grads[1])
    # One strength and one gate for all tokens: their gradients are the sums.
    gate, beta = (torch.full((N, 1), x, device=cuda, requires_grad=True) for x in (-0.1, 0.5))
    outs = race.race_delta_rule(*args[:3], gate.expand(N, T), beta.expand(N, T), args[5])
    dg, db = torch.autograd.grad(outs, (gate, beta), (dout, dfinal))
    want = reference(*args[:3], gate.detach().expand(N, T), beta.detach().expand(N, T), args[5], dout=dout, dfinal=dfinal)
    for d, name in ((dg, "dgate"), (db, "dbeta")):
        # T terms of the tokens' tolerance each
        value, square = want[name]
        bound = 8 * tolerance(name, F32) * (value.abs().sum(1) + T * (value.pow(2) + square).mean(1).sqrt())
        assert ((d[:, 0].double() - value.sum(1)).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T, cuts", [(40, (0, 1, 17, 40)), (200, (0, 64, 65, 190, 200)), (1700, (0, 100, 1700)), (30, tuple(range(31)))])
def test_a_split_sequence_gives_the_unsplit_result(race, cuda, T, cuts, dtype):
    *args, _, _ = make(4, 2, T, 64, 64, dtype, seed=11)
    whole = reference(*args, scale=0.125)
    state, outs = args[5].clone(), []
    for a, b in zip(cuts, cuts[1:]):
        out, same = race.race_delta_rule_carry(*(t[:, a:b] for t in args[:5]), state, scale=0.125, inplace=True)
        assert same.data_ptr() == state.data_ptr()
        outs.append(out)
    close("out", torch.cat(outs, 1), whole["out"], dtype), close("state", state, whole["state"], dtype)


def test_gradient_through_a_carried_state(race, cuda):
    *args, dout, dfinal = make(2, 2, 150, 32, 48, F32, seed=12)
    leaves = [t.requires_grad_(True) for t in args]
    out1, mid = race.race_delta_rule(*(t[:, :70] for t in leaves[:5]), leaves[5])
    out2, last = race.race_delta_rule(*(t[:, 70:] for t in leaves[:5]), mid)
    grads = torch.autograd.grad((torch.cat([out1, out2], 1), last), leaves, (dout, dfinal))
    want = reference(*(t.detach() for t in args), dout=dout, dfinal=dfinal)
    for name, d in zip(NAMES, grads):
        close("d" + name, d, want["d" + name], F32)


@pytest.mark.parametrize("T", [90, 1600])
def test_missing_upstream_gradients_and_inputs(race, cuda, T):
    *args, dout, dfinal = make(4, 2, T, 64, 64, F32, seed=13)
    leaves = [t.requires_grad_(True) for t in args]
    outs = race.race_delta_rule(*leaves)
    both = torch.autograd.grad(outs, leaves, (dout, dfinal), retain_graph=True)
    for name, d in zip(NAMES, torch.autograd.grad(outs[0], leaves, dout, retain_graph=True)):
        close("d" + name, d, reference(*(t.detach() for t in args), dout=dout)["d" + name], F32, "out alone")
    want = reference(*(t.detach() for t in args), dfinal=dfinal)
    grads = torch.autograd.grad(outs[1], leaves, dfinal)
    assert (grads[0] == 0).all()
    for name, d in list(zip(NAMES, grads))[1:]:
        close("d" + name, d, want["d" + name], F32, "final alone")
    # Each gradient by itself equals the one computed with the others.
    for i, leaf in enumerate(leaves):
        alone = [t if j == i else t.detach() for j, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(race.race_delta_rule(*alone), leaf, (dout, dfinal))[0], both[i]), NAMES[i]


@pytest.mark.parametrize("form", ["log", "sigmoid"])
def test_gradients_against_differences(race, cuda, form):
    # Differences of the recurrence in 64 bits: h^2 of a third derivative and 2^-53 / h, both far below the tolerance.
    *args, dout, dfinal = make(2, 1, 100, 24, 20, F32, form, seed=14)
    leaves = [t.requires_grad_(True) for t in args]
    grads = torch.autograd.grad(race.race_delta_rule(*leaves, gate_form=form, scale=0.3), leaves, (dout, dfinal))
    h = 1e-6
    for i, name in enumerate(NAMES):
        way = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).to(cuda).double()
        loss = []
        for sign in (1, -1):
            moved = [t.detach().double() + sign * h * way if j == i else t.detach() for j, t in enumerate(leaves)]
            r = reference(*moved, form=form, scale=0.3)
            loss.append(float((r["out"][0] * dout).sum() + (r["state"][0] * dfinal).sum()))
        along = float((grads[i].double() * way).sum())
        slack = tolerance("d" + name, F32) * float(grads[i].double().norm() * way.norm())
        assert abs((loss[0] - loss[1]) / (2 * h) - along) <= slack + 1e-7 * abs(along), name


def test_repeatable_and_empty(race, cuda):
    *args, dout, dfinal = make(6, 2, 500, 64, 64, BF16, seed=15)
    leaves = [t.requires_grad_(True) for t in args]
    runs = []
    for _ in range(3):
        outs = race.race_delta_rule(*leaves)
        runs.append((*outs, *torch.autograd.grad(outs, leaves, (dout, dfinal))))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))
    # No tokens: the state passes; no streams: nothing.
    for N, T in ((3, 0), (0, 5), (0, 0)):
        *args, dout, dfinal = make(N, N, T, 16, 24, F32)
        leaves = [t.requires_grad_(True) for t in args]
        out, final = race.race_delta_rule(*leaves)
        assert out.shape == (N, T, 24) and torch.equal(final, leaves[5])
        grads = torch.autograd.grad((out, final), leaves, (dout, dfinal))
        assert torch.equal(grads[5], dfinal) and all(g.shape == t.shape and (g == 0).all() for g, t in zip(grads[:5], leaves))
        out, final = race.race_delta_rule(*args[:5])
        assert (final == 0).all()
        state = args[5].detach().clone()
        race.race_delta_rule_carry(*(t.detach() for t in args[:5]), state, inplace=True)
        assert torch.equal(state, args[5])


@pytest.mark.parametrize("N, T, dtype", [(4, 200, BF16), (2, 1600, F32)])
def test_other_streams_and_captured_steps(race, cuda, N, T, dtype):
    *args, dout, dfinal = make(N, 2, T, 64, 64, dtype, seed=16)
    want = race.race_delta_rule_carry(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = race.race_delta_rule_carry(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    # A training step and a decode step that advances its state, each replayed on new inputs.
    held = [t.clone().requires_grad_(True) for t in args]
    token, carried = [t[:, :1].clone() for t in args[:5]], args[5].clone()

    def step():
        outs = race.race_delta_rule(*held)
        return (*(o.detach() for o in outs), *torch.autograd.grad(outs, held, (dout, dfinal)))

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), race.race_delta_rule_carry(*token, carried, inplace=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
        decoded, _ = race.race_delta_rule_carry(*token, carried, inplace=True)
    for i in range(3):
        fresh = make(N, 2, T, 64, 64, dtype, seed=20 + i)
        with torch.no_grad():
            for t, x in zip(held, fresh):
                t.copy_(x)
        for t, x in zip(token, fresh):
            t.copy_(x[:, :1])
        before = carried.clone()
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        wd, ws = race.race_delta_rule_carry(*token, before)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), i
        assert torch.equal(decoded, wd) and torch.equal(carried, ws), i


def test_a_live_eager_graph_refuses_the_capture(race, cuda):
    *args, _, _ = make(2, 2, 40, 32, 32, F32, seed=17)
    args[1].requires_grad_(True)
    eager, _ = race.race_delta_rule(*args)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            args[2].mul(2)  # something to record
            race.race_delta_rule(*args)
    del eager


def test_gradients_of_gradients_and_tangents_are_refused(race, cuda):
    *args, _, _ = make(2, 2, 20, 32, 32, F32, seed=18)
    leaves = [t.requires_grad_(True) for t in args]
    out, _ = race.race_delta_rule(*leaves)
    (d,) = torch.autograd.grad(out, leaves[2], torch.ones_like(out, requires_grad=True), create_graph=True)
    with pytest.raises(RuntimeError, match="trying to differentiate race_delta_rule twice"):
        d.sum().backward()
    for grad in (True, False):
        for i in range(6):
            with torch.set_grad_enabled(grad), torch.autograd.forward_ad.dual_level():
                duals = [torch.autograd.forward_ad.make_dual(t.detach(), torch.ones_like(t)) if i == j else t.detach()
                         for j, t in enumerate(args)]
                with pytest.raises(RuntimeError, match="jvp"):
                    race.race_delta_rule(*duals)


def test_refusals(race, cuda):
    q, k, v, gate, beta, state, _, _ = make(4, 2, 20, 32, 24, F32, seed=19)
    n = lambda *s: torch.zeros(s, device=cuda)
    for args, kw, message in [
        ((q[0], k[0], v[0], gate, beta), {}, "q has shape"), ((q, k[:1], v, gate, beta), {}, "k has shape"),
        ((q, k, v[:, :19], gate, beta), {}, "v has shape"), ((q, k, v[:3], gate[:3], beta[:3]), {}, "no multiple"),
        ((q, k, v, gate[:, :19], beta), {}, "gate has shape"), ((q, k, v, gate, beta[:2]), {}, "beta has shape"),
        ((q, k.bfloat16(), v, gate, beta), {}, "dtype"), ((q.half(), k.half(), v.half(), gate, beta), {}, "neither float32 nor bfloat16"),
        ((q, k, v, gate.bfloat16(), beta.bfloat16()), {}, "neither float32 nor of q's dtype"),
        ((q.bfloat16(), k.bfloat16(), v.bfloat16(), gate, beta.bfloat16()), {}, "another dtype than beta"),
        ((q, k, v.cpu(), gate, beta), {}, "CPU"), ((q, k, v, gate, beta.cpu()), {}, "CPU"),
        ((q, k, v, gate, beta, state[:1]), {}, "state has shape"), ((q, k, v, gate, beta, state.double()), {}, "state must be float32"),
        ((q, k, v, gate, beta, state.transpose(1, 2).contiguous().transpose(1, 2)), {}, "strided view"),
        ((q, k, v, gate, beta), dict(lengths=torch.zeros(3, dtype=torch.int32, device=cuda)), "do not divide"),
        ((q, k, v, gate, beta), dict(lengths=n(2)), "int32"),
        ((q, k, v, gate, beta), dict(lengths=torch.zeros(2, dtype=torch.int32)), "rows' device"),
        ((q, k, v, gate, beta), dict(scale=math.inf), "finite"),
        ((n(2, 20, 129), n(2, 20, 129), v, gate, beta), {}, "keys of 1 .. 128"),
        ((q, k, n(4, 20, 257), gate, beta), {}, "values of 1 .. 256"), ((q, k, n(4, 20, 0), gate, beta), {}, "values of 1 .. 256"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            race.race_delta_rule(*args, **kw)
    with pytest.raises(ValueError, match="gate_form"):
        race.race_delta_rule(q, k, v, gate, beta, gate_form="linear")
    state.requires_grad_(True)
    with pytest.raises(RuntimeError, match="in place"):
        race.race_delta_rule_carry(q, k, v, gate, beta, state, inplace=True)
    # A graph that saved the state notices that it was advanced.
    carried = state.detach().clone()
    leaf = torch.ones_like(carried, requires_grad=True)
    product = (leaf * carried).sum()
    race.race_delta_rule_carry(q, k, v, gate, beta, carried, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


@pytest.mark.parametrize("N, T, dtype", [(3, 200, F32), (3, 200, BF16), (1, 1600, BF16), (2, 1600, F32)])
def test_c_entry_with_used_memory(race, cuda, N, T, dtype):
    # Outputs, records and workspaces full of NaN before the calls, and bytes behind them left as they were.
    from race_attention_kernel_amd import abi

    dk, dv = 40, 56
    q, k, v, gate, beta, state, dout, dfinal = make(N, 1, T, dk, dv, dtype, seed=21)
    lengths = torch.tensor([T - 61, 33, 0][:N], dtype=torch.int32, device=cuda)
    kind = abi.RACE_BF16 if dtype == BF16 else abi.RACE_F32
    sh = abi.delta_shape(N, T, dk, dv, key_streams=1, dtype=kind, gate_dtype=kind)
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()

    def full(nbytes):
        return torch.full(((int(nbytes) + 3) // 4 + 64,), math.nan, device=cuda)

    def like(t):
        return torch.full((t.numel() + 64,), math.nan, dtype=t.dtype, device=cuda)

    st, nbytes, rec_bytes = abi.delta_workspace_bytes(sh, True)
    st, back = abi.delta_bwd_workspace_bytes(sh)
    out, final, rec, ws = like(v), like(state), full(rec_bytes), full(max(nbytes, back))
    assert abi.delta_fwd(p(q), p(k), p(v), p(gate), p(beta), p(state), p(lengths), p(out), p(final), p(rec), sh, p(ws), nbytes,
                         stream) == 0
    torch.cuda.synchronize()
    assert ws[(nbytes + 3) // 4:].isnan().all() and rec[(rec_bytes + 3) // 4:].isnan().all()
    ws.fill_(math.nan)
    grads = [like(t) for t in (q, k, v, gate, beta, state)]
    assert abi.delta_bwd(p(q), p(k), p(gate), p(beta), p(lengths), p(dout), p(dfinal), p(rec), *map(p, grads), sh, p(ws), back,
                         stream) == 0
    torch.cuda.synchronize()
    assert ws[(back + 3) // 4:].isnan().all()
    want = reference(q, k, v, gate, beta, state, lengths=lengths, dout=dout, dfinal=dfinal)
    for name, got, t in zip(("out", "state", *("d" + n for n in NAMES)), (out, final, *grads), (v, state, q, k, v, gate, beta, state)):
        assert got[t.numel():].isnan().all(), name
        close(name, got[:t.numel()].view(t.shape), want[name], dtype)


def test_offsets_past_32_bits(race, cuda):
    # 2.4e9 values a tensor: the tokens after a reset near the end against those tokens alone, both ways.
    N, Nk, T, dk, dv, tail = 64, 2, 290_000, 128, 128, 1000
    gen = torch.Generator(device=cuda).manual_seed(1)
    row = lambda n, d: torch.nn.functional.normalize(torch.randn(n, T, d, generator=gen, device=cuda), dim=-1).to(BF16)
    q, k = row(Nk, dk), row(Nk, dk)
    v = torch.randn(N, tail, dv, generator=gen, device=cuda).to(BF16).repeat(1, T // tail, 1)
    gate = torch.full((N, T), -0.01, dtype=BF16, device=cuda)
    gate[:, T - tail] = -math.inf
    beta = torch.full((N, T), 0.5, dtype=BF16, device=cuda)
    leaves = [t.requires_grad_(True) for t in (q, k, v, gate, beta)]
    out, final = race.race_delta_rule(*leaves)
    grads = torch.autograd.grad((out, final), leaves, (v.detach(), torch.ones_like(final)))
    end = [t.detach()[:, -tail:].clone().requires_grad_(True) for t in leaves]
    out2, final2 = race.race_delta_rule(*end)
    want = torch.autograd.grad((out2, final2), end, (v.detach()[:, -tail:], torch.ones_like(final)))
    for name, a, b in zip(("out", "dq", "dk", "dv", "dgate", "dbeta"), (out, *grads), (out2, *want)):
        a, b = a.detach()[:, -tail:].double(), b.detach().double()
        if name == "dgate":
            a, b = a[:, 1:], b[:, 1:]
        # Chunks start at other tokens: both sides are rounded, independently.
        assert (a - b).norm() <= 2 ** 0.5 * 2.0 ** -7 * b.norm(), name
    assert (final - final2).norm() <= 2 ** 0.5 * 2.0 ** -15 * final2.norm()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("stride", [1 << 22, (1 << 22) - 1, (1 << 22) + 1])
@pytest.mark.parametrize("T", [5, 70])
def test_the_longest_token_stride(race, cuda, T, stride, dtype):
    # Rows up to 2^22 values apart are read in place, those further apart from a copy.
    *args, _, _ = make(2, 2, T, 33, 48, dtype, seed=22)
    want = race.race_delta_rule_carry(*args)
    wide = torch.full((T * stride + 64,), math.nan, dtype=dtype, device=cuda)
    view = lambda t: torch.as_strided(wide, t.shape, (96, stride, 1))
    for i in range(3):
        moved = list(args)
        moved[i] = view(args[i])
        moved[i].copy_(args[i])
        got = race.race_delta_rule_carry(*moved)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
        wide.fill_(math.nan)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_streams_without_tokens_among_those_in_segments(race, cuda, dtype):
    T = 1600
    *args, dout, dfinal = make(3, 1, T, 64, 48, dtype, seed=23)
    lengths = torch.tensor([0, T - 5, 1], dtype=torch.int32, device=cuda)
    outs, grads = check(race, args, dout, dfinal, dtype, "segments", scale=0.125, lengths=lengths)
    assert (outs[0][0] == 0).all() and torch.equal(outs[1][0], args[5][0]) and torch.equal(grads[5][0], dfinal[0])
    for d in grads[2:5]:
        assert (d[0] == 0).all() and (d[2, 1:] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 33])
def test_one_row_for_all_tokens(race, cuda, d, dtype):
    # Token strides of zero, and rows that overlap, with padding behind them.
    N, T = 4, 100
    *args, dout, dfinal = make(N, N, T, d, d, dtype, seed=24)
    lengths = torch.tensor([100, 64, 70, 3], dtype=torch.int32, device=cuda)
    same = [t[:, :1].expand(N, T, d) for t in args[:3]]
    slide = args[2].reshape(-1)[:3 * 2048 + T * 8 + d].as_strided((N, T, d), (2048, 8, 1))
    for q, k, v in ((same[0], same[1], same[2]), (args[0], args[1], slide)):
        dense = [t.contiguous() for t in (q, k, v)]
        got = race.race_delta_rule_carry(q, k, v, *args[3:], scale=0.125, lengths=lengths)
        want = race.race_delta_rule_carry(*dense, *args[3:], scale=0.125, lengths=lengths)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        grads = []
        for rows in ((q, k, v), dense):
            leaves = [t.detach().requires_grad_(True) for t in rows]
            grads.append(torch.autograd.grad(race.race_delta_rule(*leaves, *args[3:], scale=0.125, lengths=lengths), leaves, (dout, dfinal)))
        assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_most_streams(race, cuda, dtype):
    N, T, d = 65535, 3, 8
    *args, dout, dfinal = make(N, N // 3, T, d, d, dtype, seed=25)
    leaves = [t.detach().requires_grad_(True) for t in args]
    outs = race.race_delta_rule(*leaves, scale=0.5)
    grads = torch.autograd.grad(outs, leaves, (dout, dfinal))
    stepped = race.race_delta_rule_carry(*args, scale=0.5)
    for part in (slice(0, 300), slice(N - 300, N)):
        keys = slice(part.start // 3, part.stop // 3)
        some = [t[keys] if i < 2 else t[part] for i, t in enumerate(args)]
        want = reference(*some, scale=0.5, dout=dout[part], dfinal=dfinal[part])
        for name, got in (("out", outs[0]), ("state", outs[1]), ("out", stepped[0]), ("state", stepped[1])):
            close(name, got.detach()[part], want[name], dtype)
        for i, name in enumerate(NAMES):
            close("d" + name, grads[i][keys if i < 2 else part], want["d" + name], dtype)


def test_one_long_stream(race, cuda):
    # A million tokens in 256 segments, against two calls that split them elsewhere; both keep the tolerance.
    T, cut = 1 << 20, 600_011
    *args, dout, dfinal = make(1, 1, T, 64, 64, F32, seed=26)
    args[3] = args[3] * 0.01  # decays of hundreds of tokens
    leaves = [t.detach().requires_grad_(True) for t in args]
    out, state = race.race_delta_rule(*leaves, scale=0.125)
    grads = torch.autograd.grad((out, state), leaves, (dout, dfinal))
    o1, mid = race.race_delta_rule(*(t[:, :cut] for t in leaves[:5]), leaves[5], scale=0.125)
    o2, last = race.race_delta_rule(*(t[:, cut:] for t in leaves[:5]), mid, scale=0.125)
    split = torch.autograd.grad((torch.cat([o1, o2], 1), last), leaves, (dout, dfinal))
    for name, a, b in zip(("out", "state", *("d" + n for n in NAMES)), (out, state, *grads), (torch.cat([o1, o2], 1), last, *split)):
        err = (a.detach().double() - b.detach().double()).norm() / b.detach().double().norm()
        say(name, f"{float(err):.1e}")
        assert err <= 2 * tolerance(name, F32), name
