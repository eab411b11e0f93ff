"""The gated linear recurrence against its definition in 64 bits, token by token.

Tolerances come from the arithmetic.  With u = 2^-24 (half a step of fp32), a
gate value costs at most 8 u relative (the exponential and the reciprocal are
good to one step, 2 u each, and three roundings between them), its product with x
one more, and joining the runs of a tile adds at most 32 sums on top.  With
M_t = a_t M_{t-1} + |u_t| (every term of h_t by magnitude) and M2_t = sum over
the terms of magnitude times age, h_t is off by at most u (9 M2_t + 32 M_t),
plus half a step of the output's type.  lambda is bounded the same way,
backward; a product of both by the sum of its factors' errors.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from gpu_util import say

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


def _np(t):
    return t.detach().cpu().double().numpy()


def _bounded_scan(a, u, h0, reverse=False):
    """h [T], M, M2 of h_t = a_t h_{t-1} + u_t (reverse: from the last to the first)."""
    T = a.shape[1]
    h, m, m2 = h0.copy(), np.abs(h0), np.abs(h0)
    out = [np.empty_like(a) for _ in range(3)]
    for t in (range(T - 1, -1, -1) if reverse else range(T)):
        at = a[:, t]
        m2 = at * (m2 + m) + np.abs(u[:, t])
        m = at * m + np.abs(u[:, t])
        h = at * h + u[:, t]
        for o, v in zip(out, (h, m, m2)):
            o[:, t] = v
    return out


def _err(m, m2):
    return U * (9 * m2 + 32 * m)


def reference(x, gate, state, lengths, form, complement, dout=None, dfinal=None, dtype=torch.float32):
    """name -> (value, bound) of every output, in 64 bits."""
    x, gate = _np(x), _np(gate)
    N, T, D = x.shape
    s0 = np.zeros((N, D)) if state is None else _np(state)
    if form == "sigmoid":
        t = np.exp(-np.abs(gate))
        a, b = np.where(gate >= 0, 1 / (1 + t), t / (1 + t)), np.where(gate >= 0, t / (1 + t), 1 / (1 + t))
        slope = b
    else:
        a, b, slope = np.exp(gate), -np.expm1(gate), np.ones_like(gate)
    if not complement:
        b = np.ones_like(b)
    live = np.ones((N, T, 1), bool)
    if lengths is not None:
        n = np.repeat(lengths.cpu().numpy(), N // len(lengths))
        live = (np.arange(T)[None] < n[:, None])[..., None]
    a, b, x = np.where(live, a, 1.0), np.where(live, b, 0.0), np.where(live, x, 0.0)
    h, m, m2 = _bounded_scan(a, b * x, s0)
    half = HALF[dtype]
    out = np.where(live, h, 0)
    err = _err(m, m2)
    res = {"out": (out, np.where(live, err + half * np.abs(out), 0.0)),
           "final": (h[:, -1] if T else s0, err[:, -1] + U * np.abs(h[:, -1]) if T else np.zeros_like(s0))}
    if dout is None:
        return res
    dout, dfinal = np.where(live, _np(dout), 0.0), np.zeros((N, D)) if dfinal is None else _np(dfinal)
    # mu_t = a_t lambda_t is the same recurrence run backward.
    mu, mm, mm2 = _bounded_scan(a, a * dout, dfinal, reverse=True)
    nxt = lambda y, end: np.concatenate([y[:, 1:], end[:, None]], axis=1)
    lam = dout + nxt(mu, dfinal)
    lerr = nxt(_err(mm, mm2), U * np.abs(dfinal)) + U * np.abs(lam)
    before = np.concatenate([s0[:, None], h[:, :-1]], axis=1)
    berr = np.concatenate([np.zeros_like(s0)[:, None], err[:, :-1]], axis=1)
    e = before - x if complement else before
    eerr = berr + U * np.abs(before)
    sl = np.where(live, slope, 0.0) * a
    dx, dg = lam * b, lam * sl * e
    res["dx"] = (dx, 2 * np.abs(b) * lerr + (10 * U + half) * np.abs(dx))
    res["dgate"] = (dg, 2 * sl * (np.abs(e) * lerr + (np.abs(lam) + lerr) * eerr) + (24 * U + half) * np.abs(dg))
    res["dstate"] = (mu[:, 0], _err(mm, mm2)[:, 0] + U * np.abs(mu[:, 0]))
    return res


def check(got, want, label):
    value, bound = want
    err = np.abs(_np(got) - value)
    worst = float((err / (bound + 1e-300)).max()) if err.size else 0.0
    say(label, f"{worst:.3f} of the bound")
    assert np.isfinite(_np(got)).all(), label
    assert (err <= bound + 1e-37).all(), (label, worst)


def make(N, T, D, dtype, form, seed, device, state=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, T, D, generator=g).to(dtype)
    gate = 1.5 * torch.randn(N, T, D, generator=g) + 2.0
    if form == "log":
        gate = torch.nn.functional.logsigmoid(gate)
    s = torch.randn(N, D, generator=g) if state else None
    dout = torch.randn(N, T, D, generator=g).to(dtype)
    dfinal = torch.randn(N, D, generator=g)
    to = lambda t: None if t is None else t.to(device)
    return to(x), to(gate.to(dtype)), to(s), to(dout), to(dfinal)


SHAPES = [(1, 1, 1), (3, 1, 64), (2, 16, 64), (2, 17, 68), (2, 255, 64), (1, 256, 4), (2, 257, 130), (3, 700, 33),
          (5, 63, 1), (1, 64, 7), (1, 65, 64), (2, 5000, 64), (1, 1300, 9), (300, 300, 60)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("form, complement", [("sigmoid", True), ("sigmoid", False), ("log", True), ("log", False)])
@pytest.mark.parametrize("N, T, D", SHAPES)
def test_forward_and_gradients(race, cuda, N, T, D, form, complement, dtype):
    x, gate, state, dout, dfinal = make(N, T, D, dtype, form, 7 * T + D, cuda)
    for t in (x, gate, state):
        t.requires_grad_(True)
    out, final = race.race_gated_scan(x, gate, state, gate_form=form, complement=complement)
    assert out.dtype == dtype and out.shape == x.shape and final.dtype == torch.float32
    dx, dg, ds = torch.autograd.grad((out, final), (x, gate, state), (dout, dfinal))
    ref = reference(x, gate, state, None, form, complement, dout, dfinal, dtype)
    for name, got in (("out", out), ("final", final), ("dx", dx), ("dgate", dg), ("dstate", ds)):
        check(got, ref[name], f"scan {form} {complement} {dtype} {N}x{T}x{D} {name}")
    # Without a gradient (and, for a few tokens, token by token): the same within both bounds.
    o2, f2 = race.race_gated_scan_carry(x.detach(), gate.detach(), state.detach(), gate_form=form,
                                        complement=complement)
    check(o2, ref["out"], "carry out")
    check(f2, ref["final"], "carry final")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N, T, D, lengths", [(4, 300, 64, [0, 1, 300, 299]), (6, 700, 33, [0, 256, 257]),
                                              (3, 9, 64, [0, 9, 4]), (2, 6000, 64, [0, 2500]), (4, 1030, 8, [1024, 700])])
def test_padded_batches(race, cuda, N, T, D, lengths, dtype):
    x, gate, state, dout, dfinal = make(N, T, D, dtype, "sigmoid", T, cuda)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    # What lies behind a sequence is not read.
    past = (torch.arange(T, device=cuda) >= n.repeat_interleave(N // len(lengths))[:, None])[..., None].expand_as(x)
    clean = [t.clone() for t in (x, gate, dout)]
    for t, bad in ((x, float("nan")), (gate, float("inf")), (dout, float("nan"))):
        t.masked_fill_(past, bad)
    for t in (x, gate, state):
        t.requires_grad_(True)
    out, final = race.race_gated_scan(x, gate, state, lengths=n)
    grads = torch.autograd.grad((out, final), (x, gate, state), (dout, dfinal))
    ref = reference(clean[0], clean[1], state, n, "sigmoid", True, clean[2], dfinal, dtype)
    for name, got in (("out", out), ("final", final), ("dx", grads[0]), ("dgate", grads[1]), ("dstate", grads[2])):
        check(got, ref[name], f"padded {N}x{T}x{D} {dtype} {name}")
    o2, f2 = race.race_gated_scan_carry(x.detach(), gate.detach(), state.detach(), lengths=n.long())
    check(o2, ref["out"], "carry out")
    check(f2, ref["final"], "carry final")


def test_lengths_past_the_ends_count_as_the_ends(race, cuda):
    x, gate, state, _, _ = make(2, 40, 64, torch.float32, "sigmoid", 3, cuda)
    out, final = race.race_gated_scan(x, gate, state, lengths=torch.tensor([-5, 1000], dtype=torch.int32, device=cuda))
    want, wfinal = race.race_gated_scan(x, gate, state)
    assert torch.equal(out[1], want[1]) and torch.equal(final[1], wfinal[1])
    assert (out[0] == 0).all() and torch.equal(final[0], state[0])


def test_lengths_of_64_bits(race, cuda):
    x = torch.randn(2, 40, 24, device=cuda)
    near = torch.tensor([40, 0], dtype=torch.int32, device=cuda)
    far = torch.tensor([2 ** 32 + 7, -2 ** 33], device=cuda)
    for a, b in zip(race.race_gated_scan(x, x, lengths=far), race.race_gated_scan(x, x, lengths=near)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_inputs_equal_dense_ones(race, cuda, dtype):
    N, T, D = 3, 530, 96
    x, gate, state, dout, _ = make(N, T, D, dtype, "sigmoid", 5, cuda)
    both = torch.stack([x, gate], dim=2)                       # [N, T, 2, D]: one projection's rows
    turned = both.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3)  # tokens outermost in memory
    shifted = torch.empty(N * T * 2 * D + 1, dtype=dtype, device=cuda)[1:].view(N, T, 2, D).copy_(both)
    apart = torch.empty(N, T, 2, D, 2, dtype=dtype, device=cuda)[..., 0].copy_(both)
    far = torch.empty(T, (1 << 20) + 16, dtype=dtype, device=cuda)[:, :N * 2 * D].view(T, N, 2, D).copy_(
        both.permute(1, 0, 2, 3)).permute(1, 0, 2, 3)          # tokens megabytes apart
    odd = torch.empty(N, T, 2, D + 1, dtype=dtype, device=cuda)[..., :D].copy_(both)
    want = race.race_gated_scan(x, gate, state)
    for src in (both, turned, shifted, apart, far, odd):
        xs, gs = src[:, :, 0], src[:, :, 1]
        got = race.race_gated_scan(xs, gs, state)
        exact = src is not odd  # an odd stride takes the narrow kernel, another order of sums
        for g, w in zip(got, want):
            assert torch.equal(g, w) if exact else torch.allclose(g.float(), w.float(), rtol=2 ** -7, atol=1e-5)
    # One gate for all channels, and one input for all streams: autograd adds their gradients up.
    g1 = gate[:, :, :1].clone().requires_grad_(True)
    x1 = x[:1].clone().requires_grad_(True)
    out, _ = race.race_gated_scan(x1.expand(N, T, D), g1.expand(N, T, D), state)
    dx1, dg1 = torch.autograd.grad(out, (x1, g1), dout)
    xf, gf = x1.detach().expand(N, T, D), g1.detach().expand(N, T, D)
    ref = reference(xf, gf, state, None, "sigmoid", True, dout, None, dtype)
    assert np.abs(_np(dx1) - ref["dx"][0].sum(0, keepdims=True)).max() <= \
        (ref["dx"][1].sum(0) + HALF[dtype] * 4 * np.abs(ref["dx"][0]).sum(0)).max()
    assert np.abs(_np(dg1) - ref["dgate"][0].sum(2, keepdims=True)).max() <= \
        (ref["dgate"][1].sum(2) + HALF[dtype] * 4 * np.abs(ref["dgate"][0]).sum(2)).max()


@pytest.mark.parametrize("T, cuts", [(40, [1, 2, 17]), (900, [256, 600]), (9000, [4000, 8999])])
def test_a_split_sequence_gives_the_unsplit_result(race, cuda, T, cuts):
    x, gate, state, _, _ = make(2, T, 64, torch.float32, "log", T, cuda)
    ref = reference(x, gate, state, None, "log", True)
    carried, outs, at = state.clone(), [], 0
    for cut in cuts + [T]:
        o, s = race.race_gated_scan_carry(x[:, at:cut], gate[:, at:cut], carried, gate_form="log", inplace=True)
        assert s is carried or s.data_ptr() == carried.data_ptr()
        outs.append(o)
        at = cut
    check(torch.cat(outs, 1), ref["out"], "split out")
    check(carried, ref["final"], "split final")


def test_gradient_through_a_carried_state(race, cuda):
    x, gate, state, dout, dfinal = make(2, 600, 64, torch.float32, "sigmoid", 9, cuda)
    for t in (x, gate, state):
        t.requires_grad_(True)
    o1, s1 = race.race_gated_scan(x[:, :301], gate[:, :301], state)
    o2, s2 = race.race_gated_scan(x[:, 301:], gate[:, 301:], s1)
    grads = torch.autograd.grad((torch.cat([o1, o2], 1), s2), (x, gate, state), (dout, dfinal))
    ref = reference(x, gate, state, None, "sigmoid", True, dout, dfinal)
    for name, got in zip(("dx", "dgate", "dstate"), grads):
        value, bound = ref[name]
        assert (np.abs(_np(got) - value) <= 2 * bound + 1e-37).all(), name


def test_missing_upstream_gradients_and_inputs(race, cuda):
    x, gate, state, dout, dfinal = make(2, 300, 64, torch.float32, "sigmoid", 10, cuda)
    ref = reference(x, gate, None, None, "sigmoid", True, dout, None)
    x.requires_grad_(True)
    out, final = race.race_gated_scan(x, gate)
    check(torch.autograd.grad(out, x, dout, retain_graph=True)[0], ref["dx"], "out alone, zero state")
    ref = reference(x, gate, None, None, "sigmoid", True, torch.zeros_like(dout), dfinal)
    check(torch.autograd.grad(final, x, dfinal)[0], ref["dx"], "final alone")
    s = state.clone().requires_grad_(True)
    out, final = race.race_gated_scan(x.detach(), gate, s)
    ref = reference(x, gate, state, None, "sigmoid", True, dout, dfinal)
    check(torch.autograd.grad((out, final), s, (dout, dfinal))[0], ref["dstate"], "state alone")


@pytest.mark.parametrize("form", ["sigmoid", "log"])
def test_gradients_against_differences(race, cuda, form):
    x, gate, state, dout, dfinal = make(2, 270, 68, torch.float32, form, 11, cuda)
    leaves = [t.requires_grad_(True) for t in (x, gate, state)]
    out, final = race.race_gated_scan(*leaves, gate_form=form)
    grads = torch.autograd.grad((out, final), leaves, (dout, dfinal))
    step = 2.0 ** -7
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        way = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(i)).to(cuda)
        loss = []
        for sign in (1, -1):
            moved = [t.detach() + sign * step * way if j == i else t.detach() for j, t in enumerate(leaves)]
            o, f = race.race_gated_scan_carry(*moved, gate_form=form)
            loss.append(float((o.double() * dout).sum() + (f.double() * dfinal).sum()))
        along = float((grad.double() * way).sum())
        # The third-order term of a central difference at this step, and 2^-24 of the summed magnitudes.
        size = float((out.detach().double().abs() * dout.abs()).sum())
        assert abs((loss[0] - loss[1]) / (2 * step) - along) <= 1e-3 * float(
            (grad.double().abs() * way.abs()).sum()) + size * U / step, (form, i)


def test_gates_at_their_ends(race, cuda):
    inf = float("inf")
    x, gate, state, dout, _ = make(1, 40, 64, torch.float32, "sigmoid", 12, cuda)
    gate[:, 5], gate[:, 6], gate[:, 20], gate[:, 30] = inf, -inf, 200.0, -200.0
    x.requires_grad_(True), gate.requires_grad_(True)
    out, _ = race.race_gated_scan(x, gate, state)
    grads = torch.autograd.grad(out, (x, gate), dout)
    assert torch.equal(out[:, 5], out[:, 4]) and torch.equal(out[:, 6], x[:, 6])  # keeps all, takes all
    assert torch.equal(out[:, 20], out[:, 19]) and torch.equal(out[:, 30], x[:, 30])
    assert all(torch.isfinite(g).all() for g in grads)
    assert (grads[1][:, [5, 6, 20, 30]] == 0).all()
    # A log gate of -inf starts a new sequence: what came before leaves no trace.
    xl, gl, sl, dl, _ = make(1, 600, 64, torch.float32, "log", 13, cuda)
    gl[:, 300] = -inf
    xl.requires_grad_(True), gl.requires_grad_(True)
    o, f = race.race_gated_scan(xl, gl, sl, gate_form="log", complement=False)
    dx, dg = torch.autograd.grad((o, f), (xl, gl), (dl, torch.zeros_like(f)))
    o2, f2 = race.race_gated_scan(xl[:, 300:], gl[:, 300:], gate_form="log", complement=False)
    ref = reference(xl[:, 300:], gl[:, 300:], None, None, "log", False)
    check(o[:, 300:], ref["out"], "after the start")
    check(f, ref["final"], "final after the start")
    assert (dg[:, 300] == 0).all() and torch.isfinite(dx).all() and torch.isfinite(dg).all()


def test_a_nan_stays_in_its_channel_and_after_its_token(race, cuda):
    x, gate, state, _, _ = make(2, 700, 64, torch.float32, "sigmoid", 14, cuda)
    want, _ = race.race_gated_scan(x, gate, state)
    x[1, 400, 17] = float("nan")
    out, _ = race.race_gated_scan(x, gate, state)
    bad = torch.isnan(out)
    assert bad[1, 400:, 17].all() and int(bad.sum()) == 300
    assert torch.equal(out[~bad], want[~bad])


def test_repeatable_and_empty(race, cuda):
    x, gate, state, dout, dfinal = make(4, 3000, 64, torch.bfloat16, "sigmoid", 15, cuda)
    leaves = [t.requires_grad_(True) for t in (x, gate, state)]

    def once():
        out, final = race.race_gated_scan(*leaves)
        return (out, final, *torch.autograd.grad((out, final), leaves, (dout, dfinal)))

    assert all(torch.equal(a, b) for a, b in zip(once(), once()))
    for N, T in ((0, 5), (3, 0)):
        s = torch.randn(N, 64, device=cuda, requires_grad=True)
        e = torch.empty(N, T, 64, device=cuda, requires_grad=True)
        out, final = race.race_gated_scan(e, e, s)
        assert out.shape == e.shape and torch.equal(final, s)
        (ds,) = torch.autograd.grad(final, s, torch.ones_like(final))
        assert torch.equal(ds, torch.ones_like(s))
        _, zero = race.race_gated_scan(e, e)
        assert (zero == 0).all() and zero.shape == (N, 64)


def test_other_streams_and_captured_steps(race, cuda):
    x, gate, state, dout, dfinal = make(2, 2100, 64, torch.bfloat16, "sigmoid", 16, cuda)
    want = race.race_gated_scan(x, gate, state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = race.race_gated_scan(x, gate, state)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    # A training step and a decode step that advances its state, each replayed on new inputs.
    xs, gs, ss = (t.clone().requires_grad_(True) for t in (x, gate, state))
    xd, gd = x[:, :1].clone(), gate[:, :1].clone()
    carried = state.clone()

    def step():
        out, final = race.race_gated_scan(xs, gs, ss)
        return (out.detach(), final.detach(), *torch.autograd.grad((out, final), (xs, gs, ss), (dout, dfinal)))

    with torch.cuda.stream(side):
        step(), race.race_gated_scan_carry(xd, gd, carried, inplace=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
        decoded, _ = race.race_gated_scan_carry(xd, gd, carried, inplace=True)
    for i in range(3):
        a, b, s, _, _ = make(2, 2100, 64, torch.bfloat16, "sigmoid", 20 + i, cuda)
        with torch.no_grad():
            xs.copy_(a), gs.copy_(b), ss.copy_(s)
        xd.copy_(a[:, :1]), gd.copy_(b[:, :1])
        before = carried.clone()
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        wd, ws = race.race_gated_scan_carry(xd, gd, before)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, eager)), i
        assert torch.equal(decoded, wd) and torch.equal(carried, ws), i


def test_refusals(race, cuda):
    x, gate, state, _, _ = make(2, 20, 64, torch.float32, "sigmoid", 18, cuda)
    for args, kw, message in [
        ((x[0], gate[0]), {}, "x has shape"), ((x, gate[:, :19]), {}, "gate has shape"), ((x, gate.bfloat16()), {}, "another dtype"),
        ((x.half(), gate.half()), {}, "neither float32 nor bfloat16"), ((x, gate.cpu()), {}, "CPU"),
        ((x, gate, state[:1]), {}, "state has shape"), ((x, gate, state.double()), {}, "state must be float32"),
        ((x, gate, state.t().contiguous().t()), {}, "strided view"),
        ((x, gate), dict(lengths=torch.zeros(3, dtype=torch.int32, device=cuda)), "do not divide"),
        ((x, gate), dict(lengths=torch.zeros(2, device=cuda)), "int32"),
        ((x, gate), dict(lengths=torch.zeros(2, dtype=torch.int32)), "rows' device"),
        ((x[..., :0], gate[..., :0]), {}, "1 .. 65536 channels"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            race.race_gated_scan(*args, **kw)
    state.requires_grad_(True)
    with pytest.raises(RuntimeError, match="in place"):
        race.race_gated_scan_carry(x, gate, state, inplace=True)
    # A graph that saved the state notices that it was advanced.
    carried = state.detach().clone()
    leaf = torch.ones_like(carried, requires_grad=True)
    product = (leaf * carried).sum()
    race.race_gated_scan_carry(x, gate, carried, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


def test_c_entry_with_used_memory(race, cuda):
    # Outputs, records and workspace full of NaN before the calls; two streams of lengths.
    from race_attention_kernel_amd import abi

    N, T, D = 2, 3000, 64
    x, gate, state, dout, dfinal = make(N, T, D, torch.float32, "sigmoid", 19, cuda)
    sh = abi.scan_shape(N, T, D)
    n = torch.tensor([3000, 1500], dtype=torch.int32, device=cuda)
    st, nbytes, floats = abi.gated_scan_workspace_bytes(sh)
    _, back, _ = abi.gated_scan_workspace_bytes(sh, True)
    nan = lambda *s: torch.full(s, float("nan"), device=cuda)
    ws, rec, out, final = nan(max(nbytes, back) // 4 + 4), nan(floats), nan(N, T, D), nan(N, D)
    dx, dg, ds = nan(N, T, D), nan(N, T, D), nan(N, D)
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()
    assert abi.gated_scan_fwd(p(x), p(gate), p(state), p(n), p(out), p(final), p(rec), sh, p(ws), nbytes, stream) == 0
    ws.fill_(float("nan"))
    assert abi.gated_scan_bwd(p(x), p(gate), p(n), p(dout), p(dfinal), p(rec), p(dx), p(dg), p(ds), sh, p(ws), back,
                              stream) == 0
    torch.cuda.synchronize()
    ref = reference(x, gate, state, n, "sigmoid", True, dout, dfinal)
    for name, got in (("out", out), ("final", final), ("dx", dx), ("dgate", dg), ("dstate", ds)):
        check(got, ref[name], "c entry " + name)
    assert abi.gated_scan_fwd(p(x), p(gate), p(state), p(n), p(out), p(final), p(rec), sh, p(ws), nbytes - 4, stream) == 1


def test_a_live_eager_graph_refuses_the_capture(race, cuda):
    # The backward would wait for the default stream inside the capture.
    x, gate, _, _, _ = make(1, 40, 64, torch.float32, "sigmoid", 17, cuda)
    x.requires_grad_(True)
    eager, _ = race.race_gated_scan(x, gate)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            gate.mul(2)  # something to record
            race.race_gated_scan(x, gate)
    del eager


def test_offsets_past_32_bits(race, cuda):
    # 4.6 GB of rows: the last tokens of the whole against those tokens alone.
    N, T, D = 1, 17600, 65536
    gen = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(N, T, D, generator=gen, device=cuda)
    gate = torch.full((1, 1, 1), 0.5, device=cuda).expand(N, T, D)
    gate = torch.empty(T, D, device=cuda).fill_(0.5)[None]
    out, final = race.race_gated_scan(x, gate)
    tail = 200  # sigmoid(0.5)^150 is below 2^-100: nothing older is left
    o, f = race.race_gated_scan(x[:, -tail:], gate[:, -tail:])
    assert torch.allclose(out[:, -50:], o[:, -50:], rtol=1e-5, atol=1e-5)
    assert torch.allclose(final, f, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("layout", ["shifted", "apart", "far"])
def test_a_live_eager_graph_refuses_the_capture_of_copied_rows(race, cuda, layout):
    # Rows that the op copies first are the caller's leaves all the same.
    if layout == "shifted":  # not 16-byte aligned
        x = torch.randn(1 * 40 * 64 + 1, device=cuda)[1:].view(1, 40, 64)
    elif layout == "apart":  # the last dimension strided
        x = torch.randn(1, 40, 64, 2, device=cuda)[..., 0]
    else:  # tokens further apart than the kernels address
        x = torch.randn(40, (1 << 20) + 16, device=cuda)[None, :, :64]
    gate = torch.randn(1, 40, 64, device=cuda)
    x.requires_grad_(True)
    assert x.is_leaf
    eager, _ = race.race_gated_scan(x, gate)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            gate.mul(2)  # something to record
            race.race_gated_scan(x, gate)
    del eager


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [4, 68, 5])
def test_the_longest_token_stride(race, cuda, D, dtype):
    # Lanes past the channels step over rows 2^20 values apart too; they read and write nothing.
    T, stride = 300, 1 << 20
    x, gate, state, dout, dfinal = make(1, T, D, dtype, "sigmoid", 21, cuda)
    wide = torch.full((T, stride), float("nan"), dtype=dtype, device=cuda)
    far = wide[None, :, :D]
    assert far.stride(1) == stride
    for i, rows in enumerate((x, gate)):  # each of the two in turn
        far.copy_(rows)
        leaves = [t.detach().requires_grad_(True) for t in ((far, gate) if i == 0 else (x, far))]
        out, final = race.race_gated_scan(*leaves, state)
        grads = torch.autograd.grad((out, final), leaves, (dout, dfinal))
        ref = reference(x, gate, state, None, "sigmoid", True, dout, dfinal, dtype)
        for name, got in (("out", out), ("final", final), ("dx", grads[0]), ("dgate", grads[1])):
            check(got, ref[name], f"stride 2^20 D{D} {dtype} {name}")


# Training steps as large calls launch them (tests/test_operators_cpu.py pins the shapes):
# 64 channels a workgroup and 128-token backward tiles where those workgroups fill the
# device, 128 channels where wider ones do, few workgroups split over the tokens, and
# rows past the caches.  The bound above holds: whatever the tile, the joins of one are
# fewer than 32, and the later tiles' are covered by the terms' ages.
LARGE = [(105, 1700, 128, torch.float32, "sigmoid", True, None), (24, 600, 520, torch.float32, "log", False, None),
         (24, 600, 520, torch.bfloat16, "sigmoid", True, [600, 599, 256, 257, 128, 1, 0, 384]),
         (24, 600, 520, torch.float32, "log", False, [600, 0, 511, 513]),
         (210, 1700, 128, torch.bfloat16, "sigmoid", True, None), (2, 1500, 260, torch.float32, "sigmoid", False, [1500, 700]),
         (39, 640, 260, torch.bfloat16, "sigmoid", True, [640, 1, 321]), (32, 640, 260, torch.bfloat16, "log", True, [640, 1, 321, 0]),
         (2, 45000, 256, torch.float32, "sigmoid", True, [45000, 44000]),
         (8, 65536, 64, torch.bfloat16, "sigmoid", True, None)]


@pytest.mark.parametrize("N, T, D, dtype, form, complement, lengths", LARGE)
def test_training_steps_of_large_calls(race, cuda, N, T, D, dtype, form, complement, lengths):
    x, gate, state, dout, dfinal = make(N, T, D, dtype, form, 31 * T + D, cuda)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda) if lengths else None
    for t in (x, gate, state):
        t.requires_grad_(True)
    out, final = race.race_gated_scan(x, gate, state, gate_form=form, complement=complement, lengths=n)
    grads = torch.autograd.grad((out, final), (x, gate, state), (dout, dfinal))
    got = dict(zip(("out", "final", "dx", "dgate", "dstate"), (out, final, *grads)))
    assert all(bool(torch.isfinite(t).all()) for t in got.values())
    # Streams are computed apart: some of every length against the definition, all their channels.
    group = N // len(lengths) if lengths else N
    few = sorted({*range(0, N, group), *range(0, N, 16), N - 1}) if T < 10000 else [N - 1]
    part = lambda t: t.detach()[few]
    ref = reference(part(x), part(gate), part(state), None if n is None else n.repeat_interleave(group)[few].contiguous(),
                    form, complement, part(dout), part(dfinal), dtype)
    for name, t in got.items():
        check(part(t), ref[name], f"large {N}x{T}x{D} {dtype} {name}")
