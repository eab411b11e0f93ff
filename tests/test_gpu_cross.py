"""The non-causal op between two sequences against its formulas in 64 bits.

Tolerances come from the arithmetic: products and sums in 32 bits, u = 2^-23 (a
whole step: the matrix instructions' own sums are not promised to round to
nearest).  A sum of n terms in any order is off by at most n u times the sum of
its terms' magnitudes; with K the key tokens, Q the query tokens (of all heads
that share a key head), S buckets and d columns that gives, for E = B / (A + eps),
    dE_ = ((K + 1) u sum k|v| + (K + 2) u |B|) / (A + eps),
    out within sum q (dE_ + (S + 3) u |E|),
and the like for the gradients, factor by factor.  Half a step of the output's
type on top.
"""
from __future__ import annotations

import pytest
import torch

from gpu_util import say

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
EPS = 1e-6


def _t(m):
    return m.transpose(1, 2).contiguous()


def reference(q, k, v, lengths=None, dout=None):
    """name -> (value, bound) for q [Nq, Tq, S], k [Nk, Tk, S], v [Nk, Tk, d]."""
    half = HALF[q.dtype]
    Nq, Nk, K, S, d = q.shape[0], k.shape[0], k.shape[1], k.shape[2], v.shape[2]
    n = None if lengths is None else lengths.long().clamp(0, K).repeat_interleave(Nk // len(lengths))
    dead = None if n is None else (torch.arange(K, device=q.device) >= n[:, None])[..., None]
    qd, kd, vd = q.double().reshape(Nk, -1, S), k.double(), v.double()
    if dead is not None:
        kd, vd = kd.masked_fill(dead, 0.0), vd.masked_fill(dead, 0.0)
    Q = qd.shape[1]
    A, B = kd.sum(1)[..., None], _t(kd) @ vd
    den = A + EPS
    E = B / den
    eE = ((K + 1) * U * (_t(kd) @ vd.abs()) + (K + 2) * U * B.abs()) / den
    out = qd @ E
    res = {"out": (out.reshape(Nq, -1, d), (qd @ (eE + (S + 3) * U * E.abs()) + half * out.abs()).reshape(Nq, -1, d)),
           "state": (torch.cat([B.flatten(1), A.flatten(1)], 1),
                     torch.cat([((K + 1) * U * (_t(kd) @ vd.abs())).flatten(1), ((K + 1) * U * A).flatten(1)], 1))}
    if dout is None:
        return res
    g = dout.double().reshape(Nk, -1, d)
    dq = g @ _t(E)
    res["dq"] = (dq.reshape(q.shape), (g.abs() @ _t(eE + (d + 3) * U * E.abs()) + half * dq.abs()).reshape(q.shape))
    dE, edE = _t(qd) @ g, (Q + 1) * U * (_t(qd) @ g.abs())
    dB, edB = dE / den, edE / den + dE.abs() / den * (K + 3) * U
    dA = -(dE * E).sum(-1) / den[..., 0]
    edA = ((edE * E.abs() + dE.abs() * eE).sum(-1) + (d + K + 6) * U * (dE * E).abs().sum(-1)) / den[..., 0]
    dk = vd @ _t(dB) + dA[:, None]
    edk = vd.abs() @ _t(edB) + edA[:, None] + (d + 3) * U * (vd.abs() @ _t(dB.abs()) + dA.abs()[:, None])
    dv = kd @ dB
    edv = kd @ (edB + (S + 3) * U * dB.abs())
    for name, value, err in (("dk", dk, edk), ("dv", dv, edv)):
        err = 2 * err + half * value.abs()  # second-order terms: less than the first again
        if dead is not None:
            value, err = value.masked_fill(dead, 0.0), err.masked_fill(dead, 0.0)
        res[name] = (value, err)
    return res


def check(got, want, label):
    value, bound = want
    assert got.shape == value.shape, (label, got.shape, value.shape)
    err = (got.double() - value).abs()
    worst = float((err / (bound + 1e-300)).max()) if err.numel() else 0.0
    say(label, f"{worst:.3f} of the bound")
    assert bool((err <= bound + 1e-37).all()), (label, worst)


def make(Nq, Nk, Tq, Tk, L, R, d, dtype, seed, device):
    g = torch.Generator(device=device).manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g, device=device)
    p = lambda N, T: torch.softmax(4 * n(N, T, L, R), -1).flatten(2).to(dtype)
    return p(Nq, Tq), p(Nk, Tk), n(Nk, Tk, d).to(dtype), n(Nq, Tq, d).to(dtype)


# (Nq, Nk, Tq, Tk, L, R, d)
CASES = [(3, 3, 1, 1, 4, 16, 64), (4, 2, 5, 70, 4, 16, 64), (2, 2, 16, 33, 4, 16, 64), (2, 2, 17, 300, 4, 16, 64),
         (12, 3, 65, 129, 4, 16, 64), (8, 2, 40, 257, 8, 32, 128), (6, 6, 3, 50, 8, 32, 128), (3, 1, 30, 40, 1, 7, 17),
         (3, 1, 2, 40, 1, 7, 17), (4, 4, 100, 3, 3, 10, 50), (2, 2, 77, 190, 2, 8, 32), (2, 2, 64, 64, 3, 16, 96),
         (1, 1, 50, 40000, 4, 16, 64), (1, 1, 40000, 50, 4, 16, 64), (300, 300, 1, 20, 4, 16, 64),
         (300, 300, 8, 20, 5, 6, 36), (2, 1, 7, 9, 1, 1, 1), (2, 2, 20, 30, 1, 1, 128), (5, 5, 12, 9, 7, 36, 128),
         # Widths that are no multiples of four, over one block and several.
         (4, 2, 90, 300, 8, 16, 17), (4, 4, 70, 200, 5, 7, 100), (2, 1, 200, 333, 3, 13, 121), (3, 3, 50, 70, 85, 3, 127),
         (2, 2, 300, 2100, 8, 8, 66), (2, 2, 40, 40, 7, 31, 3), (6, 2, 33, 50, 1, 2, 1), (2, 2, 33, 50, 2, 3, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Nq, Nk, Tq, Tk, L, R, d", CASES)
def test_forward_and_gradients(race, cuda, Nq, Nk, Tq, Tk, L, R, d, dtype):
    q, k, v, dout = make(Nq, Nk, Tq, Tk, L, R, d, dtype, Tq + 1000 * Tk, cuda)
    ref = reference(q, k, v, None, dout)
    leaves = [q.view(Nq, Tq, L, R).requires_grad_(True), k.view(Nk, Tk, L, R).requires_grad_(True),
              v.requires_grad_(True)]
    out = race.race_cross_fwd(*leaves)
    grads = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    label = f"cross {dtype} {Nq}/{Nk} {Tq}x{Tk} S{L * R} d{d}"
    check(out, ref["out"], label + " out")
    for name, g, leaf in zip(("dq", "dk", "dv"), grads, leaves):
        assert g.shape == leaf.shape and g.dtype == dtype
        check(g.flatten(2), ref[name], f"{label} {name}")
    # Each gradient by itself.
    for i, name in enumerate(("dq", "dk", "dv")):
        (g,) = torch.autograd.grad(race.race_cross_fwd(*[t if j == i else t.detach() for j, t in enumerate(leaves)]),
                                   leaves[i], dout)
        check(g.flatten(2), ref[name], f"{label} {name} alone")
    # Without a gradient, and through the state.
    plain = [t.detach() for t in leaves]
    check(race.race_cross_fwd(*plain), ref["out"], label + " no grad")
    state = race.race_cross_state(plain[1], plain[2])
    check(state, ref["state"], label + " state")
    check(race.race_cross_query(plain[0], state), ref["out"], label + " query")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Tq, Tk, L, R, d, lengths", [(40, 130, 4, 16, 64, [0, 1, 130, 129]), (3, 700, 4, 16, 64, [700, 0]),
                                                      (50, 90, 8, 32, 128, [64, 0]), (20, 50, 3, 10, 50, [13, 50, 0, 1]),
                                                      (30, 3000, 2, 8, 32, [1024, 1]), (70, 301, 5, 7, 33, [301, 77, 0, 1]),
                                                      (33, 200, 16, 8, 121, [150, 7]), (19, 40, 4, 16, 64, [-3, 999])])
def test_padded_keys(race, cuda, Tq, Tk, L, R, d, lengths, dtype):
    Nk = 4
    q, k, v, dout = make(2 * Nk, Nk, Tq, Tk, L, R, d, dtype, Tk, cuda)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    ref = reference(q, k, v, n, dout)
    dead = (torch.arange(Tk, device=cuda) >= n.repeat_interleave(Nk // len(lengths))[:, None])[..., None]
    k = k.masked_fill(dead, float("nan"))
    v = v.masked_fill(dead, float("inf"))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = race.race_cross_fwd(*leaves, n)
    grads = torch.autograd.grad(out, leaves, dout)
    check(out, ref["out"], "padded out")
    for name, g in zip(("dq", "dk", "dv"), grads):
        check(g, ref[name], "padded " + name)
    state = race.race_cross_state(k.detach(), v.detach(), n.long())
    check(state, ref["state"], "padded state")
    check(race.race_cross_query(q.detach(), state), ref["out"], "padded query")
    for i, length in enumerate(n.clamp(0, Tk).repeat_interleave(Nk // len(lengths)).tolist()):
        if length == 0:
            assert (out[2 * i:2 * i + 2] == 0).all() and (state[i] == 0).all()


def test_equal_lengths_give_the_non_causal_op(race, cuda):
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, _ = make(6, 6, 200, 200, 4, 16, 64, dtype, 1, cuda)
        assert torch.equal(race.race_cross_fwd(q, k, v), race.race_fused_fwd(q, k, v, False))
        full = torch.full((2,), 200, dtype=torch.int32, device=cuda)
        assert torch.equal(race.race_cross_fwd(q, k, v, full), race.race_cross_fwd(q, k, v))


def test_shared_heads_equal_repeated_ones(race, cuda):
    q, k, v, dout = make(8, 2, 33, 70, 4, 16, 64, torch.float32, 2, cuda)
    kr, vr = k.repeat_interleave(4, 0), v.repeat_interleave(4, 0)
    ref, rep = reference(q, k, v, None, dout), reference(q, kr, vr, None, dout)
    leaves = [t.requires_grad_(True) for t in (kr, vr)]
    grads = torch.autograd.grad(race.race_cross_fwd(q, *leaves), leaves, dout)
    for name, g in zip(("dk", "dv"), grads):
        value, bound = ref[name]
        total = g.double().view(2, 4, *g.shape[1:]).sum(1)
        assert bool(((total - value).abs() <= rep[name][1].view(2, 4, *g.shape[1:]).sum(1) + bound).all())


def test_gradients_against_differences(race, cuda):
    q, k, v, dout = make(4, 2, 9, 31, 2, 8, 32, torch.float32, 3, cuda)
    n = torch.tensor([31, 20], dtype=torch.int32, device=cuda)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = race.race_cross_fwd(*leaves, n)
    grads = torch.autograd.grad(out, leaves, dout)
    step = 2.0 ** -10
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        way = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(i)).to(cuda)
        if i < 2:  # probabilities stay positive
            way = way * leaf.detach()
        loss = []
        for sign in (1, -1):
            moved = [t.detach() + sign * step * way if j == i else t.detach() for j, t in enumerate(leaves)]
            loss.append(float((race.race_cross_fwd(*moved, n).double() * dout).sum()))
        along = float((grad.double() * way).sum())
        size = float((out.detach().double().abs() * dout.abs()).sum())
        assert abs((loss[0] - loss[1]) / (2 * step) - along) <= 1e-3 * float(
            (grad.double().abs() * way.abs()).sum()) + 40 * U * size / step, i


def test_non_finite_values_stay_in_their_streams(race, cuda):
    q, k, v, dout = make(3, 3, 40, 60, 4, 16, 64, torch.bfloat16, 4, cuda)
    want = race.race_cross_fwd(q, k, v)
    v[1, 7, 5] = float("nan")
    out = race.race_cross_fwd(q, k, v)
    assert torch.isnan(out[1, :, 5]).all() and torch.equal(out[[0, 2]], want[[0, 2]])
    assert torch.equal(out[1, :, :5], want[1, :, :5])


def test_empty_sides_and_refusals(race, cuda):
    q, k, v, dout = make(4, 2, 5, 6, 2, 8, 32, torch.float32, 5, cuda)
    none_q, none_k, none_v = q[:, :0].contiguous(), k[:, :0].contiguous(), v[:, :0].contiguous()
    leaves = [t.requires_grad_(True) for t in (q, none_k, none_v)]
    out = race.race_cross_fwd(*leaves)
    grads = torch.autograd.grad(out, leaves, dout)
    assert (out == 0).all() and (grads[0] == 0).all() and grads[1].shape == none_k.shape
    assert (race.race_cross_state(none_k, none_v) == 0).all()
    leaves = [t.detach().requires_grad_(True) for t in (none_q, k, v)]
    out = race.race_cross_fwd(*leaves)
    grads = torch.autograd.grad(out, leaves, torch.zeros_like(out))
    assert out.shape == (4, 0, 32) and all((g == 0).all() for g in grads)
    # No query streams at all.
    leaves = [t.detach().requires_grad_(True) for t in (q[:0], k, v)]
    out = race.race_cross_fwd(*leaves)
    assert out.shape == (0, 5, 32) and all((g == 0).all() for g in torch.autograd.grad(out, leaves, torch.zeros_like(out)))
    assert race.race_cross_query(leaves[0].detach(), race.race_cross_state(k, v).detach()).shape == (0, 5, 32)
    e = torch.empty(0, 3, 16, device=cuda)
    assert race.race_cross_fwd(e, e, torch.empty(0, 3, 32, device=cuda)).shape == (0, 3, 32)
    q, k, v = (t.detach() for t in (q, k, v))
    n = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)
    state = race.race_cross_state(k, v)
    for args, message in [
        ((q[:3].contiguous(), k, v), "no multiple"), ((q[..., :8].contiguous(), k, v), "another number of buckets"),
        ((q, k, v[:, :5].contiguous()), "V has shape"), ((q, k.bfloat16(), v), "another dtype"),
        ((q.transpose(0, 1), k, v), "strided view"), ((q, k, v, n(1, 2, 3)), "do not divide"),
        ((q, k, v, n(1, 2).float()), "int32"), ((q, k, v, n(1, 2).cpu()), "rows' device"), ((q[0], k, v), "has shape"),
        ((q, k, torch.zeros(2, 6, 129, device=cuda)), "no kernel"),
        ((torch.zeros(2, 5, 257, device=cuda), torch.zeros(2, 6, 257, device=cuda), v), "no kernel"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            race.race_cross_fwd(*args)
    for args, message in [((q, state[:, :-1].contiguous()), "state has shape"), ((q, state.double()), "float32"),
                          ((q[:3].contiguous(), state), "no multiple"), ((q.half(), state), "neither")]:
        with pytest.raises(RuntimeError, match=message):
            race.race_cross_query(*args)


def test_other_stream_and_captured_steps(race, cuda):
    q, k, v, dout = make(8, 4, 50, 300, 4, 16, 64, torch.bfloat16, 6, cuda)
    n = torch.tensor([300, 7], dtype=torch.int32, device=cuda)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    token = q.detach()[:, :1].clone()

    def step():
        out = race.race_cross_fwd(*leaves, n)
        state = race.race_cross_state(leaves[1].detach(), leaves[2].detach(), n)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout), state, race.race_cross_query(token, state))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        new = make(8, 4, 50, 300, 4, 16, 64, torch.bfloat16, 20 + i, cuda)
        with torch.no_grad():
            for leaf, t in zip(leaves, new):
                leaf.copy_(t)
        token.copy_(new[0][:, :1])
        n.copy_(torch.tensor([100 * i, 300 - i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), i
    held = race.race_cross_fwd(*leaves, n)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            dout.mul(2)
            race.race_cross_fwd(*leaves, n)
    del held


@pytest.mark.parametrize("S, d, Tq", [(64, 64, 200), (64, 64, 9), (256, 128, 70), (30, 50, 40)])
def test_c_entry_with_used_memory(race, cuda, S, d, Tq):
    from race_attention_kernel_amd import abi

    N, Tk = 2, 5000
    q, k, v, g = make(N, N, Tq, Tk, 1, S, d, torch.float32, 7, cuda)
    n = torch.tensor([5000, 2100], dtype=torch.int32, device=cuda)
    sh = abi.cross_shape(N, Tq, Tk, 1, S, d)
    nan = lambda *s: torch.full(s, float("nan"), device=cuda)
    (_, fwd), (_, bwd) = abi.cross_workspace_bytes(sh), abi.cross_workspace_bytes(sh, True)
    ws, state = nan(max(fwd, bwd) // 4), nan(N, S * d + S)
    out, dq, dk, dv = nan(N, Tq, d), nan(N, Tq, S), nan(N, Tk, S), nan(N, Tk, d)
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()
    assert abi.cross_fwd(p(q), p(k), p(v), p(n), p(out), p(state), sh, p(ws), fwd, stream) == 0
    ws.fill_(float("nan"))
    assert abi.cross_bwd(p(q), p(k), p(v), p(n), p(g), p(state), p(dq), p(dk), p(dv), sh, p(ws), bwd, stream) == 0
    again = nan(N, Tq, d)
    assert abi.cross_query(p(q), p(state), p(again), sh, stream) == 0
    torch.cuda.synchronize()
    ref = reference(q, k, v, n, g)
    for name, got in (("out", out), ("state", state), ("dq", dq), ("dk", dk), ("dv", dv), ("out", again)):
        check(got, ref[name], f"c entry {name}")
    assert abi.cross_fwd(p(q), p(k), p(v), p(n), p(out), p(state), sh, p(ws), fwd - 4, stream) == 1


def test_offsets_past_32_bits(race, cuda):
    # 4.4 GB of key probabilities: the last stream against itself alone.
    N, Tk, S, d = 17, 65536, 256, 16
    gen = torch.Generator(device=cuda).manual_seed(1)
    k = torch.rand(N, Tk, S, generator=gen, device=cuda)
    v, q = torch.randn(N, Tk, d, generator=gen, device=cuda), torch.rand(N, 40, S, generator=gen, device=cuda)
    g = torch.randn(N, 40, d, generator=gen, device=cuda)
    k.requires_grad_(True)
    out = race.race_cross_fwd(q, k, v)
    (dk,) = torch.autograd.grad(out, k, g)
    last = [t.detach()[-1:].clone() for t in (q, k, v, g)]
    ref = reference(last[0], last[1], last[2], None, last[3])
    check(out[-1:], ref["out"], "last stream out")
    check(dk[-1:], ref["dk"], "last stream dk")


def test_zeros_past_32_bits(race, cuda):
    # No keys: 33 x 2^20 rows of 128 zeros, more than 2^32 values.
    N, Tq, d = 33, 1 << 20, 128
    used = torch.ones(N, Tq, d, dtype=torch.bfloat16, device=cuda)
    del used
    q = torch.ones(N, Tq, 2, dtype=torch.bfloat16, device=cuda)
    out = race.race_cross_fwd(q, q[:, :0].contiguous(), torch.empty(N, 0, d, dtype=torch.bfloat16, device=cuda))
    assert out.shape == (N, Tq, d) and not any(bool(rows.any()) for rows in out)


def test_lengths_of_64_bits(race, cuda):
    q, k, v, _ = make(3, 3, 20, 50, 2, 8, 32, torch.float32, 8, cuda)
    far = torch.tensor([2 ** 40, 2 ** 31 + 5, -2 ** 40], device=cuda)
    near = torch.tensor([50, 50, 0], dtype=torch.int32, device=cuda)
    assert torch.equal(race.race_cross_fwd(q, k, v, far), race.race_cross_fwd(q, k, v, near))
    pairs = torch.stack([near, near], 1).long()
    assert torch.equal(race.race_cross_fwd(q, k, v, pairs[:, 0]), race.race_cross_fwd(q, k, v, near))


@pytest.mark.parametrize("options", [dict(), dict(qk_norm=True, rope_pairs=32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_module_decoder_step_by_step(race, cuda, dtype, options):
    # An encoder's sums kept, a decoder's tokens one by one: forward's rows.
    torch.manual_seed(1)
    M, B, Tq, Tk, H, Hk, d = 1, 2, 6, 90, 4, 2, 64
    module = race.CrossACE(d, 4, 4, M, device=cuda, **options)
    K, V = (torch.randn(M, B, Tk, Hk, d, device=cuda).to(dtype) for _ in range(2))
    Q = torch.randn(M, B, Tq, H, d, device=cuda).to(dtype)
    n = torch.tensor([90, 41], dtype=torch.int32, device=cuda)
    leaves = [t.requires_grad_(True) for t in (K, V, Q)]
    out = module(*leaves, n)
    assert out.shape == Q.shape and out.dtype == dtype
    up = torch.randn_like(out)
    grads = torch.autograd.grad(out, leaves + list(module.parameters()), up)
    assert all(torch.isfinite(g).all() and (g != 0).any() for g in grads)
    assert (grads[0][0, 1, 41:] == 0).all() and (grads[1][0, 1, 41:] == 0).all()
    state = module.encode(K, V, n)
    steps = [module.query(Q[:, :, t:t + 1], state, torch.tensor([t], device=cuda)) for t in range(Tq)]
    # The same probabilities and state; only the order of the sums over buckets differs.
    got, want = torch.cat(steps, 2).double(), out.detach().double()
    size = want.abs().amax(dim=-1, keepdim=True)
    assert bool(((got - want).abs() <= (64 * 4 * U + 2 * HALF[dtype]) * size + 1e-30).all())


# Sizes where the bf16 maps' matrices stay in registers: many streams, many tokens, key
# lengths of one record and of several (csrc/noncausal_mfma.hip, map_in_registers).
LARGE = [(256, 256, 40, 70, 8, 32, 128, None), (512, 512, 20, 30, 8, 16, 128, [30, 0, 7, 17]), (1, 1, 66000, 40, 8, 32, 128, None),
         (2, 1, 50000, 3000, 8, 32, 72, [2999]), (260, 260, 33, 300, 8, 32, 128, [300, 64])]


@pytest.mark.parametrize("Nq, Nk, Tq, Tk, L, R, d, lengths", LARGE)
def test_large_calls(race, cuda, Nq, Nk, Tq, Tk, L, R, d, lengths):
    q, k, v, dout = make(Nq, Nk, Tq, Tk, L, R, d, torch.bfloat16, Tq + Tk, cuda)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda) if lengths else None
    ref = reference(q, k, v, n, dout)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = race.race_cross_fwd(*leaves, n)
    grads = torch.autograd.grad(out, leaves, dout)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        check(got.detach(), ref[name], f"large {Nq}/{Nk} {Tq}x{Tk} S{L * R} d{d} {name}")


@pytest.mark.parametrize("N, L, R, d", [(256, 8, 32, 128), (512, 8, 16, 128), (460, 8, 32, 72), (400, 9, 8, 128)])
def test_streams_do_not_depend_on_their_number(race, cuda, N, L, R, d):
    # Few streams and many take different kernels; a stream's bits are the same, tokens with infinities and NaN too.
    q, k, v, dout = make(N, N, 40, 50, L, R, d, torch.bfloat16, 9, cuda)
    q[1, 3, 5], v[2, 7, 11], dout[3, 17, 2] = float("inf"), float("nan"), float("-inf")
    state = race.race_cross_state(k, v)

    def run(few):
        leaves = [t[:few].clone().requires_grad_(True) for t in (q, k, v)]
        out = race.race_cross_fwd(*leaves)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout[:few].contiguous()),
                race.race_cross_query(q[:few].contiguous(), state[:few].contiguous()))

    for a, b in zip(run(N), run(6)):
        a = a[:6]
        assert bool(((a == b) | (a.isnan() & b.isnan())).all())
