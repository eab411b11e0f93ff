"""The gated delta rule's layer as a model runs it: the residual's norm, projections,
race_norm_rope of queries and keys, race_delta_rule with shared key heads,
race_gate_norm, and the residual again; whole, as a prompt and single tokens from the
carried state, padded, on another stream and replayed from a captured graph."""
from __future__ import annotations

import pytest
import torch

from gpu_util import say

pytestmark = pytest.mark.gpu

B, H, Hk, d, dv, D, T = 3, 4, 2, 64, 48, 256, 70
EPS = 2.0 ** -24


class Layer(torch.nn.Module):
    def __init__(self, race, device, dtype=torch.float32):
        super().__init__()
        self.race = race
        g = torch.Generator(device=device).manual_seed(0)
        n = lambda *s: torch.nn.Parameter((torch.randn(s, generator=g, device=device) / s[-1] ** 0.5).to(dtype))
        one = lambda m: torch.nn.Parameter((1 + 0.1 * torch.randn(m, generator=g, device=device)).to(dtype))
        self.qk, self.v, self.z, self.small, self.out = n(2 * Hk * d, D), n(H * dv, D), n(H * dv, D), n(2 * H, D), n(D, H * dv)
        self.norm, self.head_norm = one(D), one(dv)
        # Rows of length 1: their root mean square times d^-1/2.
        self.unit = torch.full((d,), 0.99 * d ** -0.5, device=device, dtype=dtype)
        self.freq = (10000.0 ** (-torch.arange(d // 4, device=device) / (d // 4))).float()

    def rows(self, x, first):
        t = x.shape[1]
        qk = (x @ self.qk.t()).view(B, t, 2 * Hk, d)
        pos = torch.arange(first, first + t, device=x.device)
        q, k = self.race.race_norm_rope(qk[:, :, :Hk], qk[:, :, Hk:], pos, self.freq, q_weight=self.unit, k_weight=self.unit)
        v = (x @ self.v.t()).view(B, t, H, dv).transpose(1, 2).reshape(B * H, t, dv)
        gate, beta = (x @ self.small.t()).view(B, t, 2, H).permute(2, 0, 3, 1).reshape(2, B * H, t).unbind(0)
        return q, k, v, gate + 2.0, torch.sigmoid(beta), (x @ self.z.t()).view(B, t, H, dv)

    def forward(self, x, residual, state=None, lengths=None):
        race = self.race
        x, residual = race.race_add_norm(x, residual, self.norm)
        q, k, v, gate, beta, z = self.rows(x, 0)
        o, state = race.race_delta_rule(q, k, v, gate, beta, state, gate_form="sigmoid", scale=d ** -0.5, lengths=lengths)
        return race.race_gate_norm(o, z, self.head_norm).flatten(2) @ self.out.t(), residual, state

    @torch.no_grad()
    def step(self, x, residual, first, state):
        """A call's tokens; the state advances in place."""
        race = self.race
        x, residual = race.race_add_norm(x, residual, self.norm)
        q, k, v, gate, beta, z = self.rows(x, first)
        o, _ = race.race_delta_rule_carry(q, k, v, gate, beta, state, gate_form="sigmoid", scale=d ** -0.5, inplace=True)
        return race.race_gate_norm(o, z, self.head_norm).flatten(2) @ self.out.t(), residual


def _inputs(device, dtype=torch.float32):
    g = torch.Generator(device=device).manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g, device=device)
    return n(B, T, D).to(dtype), (2 * n(B, T, D)).to(dtype), n(B * H, d, dv) / 8, n(B, T, D).to(dtype)


# Two ways of fp32 sums of up to 256 terms, 2^-24 each, through six operators; the gated norm
# divides by a root mean square that is a part of its terms.
TOL = 6 * 256 * EPS


def test_prompt_and_single_tokens_equal_the_whole(race, cuda):
    layer = Layer(race, cuda)
    x, residual, state, _ = _inputs(cuda)
    with torch.no_grad():
        whole, total, final = layer(x, residual, state)
    for prompt in (0, 20, 69):
        carried, outs, at = state.clone(), [], 0
        for size in ([prompt] if prompt else []) + [1] * (T - prompt):
            y, r = layer.step(x[:, at:at + size], residual[:, at:at + size], at, carried)
            assert torch.equal(r, total[:, at:at + size])
            outs.append(y)
            at += size
        err = (torch.cat(outs, 1) - whole).norm() / whole.norm(), (carried - final).norm() / final.norm()
        say("prompt", prompt, f"rel err {float(err[0]):.2e} {float(err[1]):.2e}")
        assert max(err) <= TOL, prompt


def test_a_padded_batch_equals_its_sequences(race, cuda):
    layer = Layer(race, cuda)
    x, residual, state, _ = _inputs(cuda)
    lengths = torch.tensor([T, 0, 33], dtype=torch.int32, device=cuda)
    with torch.no_grad():
        y, _, final = layer(x, residual, state, lengths)
        whole, _, _ = layer(x, residual, state)
        short, _, ends = layer(x[:, :33], residual[:, :33], state)
    norm = whole.norm() / whole.numel() ** 0.5
    assert (y[0] - whole[0]).norm() <= TOL * norm * y[0].numel() ** 0.5
    assert (y[2, :33] - short[2]).norm() <= TOL * norm * short[2].numel() ** 0.5
    assert torch.isfinite(y).all() and (y[2, 33:] == 0).all() and (y[1] == 0).all()  # normed rows of zeros
    assert torch.equal(final[H:2 * H], state[H:2 * H]) and (final[2 * H:] - ends[2 * H:]).norm() <= TOL * ends[2 * H:].norm()


def test_gradients_reach_every_parameter(race, cuda):
    layer = Layer(race, cuda)
    x, residual, state, up = _inputs(cuda)
    leaves = [x.requires_grad_(True), residual.requires_grad_(True), state.requires_grad_(True), *layer.parameters()]
    down = torch.ones_like(state)

    def loss():
        y, r, s = layer(x, residual, state)
        return (y.double() * up).sum() + (r.double() * up).sum() + (s.double() * down).sum()

    grads = torch.autograd.grad(loss(), leaves)
    assert all(torch.isfinite(g).all() and (g != 0).any() for g in grads)
    # Along a direction in every leaf at once, against differences in the layer itself: the third-order term, and the
    # rounding of what is summed over the step.
    way = [torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).to(cuda) for i, t in enumerate(leaves)]
    way = [w * (1.0 if i < 3 else 0.1) for i, w in enumerate(way)]
    along = sum(float((g.double() * w).sum()) for g, w in zip(grads, way))
    step, sides = 2.0 ** -10, []
    for sign in (1, -1):
        with torch.no_grad():
            for t, w in zip(leaves, way):
                t.add_(w, alpha=sign * step)
            sides.append(float(loss()))
            for t, w in zip(leaves, way):
                t.add_(w, alpha=-sign * step)
    size = sum(float((g.double().abs() * w.abs()).sum()) for g, w in zip(grads, way))
    assert abs((sides[0] - sides[1]) / (2 * step) - along) <= 5e-3 * size + TOL * (B * T * D) ** 0.5 / step


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_training_and_decode_steps(race, cuda, dtype):
    layer = Layer(race, cuda, dtype)
    x, residual, state, up = (t.clone() for t in _inputs(cuda, dtype))
    leaves = [x.requires_grad_(True), residual.requires_grad_(True), state.requires_grad_(True), *layer.parameters()]
    token, rest, carried = x.detach()[:, :1].clone(), residual.detach()[:, :1].clone(), state.detach().clone()
    down = torch.ones_like(state)

    def train():
        y, r, s = layer(x, residual, state)
        return (y.detach(), r.detach(), s.detach(), *torch.autograd.grad((y, r, s), leaves, (up, up, down)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(), layer.step(token, rest, 5, carried)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = train()
        decoded = layer.step(token, rest, 5, carried)
    for i in range(3):
        g = torch.Generator(device=cuda).manual_seed(30 + i)
        with torch.no_grad():
            for t in (x, residual, state, token, rest):
                t.copy_(torch.randn(t.shape, generator=g, device=cuda))
        before = carried.clone()
        graph.replay()
        torch.cuda.synchronize()
        eager, single = train(), layer.step(token, rest, 5, before)
        torch.cuda.synchronize()
        for a, b in zip((*outs[:3], *decoded, carried), (*eager[:3], *single, before)):
            assert torch.equal(a, b), i
        for a, b in zip(outs[3:], eager[3:]):
            # The projections' gradients are the library's, which may sum in another order here.
            half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
            assert (a.double() - b.double()).norm() <= 2 * half * b.double().norm() * (1 if dtype != torch.float32 else 256), i


def test_norms_on_other_streams_and_captured(race, cuda):
    n = lambda *s: torch.randn(*s, device=cuda)
    for rows, width in ((5, 96), (3000, 512)):
        x, res, w = (t.requires_grad_(True) for t in (n(rows, width), n(rows, width), n(width)))
        h, z, hw = (t.requires_grad_(True) for t in (n(6, rows, 32), n(2, rows, 3, 32), n(32)))
        ups = [n(rows, width), n(rows, width), n(2, rows, 3, 32)]

        def step():
            y, s = race.race_add_norm(x, res, w)
            y8, scales, _ = race.race_add_norm_e4m3(x.detach(), res.detach(), w.detach(), group=32)
            g = race.race_gate_norm(h, z, hw)
            grads = torch.autograd.grad((y, s, g), (x, res, w, h, z, hw), ups)
            return (y.detach(), s.detach(), y8.view(torch.uint8), scales, g.detach(), *grads)

        want = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del got, want
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for i in range(3):
            with torch.no_grad():
                for t in (x, res, w, h, z, hw):
                    t.copy_(torch.randn_like(t))
            graph.replay()
            torch.cuda.synchronize()
            eager = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, eager)), (rows, i)


@pytest.mark.parametrize("which", ["add_norm", "gate_norm"])
def test_a_live_eager_graph_refuses_the_capture(race, cuda, which):
    x = torch.randn(6, 40, 32, device=cuda, requires_grad=True)
    z = torch.randn(2, 40, 3, 32, device=cuda)
    run = (lambda: race.race_add_norm(x)[0]) if which == "add_norm" else (lambda: race.race_gate_norm(x, z))
    eager = run()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            z.mul(2)  # something to record
            run()
    del eager
