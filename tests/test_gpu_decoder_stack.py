"""The operators as a decoder layer uses them: queries and keys normed and
rotated, the causal op, the gated recurrence over its output, and cross
attention to a padded batch of encoder sequences; whole, and token by token from
the three carried states."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from gpu_util import FP32_TOL, per_stream_rel_err, say

pytestmark = pytest.mark.gpu

B, H, d, T, Te, L, K = 3, 4, 64, 37, 90, 4, 4
D = H * d


class Layer(torch.nn.Module):
    def __init__(self, race, device):
        super().__init__()
        self.race = race
        g = torch.Generator(device=device).manual_seed(0)
        n = lambda *s: torch.nn.Parameter(torch.randn(s, generator=g, device=device) / s[-1] ** 0.5)
        self.qkv, self.gates, self.cross_q, self.cross_kv = n(3 * D, D), n(D, D), n(D, D), n(2 * D, D)
        self.q_norm, self.k_norm = (torch.nn.Parameter(torch.ones(d, device=device)) for _ in range(2))
        self.planes = torch.randn(d, L * K, generator=g, device=device)
        self.cross = race.CrossACE(d, K, L, 1, device=device, qk_norm=True)
        self.freq = (10000.0 ** (-torch.arange(16, device=device) / 16)).float()

    def heads(self, streams, t):
        return streams.view(B, H, t, d).transpose(1, 2).reshape(B, t, D)

    def rows(self, x, first):
        """Bucket probabilities of queries and keys, and values, of tokens first .. as streams."""
        t, race = x.shape[1], self.race
        y = (x @ self.qkv.t()).view(B, t, 3 * H, d)
        pos = torch.arange(first, first + t, device=x.device)
        q, k = race.race_norm_rope(y[:, :, :H], y[:, :, H:2 * H], pos, self.freq, q_weight=self.q_norm,
                                   k_weight=self.k_norm)
        v, _ = race.race_norm_rope(y[:, :, 2 * H:], None, eps=None)
        return race.race_hash_probs(q, self.planes, L, K), race.race_hash_probs(k, self.planes, L, K), v

    def forward(self, x, encoder, lengths):
        race, t = self.race, x.shape[1]
        q, k, v = self.rows(x, 0)
        y = self.heads(race.race_fused_fwd(q, k, v, causal=True), t)
        y, _ = race.race_gated_scan(y, x @ self.gates.t() + 2.0)
        ek, ev = (encoder @ self.cross_kv.t()).view(1, B, Te, 2, H, d).unbind(3)
        eq = (y @ self.cross_q.t()).view(1, B, t, H, d)
        return y + self.cross(ek, ev, eq, lengths).reshape(B, t, D)

    @torch.no_grad()
    def encode(self, encoder, lengths):
        ek, ev = (encoder @ self.cross_kv.t()).view(1, B, Te, 2, H, d).unbind(3)
        return self.cross.encode(ek, ev, lengths)

    @torch.no_grad()
    def step(self, x, first, states):
        """A call's tokens from (op state, scan state, encoder state); the first two advance in place."""
        race, t = self.race, x.shape[1]
        op_state, scan_state, encoder_state = states
        q, k, v = self.rows(x, first)
        y, _ = race.race_fused_fwd_carry(q, k, v, op_state, inplace=True)
        y, _ = race.race_gated_scan_carry(self.heads(y, t), x @ self.gates.t() + 2.0, scan_state, inplace=True)
        eq = (y @ self.cross_q.t()).view(1, B, t, H, d)
        return y + self.cross.query(eq, encoder_state).reshape(B, t, D)


def _inputs(device):
    g = torch.Generator(device=device).manual_seed(1)
    x = torch.randn(B, T, D, generator=g, device=device)
    encoder = torch.randn(B, Te, D, generator=g, device=device)
    lengths = torch.tensor([Te, 0, 33], dtype=torch.int32, device=device)
    return x, encoder, lengths


def test_prompt_and_single_tokens_equal_the_whole(race, cuda):
    layer = Layer(race, cuda)
    x, encoder, lengths = _inputs(cuda)
    whole = layer(x, encoder, lengths).detach()
    S = L * 2 ** K
    for prompt in (0, 20):
        states = (torch.zeros(B * H, S * d + S, device=cuda), torch.zeros(B, D, device=cuda),
                  layer.encode(encoder, lengths))
        outs, at = [], 0
        for size in ([prompt] if prompt else []) + [1] * (T - prompt):
            outs.append(layer.step(x[:, at:at + size], at, states))
            at += size
        got = torch.cat(outs, 1)
        # Both ways keep the causal op's tolerance (twice), and the layers behind it pass it on.
        err = per_stream_rel_err(got.cpu().numpy(), whole.cpu().numpy())
        say("prompt", prompt, f"rel err {err:.2e}")
        assert err <= 4 * FP32_TOL, prompt


def test_gradients_reach_every_parameter(race, cuda):
    layer = Layer(race, cuda)
    x, encoder, lengths = _inputs(cuda)
    leaves = [x.requires_grad_(True), encoder.requires_grad_(True), *layer.parameters()]
    up = torch.randn(B, T, D, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda)
    grads = torch.autograd.grad(layer(x, encoder, lengths), leaves, up)
    assert all(torch.isfinite(g).all() and (g != 0).any() for g in grads)
    assert (grads[1][1] == 0).all() and (grads[1][2, 33:] == 0).all()  # no keys there
    # Along a direction in every leaf at once, against differences in the layer itself.
    way = [torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).to(cuda) for i, t in enumerate(leaves)]
    along = sum(float((g.double() * w).sum()) for g, w in zip(grads, way))
    step, loss = 2.0 ** -10, []
    for sign in (1, -1):
        with torch.no_grad():
            for t, w in zip(leaves, way):
                t.add_(w, alpha=sign * step)
            loss.append(float((layer(x, encoder, lengths).double() * up).sum()))
            for t, w in zip(leaves, way):
                t.add_(w, alpha=-sign * step)
    size = sum(float((g.double().abs() * w.abs()).sum()) for g, w in zip(grads, way))
    assert abs((loss[0] - loss[1]) / (2 * step) - along) <= 5e-3 * size + FP32_TOL * np.sqrt(B * T * D) / step


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", ["norm_rope q", "norm_rope weight", "scan gate", "scan state", "cross V"])
def test_forward_mode_derivatives_are_refused(race, cuda, which, grad):
    # None of the operators has one: an output without a tangent would count as a zero derivative.
    n = lambda *s: torch.randn(*s, device=cuda)
    q, k, w, x, gate, state, probs, v = (n(2, 5, 3, 64), n(2, 5, 1, 64), n(64), n(2, 5, 64), n(2, 5, 64), n(2, 64),
                                         torch.rand(2, 5, 16, device=cuda), n(2, 5, 64))
    plain = {"norm_rope q": (q, lambda t: race.race_norm_rope(t, k)),
             "norm_rope weight": (w, lambda t: race.race_norm_rope(q, k, q_weight=w, k_weight=t)),
             "scan gate": (gate, lambda t: race.race_gated_scan(x, t)),
             "scan state": (state, lambda t: race.race_gated_scan(x, gate, t)),
             "cross V": (v, lambda t: race.race_cross_fwd(probs, probs, t))}
    at, run = plain[which]
    with torch.set_grad_enabled(grad), torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="jvp"):
            run(torch.autograd.forward_ad.make_dual(at, torch.ones_like(at)))
        run(at)
