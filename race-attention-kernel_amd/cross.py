"""The non-causal op between two sequences: the queries of a decoder over the
keys and values of an encoder, of another length.

    out[t] = sum_s probsQ[t, s] * B[s, :] / (A[s] + 1e-6)

with A and B the sums of the encoder's probsK and probsK (x) V, of which each
batch entry has its own number of tokens.  Those sums are all the queries need:
race_cross_state keeps them, [S*d + S] floats a stream however long the encoder's
sequence was, and race_cross_query answers each new token from them.  The
reference's non-causal op (analysis/hot-path.md:157-162) has one length.
"""
from __future__ import annotations

import torch

from . import _lib
from .batched_ace import BatchedACE
from .rope import race_norm_rope


def race_cross_fwd(probsQ: torch.Tensor, probsK: torch.Tensor, V: torch.Tensor,
                   lengths: torch.Tensor | None = None) -> torch.Tensor:
    """The non-causal op of probsQ's tokens over another sequence's keys.

    Args:
        probsQ: [Nq, Tq, L, R] (or [Nq, Tq, S]) bucket probabilities, float32 or
            bfloat16, contiguous.
        probsK: [Nk, Tk, L, R] (or [Nk, Tk, S]), V: [Nk, Tk, d], same dtype and
            device.  Nq = g Nk: query streams g n .. g n + g - 1 share key
            stream n (query heads that share a key head).
        lengths: int32 (or int64) [Nk] or [Nk / h] (entry i for key streams h i .. h i + h -
            1: one per batch entry): keys from lengths on are not read and get
            zero gradients.  A stream without keys gives zeros.

    Returns [Nq, Tq, d] in V's dtype.  Differentiable once, w.r.t. probsQ, probsK
    and V.  A backward is captured into a graph together with its forward, and not
    while an eager graph of the same leaves is alive."""
    return _lib.ext().cross(probsQ, probsK, V, lengths)


def race_cross_state(probsK: torch.Tensor, V: torch.Tensor, lengths: torch.Tensor | None = None) -> torch.Tensor:
    """The sums [Nk, S*d + S] (float32, B then A) that race_cross_query reads; no
    autograd."""
    return _lib.ext().cross_state(probsK, V, lengths)


def race_cross_query(probsQ: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
    """race_cross_fwd against a kept state: [Nq, Tq, d] in probsQ's dtype; no
    autograd.  At most 16 tokens per key stream run one small launch."""
    return _lib.ext().cross_query(probsQ, state)


class CrossACE(BatchedACE):
    """BatchedACE over another sequence's keys: Khf, Vhf [M, B, Tk, Hk, d_k], Qhf
    [M, B, Tq, H, d_k], H a multiple of Hk.  Constructor as BatchedACE's (never
    causal); with rope_pairs the two sides take positions of their own."""

    def __init__(self, d_k, K, L, M, device="cpu", share_planes=True, **options):
        super().__init__(d_k, K, L, M, device=device, share_planes=share_planes, causal=False, **options)

    def _side(self, x, weight, positions):
        """Rows [M, B, T, H, d_k] as bucket probabilities of streams."""
        rows = x.flatten(0, 1)
        freq = self.inv_freq(rows.device)
        if freq is not None and positions is None:
            positions = torch.arange(rows.shape[1], device=rows.device)
        streams, _ = race_norm_rope(rows, None, positions, freq, q_weight=weight, eps=self.norm_eps,
                                    sections=self.rope_sections, interleaved=self.rope_interleaved)
        return self.bucket_probs(streams)

    def _values(self, Vhf):
        return race_norm_rope(Vhf.flatten(0, 1), None, eps=None)[0]

    def _heads(self, out, Qhf):
        M, B, T, H, dk = Qhf.shape
        return out.view(M, B, H, T, dk).permute(0, 1, 3, 2, 4)

    def forward(self, Khf, Vhf, Qhf, lengths=None, k_positions=None, q_positions=None):
        """lengths: int32 [M * B], the live keys of every batch entry.
        k_positions, q_positions (read with rope_pairs only): as BatchedACE's."""
        probsK = self._side(Khf, self.k_norm, k_positions)
        probsQ = self._side(Qhf, self.q_norm, q_positions)
        return self._heads(race_cross_fwd(probsQ, probsK, self._values(Vhf), lengths), Qhf)

    @torch.no_grad()
    def encode(self, Khf, Vhf, lengths=None, k_positions=None):
        """The encoder's sums [M * B * Hk, S * d_k + S], for query()."""
        return race_cross_state(self._side(Khf, self.k_norm, k_positions), self._values(Vhf), lengths)

    @torch.no_grad()
    def query(self, Qhf, state, q_positions=None):
        """forward's output for Qhf against encode()'s sums: a decode step.  With
        rope_pairs the tokens' q_positions are needed."""
        if self.rope_pairs > 0 and q_positions is None:
            raise ValueError("CrossACE.query: q_positions are needed where rows are rotated (a step's tokens do not "
                             "start at position 0)")
        return self._heads(race_cross_query(self._side(Qhf, self.q_norm, q_positions), state), Qhf)
