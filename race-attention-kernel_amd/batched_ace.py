"""Drop-in BatchedACE (src/race_baseline.py:21-52) running the op on MI355X.

Same constructor and forward signature as the reference module.  The whole
forward is one op, ModuleRaceFunction: the permutes of lines 35-40 are one
copy kernel for the three inputs, and the output has the strides of the permute
of line 52.
For the causal module the hashing of lines 41-44 (shared hash planes, tanh,
corner softmax) and the hot span of lines 45-51 run in the same kernels, which
hash the Q and K rows themselves (the reference's fused forward,
src/race_fused_fwd.cu:80-146), so the bucket probabilities never reach memory.
The non-causal module runs the hashing kernels and the non-causal op.  A
causal module whose L, K, d_k the hashed kernels do not take, and a module
whose bucket_probs is not the one below, go through the separate ops.  Gradients reach
Khf, Qhf and Vhf on every path, as through the reference's torch composition;
planes_T is a buffer there and here.

With qk_norm or rope_pairs the rows the hashing reads are normed and rotated on
their way to the streams (race_norm_rope), which the reference's module has not.
"""
from __future__ import annotations

import itertools

import torch
from torch import nn

from .ops import (ModuleRaceFunction, hashed_supported, race_fused_fwd, race_fused_fwd_hashed,
                  race_hash_probs)
from .rope import race_norm_rope


class BatchedACE(nn.Module):
    """The reference's module; further keywords:

    qk_norm: norm every query and key row by its root mean square, with a learned
        weight per column (q_norm, k_norm).
    rope_pairs: pairs of values of each query and key row that are turned by the
        token's position (2 * rope_pairs <= d_k), at the frequencies
        rope_theta^(-p / rope_pairs); rope_sections: pairs per position axis;
        rope_interleaved: see race_norm_rope.
    """

    def __init__(self, d_k, K, L, M, device="cpu", share_planes=True, causal=True, *, qk_norm=False, norm_eps=1e-6,
                 rope_pairs=0, rope_sections=None, rope_theta=10000.0, rope_interleaved=False):
        super().__init__()
        assert share_planes, "reference config uses shared planes"
        self.d_k, self.K, self.L, self.M = d_k, K, L, M
        self.R = 1 << K
        self.causal = causal
        planes = torch.randn(L, K, d_k, device=device)
        self.register_buffer("planes_T", planes.view(L * K, d_k).T)  # [d_k, L*K]
        corners = torch.tensor(list(itertools.product([-1.0, 1.0], repeat=K)), device=device)
        self.register_buffer("protos_T", corners.T)  # [K, R]
        assert 0 <= 2 * rope_pairs <= d_k, "the rotated pairs are within a row"
        self.norm_eps = norm_eps if qk_norm else None
        self.q_norm = nn.Parameter(torch.ones(d_k, device=device)) if qk_norm else None
        self.k_norm = nn.Parameter(torch.ones(d_k, device=device)) if qk_norm else None
        self.rope_pairs, self.rope_theta = rope_pairs, rope_theta
        self.rope_sections, self.rope_interleaved = rope_sections, rope_interleaved
        self._inv_freq = {}  # by device; float32 whatever the module is cast to, so no buffer

    def __setstate__(self, state):
        super().__setstate__(state)
        self._inv_freq = {}  # a pickle's may come back on another device
        if "rope_pairs" not in self.__dict__:  # pickled before there were these keywords
            self.norm_eps = self.q_norm = self.k_norm = self.rope_sections = None
            self.rope_pairs, self.rope_theta, self.rope_interleaved = 0, 10000.0, False

    def inv_freq(self, device) -> torch.Tensor | None:
        """The rotation's frequencies [rope_pairs], float32."""
        if self.rope_pairs == 0:
            return None
        kept = self._inv_freq.get(device)
        if kept is not None:
            return kept
        with torch.inference_mode(False):  # kept for training calls too, whose node saves them
            p = torch.arange(self.rope_pairs, dtype=torch.float64, device=device)
            freq = (self.rope_theta ** (-p / self.rope_pairs)).float()
        if freq.is_cuda:
            if torch.cuda.is_current_stream_capturing():
                return freq  # the graph's own: it holds values during its replays only
            torch.cuda.current_stream(freq.device).synchronize()  # once a device: later calls read it on any stream
        self._inv_freq[device] = freq
        return freq

    def _streams(self, Khf, Vhf, Qhf, positions):
        """K, Q (normed, rotated) and V rows as streams [M * B * H, T, d_k]."""
        k, v, q = (x.flatten(0, 1) for x in (Khf, Vhf, Qhf))
        freq = self.inv_freq(q.device)
        if freq is not None and positions is None:
            positions = torch.arange(q.shape[1], device=q.device)
        q2, k2 = race_norm_rope(q, k, positions, freq, q_weight=self.q_norm, k_weight=self.k_norm, eps=self.norm_eps,
                                sections=self.rope_sections, interleaved=self.rope_interleaved)
        v2, _ = race_norm_rope(v, None, eps=None)  # to streams as it is
        return k2, q2, v2

    def bucket_probs(self, x2: torch.Tensor) -> torch.Tensor:
        """[N, T, d] -> [N, T, L, R] corner probabilities (reference lines 41-44)."""
        return race_hash_probs(x2, self.planes_T.float(), self.L, self.K)

    def forward(self, Khf, Vhf, Qhf, positions=None):
        """positions (read with rope_pairs only): [T] or [M * B, T], or [axes,
        M * B, T] with rope_sections; None: 0 .. T-1."""
        M, B, T, H, dk = Khf.shape
        N = M * B * H
        hashed = self.causal and hashed_supported(self.L, self.K, dk)
        own = getattr(self.bucket_probs, "__func__", None) is not _BUCKET_PROBS
        placed = self.q_norm is not None or self.rope_pairs > 0
        if not own and not placed and (hashed or not self.causal):
            return ModuleRaceFunction.apply(Khf, Vhf, Qhf, self.planes_T, self.L, self.K, bool(self.causal),
                                            torch.is_grad_enabled())
        if placed:
            Kh2, Qh2, V2 = self._streams(Khf, Vhf, Qhf, positions)
        else:
            Kh2 = Khf.permute(0, 1, 3, 2, 4).contiguous().view(N, T, dk)
            Qh2 = Qhf.permute(0, 1, 3, 2, 4).contiguous().view(N, T, dk)
            V2 = Vhf.permute(0, 1, 3, 2, 4).contiguous().view(N, T, dk)
        if hashed:
            planes = self.planes_T.t().contiguous().float()  # [L*K, d_k]
            out2 = race_fused_fwd_hashed(Kh2, Qh2, V2, planes, self.L)
        else:
            probsK = self.bucket_probs(Kh2).contiguous()
            probsQ = self.bucket_probs(Qh2).contiguous()
            out2 = race_fused_fwd(probsQ, probsK, V2, self.causal)
        return out2.view(M, B, H, T, dk).permute(0, 1, 3, 2, 4)


# The hashing the one-op forward stands for; any other bucket_probs (a
# subclass's, an instance's, one put on the class) is called instead.
_BUCKET_PROBS = BatchedACE.bucket_probs
