"""What a gradient of the recurrent layer with a path missing looks like, on the CPU in 64 bits: far
outside the tolerance that test_gpu_recurrent_layer_gradients holds the layer's to."""
from __future__ import annotations

import pytest
import torch

import layer_reference

B, T, H, Hk, d, dv, D = 3, 70, 4, 2, 64, 48, 256
TOLERANCE = 2 * 6 * 256 * 2.0 ** -24


@pytest.fixture(scope="module")
def plain():
    g = torch.Generator().manual_seed(0)
    n = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)
    leaves = {}
    for name, shape in layer_reference.shapes(B, T, H, Hk, d, dv, D).items():
        t = 1 + 0.1 * n(*shape) if len(shape) == 1 else n(*shape) / (shape[-1] ** 0.5 if len(shape) == 2 else 1)
        leaves[name] = {"residual": 2 * t, "state": t / 8}.get(name, t).requires_grad_(True)
    ups = n(B, T, D), n(B, T, D), n(B * H, d, dv)
    unit = torch.full((d,), 0.99 * d ** -0.5, dtype=torch.float64)
    freq = 10000.0 ** (-torch.arange(d // 4, dtype=torch.float64) / (d // 4))

    def grads(cut=()):
        outs = layer_reference.layer(leaves, unit, freq, H, Hk, cut)
        got = torch.autograd.grad(outs, list(leaves.values()), ups, allow_unused=True)
        return [torch.zeros_like(t) if d is None else d for t, d in zip(leaves.values(), got)]

    return grads, grads()


@pytest.mark.parametrize("path", layer_reference.PATHS)
def test_a_missing_path_is_seen(plain, path):
    grads, whole = plain
    off = [float((a - b).norm() / b.norm()) for a, b in zip(grads((path,)), whole)]
    assert max(off) > 100 * TOLERANCE, off
