"""race_add_norm_e4m3 where the exact value lies half way between two of 8 bits: the rounding of
the factors decides, and it is that of the formula in elementary operations."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows, D, group", [(4000, 256, 0), (4000, 256, 32), (1000, 2048, 128), (200, 8192, 64), (1500, 1000, 0)])
def test_halves_fall_as_in_elementary_operations(race, cuda, rows, D, group, dtype):
    # Rows of small whole numbers: their sums of squares are exact in any order, so both forms have the same norm.
    g = torch.Generator(device=cuda).manual_seed(D + group)
    whole = lambda: torch.randint(-7, 8, (rows, D), generator=g, device=cuda).to(dtype)
    x, res = whole(), whole()
    w = (1 + 0.1 * torch.randn(D, generator=g, device=cuda)).bfloat16().to(dtype)
    y8, scales, s = race.race_add_norm_e4m3(x, res, w, eps=2.0 ** -20, group=group)
    assert torch.equal(s, x + res)
    mean = (s.double().pow(2).sum(-1, keepdim=True).float() / D) + 2.0 ** -20
    y = (s.float() * torch.rsqrt(mean)) * w.float()
    size = group or D
    parts = torch.nn.functional.pad(y, (0, -D % size)).view(rows, -1, size)
    most = parts.abs().amax(-1, keepdim=True)
    want = (parts * (most.reciprocal() * 448.0)).flatten(1)[:, :D].to(torch.float8_e4m3fn)
    differ = (y8.float() != want.float())
    assert not differ.any(), f"{int(differ.sum())} of {differ.numel()}"
