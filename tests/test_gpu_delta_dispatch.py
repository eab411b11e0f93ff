"""The delta rule's launches that few sizes reach: maps and joins of rows in no whole pieces, and chunks' gradients
with more chunks than workgroups."""
from __future__ import annotations

import pytest
import torch

from test_gpu_delta_rule import BF16, F32, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N, Nk, T, dk, dv", [(1, 1, 1600, 33, 17), (2, 1, 1700, 127, 50), (2, 2, 1600, 128, 50), (1, 1, 1600, 64, 50),
                                              (2, 2, 1700, 66, 100)])
def test_segments_of_any_rows(race, cuda, N, Nk, T, dk, dv, dtype):
    *args, dout, dfinal = make(N, Nk, T, dk, dv, dtype, seed=61)
    args[3].clamp_(min=-0.5)
    lengths = torch.tensor([T, 1025][:N], dtype=torch.int32, device=cuda)
    check(race, args, dout, dfinal, dtype, f"{dk} x {dv}", scale=dk ** -0.5, lengths=lengths)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N, Nk, T, dk, dv", [(100, 100, 200, 33, 17), (100, 100, 200, 100, 50), (140, 70, 250, 64, 50), (100, 100, 200, 128, 36),
                                              (140, 70, 250, 128, 64)])
def test_more_chunks_than_workgroups(race, cuda, N, Nk, T, dk, dv, dtype):
    *args, dout, dfinal = make(N, Nk, T, dk, dv, dtype, seed=62)
    lengths = torch.randint(0, T + 1, (N,), generator=torch.Generator().manual_seed(63), dtype=torch.int32).to(cuda)
    for n in (None, lengths):
        check(race, args, dout, dfinal, dtype, f"{dk} x {dv}", scale=dk ** -0.5, lengths=n)
