"""Value streams of one key stream that end at different tokens: what the key stream holds
behind a value stream's end does not reach that stream."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_delta_rule import BF16, F32, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T, lengths, at", [(100, (40, 90, 64, 100), (50, 70)), (1600, (700, 1600, 0, 1300), (705, 1290))])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_tokens_behind_a_value_streams_end(race, cuda, T, lengths, at, bad, dtype):
    # Streams 0 and 2 have ended where their key stream's token `at` is not finite; 1 and 3 read it.
    *args, dout, dfinal = make(4, 2, T, 40, 48, dtype, seed=41)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    runs = []
    for x in (None, bad):
        leaves = [t.clone() for t in args]
        if x is not None:
            for stream, t in enumerate(at):
                leaves[0][stream, t, 3], leaves[1][stream, t] = x, x
        leaves = [t.requires_grad_(True) for t in leaves]
        outs = race.race_delta_rule(*leaves, scale=0.25, lengths=n)
        runs.append((*outs, *torch.autograd.grad(outs, leaves, (dout, dfinal))[2:]))
    for clean, got in zip(*runs):
        assert torch.equal(got[0::2], clean[0::2])
    assert not torch.isfinite(runs[1][0][1::2]).all()
