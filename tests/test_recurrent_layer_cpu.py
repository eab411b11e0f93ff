"""CPU tests of the gated delta rule's layer: what it refuses, before any device
is touched, and the sizes it reports."""
from __future__ import annotations

import pytest
import torch


def test_add_norm_refuses_on_the_host(race):
    from race_attention_kernel_amd import abi

    bad = abi.RACE_ERROR_INVALID_VALUE
    ok = abi.add_norm_shape(300, 2048)
    st, nbytes = abi.add_norm_bwd_workspace_bytes(ok)
    assert st == abi.RACE_SUCCESS and nbytes > 0 and nbytes % (2048 * 4) == 0
    for kw in (dict(rows=-1), dict(rows=1 << 46), dict(D=0), dict(D=16385), dict(dtype=2), dict(weight_dtype=2), dict(eps=-1.0),
               dict(eps=float("nan")), dict(out=2), dict(group=32), dict(out=1, group=16), dict(out=1, group=32, D=60),
               dict(out=1, group=32, x_stride=2050), dict(x_stride=-8), dict(residual_stride=(1 << 40) + 1)):
        assert abi.add_norm_bwd_workspace_bytes(abi.add_norm_shape(**(dict(rows=300, D=2048) | kw)))[0] == bad, kw
    e4m3 = abi.add_norm_shape(300, 2048, out=1, group=128)
    assert abi.add_norm_fwd(0, None, None, 16, None, None, ok, 0) == bad
    assert abi.add_norm_fwd(16, None, None, 8, None, None, ok, 0) == bad
    assert abi.add_norm_fwd(16, 16, None, 16, None, None, ok, 0) == bad  # nowhere for the sum
    assert abi.add_norm_fwd(16, None, None, 16, None, None, e4m3, 0) == bad  # nowhere for the scales
    assert abi.add_norm_bwd(16, None, 16, None, 16, None, e4m3, None, 0, 0) == bad
    assert abi.add_norm_bwd(0, None, 16, None, 16, None, ok, None, 0, 0) == bad
    assert abi.add_norm_bwd(16, 16, 16, None, 16, 16, ok, None, 0, 0) == bad
    assert abi.add_norm_bwd(16, 16, 16, None, 16, 16, ok, 16, nbytes - 1, 0) == bad
    # Nothing to do touches no device.
    assert abi.add_norm_fwd(0, None, None, 0, None, None, abi.add_norm_shape(0, 64), 0) == 0
    assert abi.add_norm_bwd(16, None, 16, None, None, None, ok, None, 0, 0) == 0
    assert abi.add_norm_bwd(0, None, None, None, 16, None, abi.add_norm_shape(0, 64), None, 0, 0) == 0
    x = torch.zeros(3, 64)
    with pytest.raises(RuntimeError, match="race_add_norm: x lives on the CPU"):
        race.race_add_norm(x, x)
    with pytest.raises(RuntimeError, match="race_add_norm_e4m3: x lives on the CPU"):
        race.race_add_norm_e4m3(x)


def test_gate_norm_refuses_on_the_host(race):
    from race_attention_kernel_amd import abi

    bad = abi.RACE_ERROR_INVALID_VALUE
    ok = abi.gate_norm_shape(2, 300, 12, 128)
    st, nbytes = abi.gate_norm_bwd_workspace_bytes(ok)
    assert st == abi.RACE_SUCCESS and nbytes > 0 and nbytes % (128 * 4) == 0
    for kw in (dict(B=-1), dict(T=-1), dict(B=1 << 16, T=1 << 15), dict(H=0), dict(H=65536), dict(d=0), dict(d=257), dict(dtype=2),
               dict(weight_dtype=-1), dict(eps=-1.0)):
        assert abi.gate_norm_bwd_workspace_bytes(abi.gate_norm_shape(**(dict(B=2, T=300, H=12, d=128) | kw)))[0] == bad, kw
    assert abi.gate_norm_fwd(16, 0, None, 16, ok, 0) == bad
    assert abi.gate_norm_fwd(16, 16, 4, 16, ok, 0) == bad
    assert abi.gate_norm_bwd(16, 16, None, 0, 16, 16, None, ok, None, 0, 0) == bad
    assert abi.gate_norm_bwd(16, 16, 16, 16, 16, 16, 16, ok, 16, nbytes - 4, 0) == bad
    # Nothing to do touches no device.
    assert abi.gate_norm_fwd(0, 0, None, 0, abi.gate_norm_shape(0, 5, 1, 64), 0) == 0
    assert abi.gate_norm_bwd(16, 16, None, 16, None, None, None, ok, None, 0, 0) == 0
    with pytest.raises(RuntimeError, match="race_gate_norm: x lives on the CPU"):
        race.race_gate_norm(torch.zeros(6, 4, 64), torch.zeros(2, 4, 3, 64))
