"""CPU tests of the gated delta rule's layer: what it refuses, before any device
is touched, the sizes it reports, and the plain forms of its timed cases."""
from __future__ import annotations

import pytest
import torch

from perf import more_operators as more


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


def test_delta_rule_refuses_on_the_host(race):
    from race_attention_kernel_amd import abi

    bad = abi.RACE_ERROR_INVALID_VALUE
    ok = abi.delta_shape(4, 300, 64, 48, key_streams=2)
    st, nbytes, records = abi.delta_workspace_bytes(ok, True)
    assert st == abi.RACE_SUCCESS and records > 0
    st, alone, _ = abi.delta_workspace_bytes(ok)
    assert st == abi.RACE_SUCCESS and alone > nbytes >= 0  # with records, they hold what else is workspace
    st, back = abi.delta_bwd_workspace_bytes(ok)
    assert st == abi.RACE_SUCCESS and back > 0
    base = dict(N=4, T=300, dk=64, dv=48, key_streams=2)
    for kw in (dict(N=-4), dict(N=65536), dict(N=5), dict(key_streams=0), dict(key_streams=8), dict(key_streams=-2), dict(T=-1),
               dict(T=(1 << 30) + 1), dict(N=64, T=1 << 25), dict(dk=0), dict(dk=129), dict(dv=0), dict(dv=257), dict(dtype=2),
               dict(gate_dtype=2), dict(gate_dtype=-1), dict(gate_form=2), dict(gate_form=-1), dict(lengths_group=0),
               dict(scale=float("inf")), dict(scale=float("nan")), dict(strides=(-1, 64, 19200, 64, 14400, 48)),
               dict(strides=(19200, 64, 19200, (1 << 30) + 1, 14400, 48)), dict(strides=(19200, 64, 19200, 64, (1 << 40) + 1, 48))):
        sh = abi.delta_shape(**(base | kw))
        assert abi.delta_workspace_bytes(sh)[0] == bad, kw
        assert abi.delta_bwd_workspace_bytes(sh)[0] == bad, kw
        assert abi.delta_fwd(16, 16, 16, 16, 16, None, None, 16, 16, None, sh, 16, 1 << 40, 0) == bad, kw
        assert abi.delta_bwd(16, 16, 16, 16, None, 16, None, 16, 16, None, None, None, None, None, sh, 16, 1 << 40, 0) == bad, kw

    fwd = dict(q=16, k=16, v=16, gate=16, beta=16, state=None, lengths=None, out=16, final=16, records=None, sh=ok, ws=16,
               bytes=alone, stream=0)
    for kw in (dict(q=0), dict(k=0), dict(v=0), dict(beta=0), dict(out=0), dict(q=24), dict(gate=20), dict(state=8), dict(final=4),
               dict(records=8), dict(ws=0), dict(ws=8), dict(bytes=alone - 1), dict(bytes=0)):
        assert abi.delta_fwd(*(fwd | kw).values()) == bad, kw
    bwd = dict(q=16, k=16, gate=16, beta=16, lengths=None, dout=16, dfinal=None, records=16, dq=16, dk=None, dv=None, dgate=None,
               dbeta=None, dstate=None, sh=ok, ws=16, bytes=back, stream=0)
    for kw in (dict(q=0), dict(k=0), dict(beta=0), dict(dout=0), dict(records=0), dict(records=8), dict(dq=8), dict(dstate=4),
               dict(gate=None, dgate=16), dict(ws=0), dict(ws=4), dict(bytes=back - 1)):
        assert abi.delta_bwd(*(bwd | kw).values()) == bad, kw
    # Nothing to do touches no device.
    none = abi.delta_shape(0, 300, 64, 48)
    assert abi.delta_workspace_bytes(none)[:2] == (0, 0)
    assert abi.delta_fwd(0, 0, 0, None, 0, None, None, 0, None, None, none, None, 0, 0) == 0
    assert abi.delta_bwd(0, 0, None, 0, None, 0, None, 0, None, None, None, None, None, None, none, None, 0, 0) == 0
    assert abi.delta_bwd(*(bwd | dict(dq=None)).values()) == 0
    assert abi.delta_fwd(0, 0, 0, None, 0, 16, None, 0, 16, None, abi.delta_shape(4, 0, 64, 48), None, 0, 0) == 0
    # A few tokens need no memory, and long sequences of few streams more than the sum of their chunks.
    assert abi.delta_workspace_bytes(abi.delta_shape(4, 16, 64, 48))[1] == 0
    one, two = (abi.delta_workspace_bytes(abi.delta_shape(1, T, 64, 48))[1] for T in (512, 2048))
    assert two > 4 * one > 0


def test_delta_rule_refuses_tensors_of_the_host(race):
    q, v, g = torch.zeros(2, 5, 16), torch.zeros(2, 5, 8), torch.zeros(2, 5)
    with pytest.raises(RuntimeError, match="race_delta_rule: q lives on the CPU"):
        race.race_delta_rule(q, q, v, g, g)
    with pytest.raises(RuntimeError, match="race_delta_rule_carry: q lives on the CPU"):
        race.race_delta_rule_carry(q, q, v, g, g, torch.zeros(2, 16, 8))
    with pytest.raises(ValueError, match="gate_form"):
        race.race_delta_rule_carry(q, q, v, g, g, torch.zeros(2, 16, 8), gate_form="exp")


# ---- the timed cases' plain forms ----

def _tensors(case):
    g = torch.Generator().manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)
    if case["op"] == "delta":
        B, H, Hk, T, dk, dv = (case[i] for i in ("B", "H", "Hk", "T", "dk", "dv"))
        gate = n(B * H, T) + 2.0
        if case["form"] == "log":
            gate = torch.nn.functional.logsigmoid(gate)
        if case["resets"]:
            gate[:, T // 3] = -float("inf")
        x = dict(q=unit(n(B * Hk, T, dk)), k=unit(n(B * Hk, T, dk)), v=n(B * H, T, dv), gate=gate, beta=torch.sigmoid(n(B * H, T)),
                 dout=n(B * H, T, dv))
        if case["state"]:
            x.update(state=n(B * H, dk, dv), dfinal=n(B * H, dk, dv))
        if case["ragged"]:
            x["lengths"] = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
        return x
    if case["op"] == "add_norm":
        rows, D = case["rows"], case["D"]
        x = dict(x=n(rows, D), weight=1 + 0.1 * n(D), dy=n(rows, D))
        return dict(x, residual=n(rows, D), dsum=n(rows, D)) if case["residual"] else x
    B, T, H, d = (case[i] for i in ("B", "T", "H", "d"))
    return dict(x=n(B * H, T, d), gate=n(B, T, H, d), weight=1 + 0.1 * n(d), dy=n(B, T, H, d))


CASES = ([more._delta("", 2, 4, 2, T, 16, 12, "f32", form, True, ragged, False, train)
          for T in (5, 130, 200) for form in ("log", "sigmoid") for ragged in (False, True) for train in (False, True)]
         + [more._delta("", 2, 2, 2, 1, 16, 12, "f32", form, True) for form in ("log", "sigmoid")]
         + [more._delta("", 2, 2, 2, 150, 16, 12, "f32", "log", False, False, True, train) for train in (False, True)]
         + [more._add_norm("", 5, 37, "f32", "same", 0, residual, train) for residual in (False, True) for train in (False, True)]
         + [more._gate_norm("", 2, 7, 3, 16, "f32", train) for train in (False, True)])


@pytest.mark.parametrize("case", CASES, ids=lambda c: " ".join(str(v) for v in c.values()))
def test_plain_passes_repeat_and_leave_their_inputs(case):
    # fp32 sums of at most a few hundred terms of size up to 10, 2^-24 each: 1e-4 of the largest output.
    x = _tensors(case)
    before = {name: t.clone() for name, t in x.items()}
    x["case"] = case
    assert not more.own
    first, second = more.run(x), more.run(x)
    for name, t in before.items():
        assert torch.equal(x[name], t), f"{name} changed"
    exact = {"delta": more._exact_delta, "add_norm": more._exact_add_norm, "gate_norm": more._exact_gate_norm}[case["op"]](case, before)
    assert len(first) == len(second) == len(exact)
    for a, b, want in zip(first, second, exact):
        assert torch.equal(a, b)
        assert (a.double() - want).abs().max() <= 1e-4 * want.abs().max().clamp(min=1.0)
