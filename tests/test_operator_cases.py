"""The plain forms of perf/operators.py on the CPU: a pass leaves its inputs as
they were, a second pass gives the same outputs, and both agree with the
definitions in 64 bits.

Tolerance: fp32 sums of at most a few hundred terms of size up to 10, 2^-24 each:
1e-4 of the largest output."""
from __future__ import annotations

import pytest
import torch

from perf import operators as ops


def _tensors(case):
    g = torch.Generator().manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g)
    if case["op"] == "norm_rope":
        B, T, Hq, Hk, d = (case[i] for i in ("B", "T", "Hq", "Hk", "d"))
        axes = 3 if case["sections"] else 1
        pos = torch.randint(0, 1000, (axes, B, T), generator=g)
        return dict(q=n(B, T, Hq, d), k=n(B, T, Hk, d), q_weight=1 + 0.1 * n(d), k_weight=1 + 0.1 * n(d),
                    inv_freq=torch.rand(case["pairs"], generator=g), positions=pos if axes > 1 else pos[0],
                    dq=n(B * Hq, T, d), dk=n(B * Hk, T, d))
    if case["op"] == "scan":
        N, T, D = case["N"], case["T"], case["D"]
        gate = n(N, T, D) + 2.0
        x = dict(x=n(N, T, D), gate=gate if case["form"] == "sigmoid" else torch.nn.functional.logsigmoid(gate),
                 state=n(N, D), dout=n(N, T, D), dfinal=n(N, D))
        if case["ragged"]:
            x["lengths"] = torch.randint(0, T + 1, (N,), generator=g, dtype=torch.int32)
        return x
    B, H, Hk, Tq, Tk, L, R, d = (case[i] for i in ("B", "H", "Hk", "Tq", "Tk", "L", "R", "d"))
    p = lambda N, T: torch.softmax(n(N, T, L, R), -1)
    x = dict(q=p(B * H, Tq), k=p(B * Hk, Tk), v=n(B * Hk, Tk, d), dout=n(B * H, Tq, d))
    if case["op"] == "cross_query":
        k = x.pop("k").flatten(2)
        x["state"] = torch.cat([torch.matmul(k.transpose(1, 2), x.pop("v")).flatten(1), k.sum(1)], 1)
    elif case["ragged"]:
        x["lengths"] = torch.randint(0, Tk + 1, (B,), generator=g, dtype=torch.int32)
    return x


CASES = ([ops._norm_rope("", 2, 9, 4, 2, 24, 8, "f32", sections, interleaved, train)
          for sections, interleaved, train in (("", False, True), ("2,3,3", True, True), ("", True, False))]
         + [ops._scan("", 3, 37, 5, "f32", form, complement, ragged, train)
            for form, complement in (("sigmoid", True), ("log", False)) for ragged in (False, True) for train in (False, True)]
         + [ops._cross("", 2, 4, 2, 7, 20, 2, 4, 6, "f32", ragged, train) for ragged in (False, True) for train in (False, True)]
         + [ops._cross("", 2, 4, 2, 3, 20, 2, 4, 6, "f32", False, False, "cross_query")])


def _list(outs):
    return list(outs) if isinstance(outs, tuple) else [outs]


@pytest.mark.parametrize("case", CASES, ids=lambda c: " ".join(str(v) for v in c.values()))
def test_plain_passes_repeat_and_leave_their_inputs(case):
    x = _tensors(case)
    before = {name: t.clone() for name, t in x.items()}
    x["case"] = case
    assert not ops.own
    first, second = _list(ops.run(x)), _list(ops.run(x))
    for name, t in before.items():
        assert torch.equal(x[name], t), f"{name} changed"
    exact = _list({"norm_rope": ops._exact_norm_rope, "scan": ops._exact_scan}.get(case["op"], ops._exact_cross)(case, before))
    assert len(first) == len(second) == len(exact)
    for a, b, want in zip(first, second, exact):
        assert torch.equal(a, b)
        assert (a.double() - want).abs().max() <= 1e-4 * want.abs().max().clamp(min=1.0)
