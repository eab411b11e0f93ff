"""race_add_norm, race_add_norm_e4m3 and race_gate_norm against their formulas in 64 bits.

Tolerances come from the arithmetic, with u = 2^-24 (half a step of fp32).  The
sum of a row's D positive squares runs over at most 32 values a lane, then over
lanes and waves: 48 u relative, half of that in the root, the reciprocal root 4 u,
and a few products: y is within 40 u of itself plus half a step of its type.  A
mean of signed products m = mean(g u) has the same 48 u of mean |g u|, so
    dx = r (g - u m) + ds   is within   80 u r (|g| + |u| mean |g u|) + 2 u |ds|
plus half a step; a sum over R rows in runs of at most R within (R + 48) u of the
sum of magnitudes.  sigmoid(z) is good to (8 + 2 |z|) u, its exponential taking
z log2(e) rounded once.
"""
from __future__ import annotations

import pytest
import torch

from gpu_util import say

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
EPS = 1e-6
F32, BF16 = torch.float32, torch.bfloat16


def close(name, got, want, bound, dtype):
    got, want, bound = got.detach().double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bound = bound + HALF[dtype] * (want.abs() + bound) + 1e-37
    over = ((got - want).abs() / bound)
    say(name, tuple(want.shape), f"error {float(over.max()) if over.numel() else 0:.3f} of the bound")
    assert torch.isfinite(got).all() and (over <= 1).all(), f"{name}: {float(over.max())} of the bound"


def normal(*shape, seed=0, device="cuda"):
    return torch.randn(*shape, generator=torch.Generator(device=device).manual_seed(seed), device=device)


def reference(s, w, dy=None, ds=None):
    """y, dx, dw with their bounds for normed rows s [rows, D] (64 bits)."""
    s, w = s.double(), w.double()
    r = (s.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    unit = s * r
    out = {"y": (unit * w, 40 * U * (unit * w).abs())}
    if dy is not None:
        g = dy.double() * w
        dx = r * (g - unit * (g * unit).mean(-1, keepdim=True)) + ds.double()
        err = 80 * U * r * (g.abs() + unit.abs() * (g * unit).abs().mean(-1, keepdim=True)) + 2 * U * ds.double().abs()
        terms = dy.double() * unit
        out["dx"], out["dw"] = (dx, err), (terms.sum(0), (len(s) + 48) * U * terms.abs().sum(0))
    return out


# Each launch shape: a wave or a workgroup a row, pieces of 8, 4 or 1; and the widths around them.
WIDTHS = [1, 7, 64, 65, 250, 256, 512, 520, 1000, 1001, 1024, 2048, 2056, 4096, 4100, 8192, 12000, 16376, 16384, 16383]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", WIDTHS)
def test_add_norm_and_gradients(race, cuda, D, dtype):
    rows = 13
    x, res, dy, ds = (normal(rows, D, seed=i).to(dtype) for i in range(4))
    w = (1 + 0.3 * normal(D, seed=9)).to(dtype)
    leaves = [t.requires_grad_(True) for t in (x, res, w)]
    y, s = race.race_add_norm(*leaves, eps=EPS)
    assert torch.equal(s, (x.float() + res.float()).to(dtype))
    got = torch.autograd.grad((y, s), leaves, (dy, ds))
    want = reference(s.detach(), w.detach(), dy, ds)
    close("y", y, *want["y"], dtype)
    close("dx", got[0], *want["dx"], dtype)
    assert torch.equal(got[0], got[1])
    close("dw", got[2], *want["dw"], dtype)


@pytest.mark.parametrize("rows, D, dtype", [(1, 64, BF16), (4099, 256, BF16), (9001, 130, F32), (2500, 4096, BF16), (5000, 33, BF16)])
def test_add_norm_of_many_rows(race, cuda, rows, D, dtype):
    x, dy = (normal(rows, D, seed=i).to(dtype) for i in range(2))
    w = (1 + 0.3 * normal(D, seed=9)).requires_grad_(True)  # float32 whatever the rows
    y, s = race.race_add_norm(x.requires_grad_(True), weight=w, eps=EPS)
    assert s is None
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert dw.dtype == F32
    want = reference(x.detach(), w.detach(), dy, torch.zeros_like(dy))
    close("y", y, *want["y"], dtype)
    close("dx", dx, *want["dx"], dtype)
    close("dw", dw, *want["dw"], F32)


def test_add_norm_with_parts_missing(race, cuda):
    x, res, up = (normal(3, 5, 96, seed=i).requires_grad_(True) for i in range(3))
    zero = torch.zeros(15, 96, device=cuda)
    y, s = race.race_add_norm(x, res, eps=EPS)  # no weight
    assert y.shape == s.shape == x.shape
    one = torch.ones(96, device=cuda)
    for outs, grads, dy, ds in (((y,), (up,), up, zero), ((s,), (up,), zero, up)):  # one of the two upstreams
        got = torch.autograd.grad(outs, (x, res), grads, retain_graph=True)
        want = reference(s.detach().flatten(0, 1), one, dy.detach().view(15, 96), ds.detach().view(15, 96))
        close("dx", got[0].flatten(0, 1), *want["dx"], F32)
    only = torch.autograd.grad(y, res, up, retain_graph=True)
    assert torch.equal(only[0], torch.autograd.grad(y, x, up)[0])
    with torch.no_grad():
        assert torch.equal(race.race_add_norm(x, res, eps=EPS)[0], y)


def test_add_norm_strides(race, cuda):
    joint = normal(6, 4, 300).to(BF16)
    for view in (joint[:, 1], joint[..., 8:264], joint[..., 3:259], joint.transpose(0, 1), joint[:, :, ::2], joint[:, :1].expand(6, 4, 300)):
        res = normal(*view.shape, seed=3).to(BF16)
        y, s = race.race_add_norm(view, res, eps=EPS)
        assert torch.equal(s, (view.float() + res.float()).to(BF16))
        want, bound = reference(s, torch.ones(s.shape[-1], device=cuda))["y"]
        close("strides", y, want, bound, BF16)
        y2, s2 = race.race_add_norm(res, view, eps=EPS)
        assert torch.equal(s2, s)
        close("strides", y2, want, bound, BF16)
    # A residual that all rows share: its gradient is the sum of theirs.
    x, one = normal(9, 64), normal(64, seed=5).requires_grad_(True)
    y, _ = race.race_add_norm(x, one.expand(9, 64), eps=EPS)
    up = normal(9, 64, seed=6)
    (got,) = torch.autograd.grad(y, one, up)
    want, bound = reference((x + one.detach()), torch.ones(64, device=cuda), up, torch.zeros_like(up))["dx"]
    close("shared", got, want.sum(0), bound.sum(0) + 9 * U * want.abs().sum(0), F32)


@pytest.mark.parametrize("rows, D", [(0, 64), (5, 64)])
def test_add_norm_empty_and_special_rows(race, cuda, rows, D):
    x = normal(rows, D).requires_grad_(True)
    w = torch.ones(D, device=cuda, requires_grad=True)
    y, s = race.race_add_norm(x, torch.zeros_like(x), w, eps=EPS)
    dx, dw = torch.autograd.grad((y, s), (x, w), (torch.ones_like(y), torch.ones_like(y)))
    assert y.shape == dx.shape == (rows, D) and dw.shape == (D,)
    if rows == 0:
        assert (dw == 0).all()
        return
    odd = torch.stack([torch.zeros(D, device=cuda), torch.full((D,), float("inf"), device=cuda),
                       normal(D).index_fill(0, torch.tensor([3], device=cuda), float("nan")), normal(D, seed=2)])
    y, _ = race.race_add_norm(odd, eps=EPS)
    assert (y[0] == 0).all() and y[1].isnan().all() and y[2].isnan().all() and torch.isfinite(y[3]).all()
    assert torch.equal(y[3], race.race_add_norm(odd[3:], eps=EPS)[0][0])  # the others do not reach it


def _check_e4m3(y8, scales, y, group, dtype):
    rows, D = y.shape
    size = group or D
    parts = y.abs().split(size, -1)
    most = torch.stack([p.amax(-1) for p in parts], -1)
    assert scales.shape == most.shape and scales.dtype == F32 and y8.dtype == torch.float8_e4m3fn
    assert ((scales.double() - most / 448).abs() <= 48 * U * most / 448).all()
    wide = scales.double().repeat_interleave(size, -1)[:, :D]
    # Half a step of e4m3: 2^-4 of the value, or 2^-10 where it is subnormal; the fp32 value in front of it is 48 u off.
    bound = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * wide) + 64 * U * y.abs()
    off = (y8.double() * wide - y).abs()
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D, group", [(64, 0), (4096, 0), (1001, 0), (5, 0), (16384, 0), (4096, 128), (4096, 64), (4096, 32),
                                      (200, 128), (8, 32), (1000, 64), (16376, 128)])
def test_e4m3_rows(race, cuda, D, group, dtype):
    x, res = (3 * normal(7, D, seed=1)).to(dtype), normal(7, D, seed=2).to(dtype)
    w = (1 + 0.3 * normal(D, seed=9)).to(dtype)
    y8, scales, s = race.race_add_norm_e4m3(x, res, w, eps=EPS, group=group)
    assert torch.equal(s, race.race_add_norm(x, res, w, eps=EPS)[1])
    _check_e4m3(y8, scales, reference(s, w)["y"][0], group, dtype)
    y8n, scales_n, none = race.race_add_norm_e4m3(s, None, w, eps=EPS, group=group)
    assert none is None and torch.equal(y8n.view(torch.uint8), y8.view(torch.uint8)) and torch.equal(scales_n, scales)


def test_e4m3_special_rows(race, cuda):
    D = 256
    rows = torch.stack([torch.zeros(D, device=cuda), 1e-30 * normal(D), normal(D).index_fill(0, torch.tensor([200], device=cuda), float("nan")),
                        1e18 * normal(D)])
    for group in (0, 128):
        y8, scales, _ = race.race_add_norm_e4m3(rows, eps=0.0 if group else EPS, group=group)
        y = y8.float().view(4, -1, group or D) * scales[..., None]
        assert y[2].isnan().all() and torch.isfinite(y[3]).all()
        if group == 0:
            assert (y8[0].float() == 0).all() and (scales[0] == 0).all() and torch.isfinite(y[1]).all()
    # A group of zeros beside a group that is not.
    one = normal(1, D)
    one[0, :128] = 0
    y8, scales, _ = race.race_add_norm_e4m3(one, group=128)
    assert scales[0, 0] == 0 and (y8[0, :128].float() == 0).all() and scales[0, 1] > 0


def test_e4m3_strides_and_shapes(race, cuda):
    joint = normal(3, 5, 300).to(BF16)
    for view in (joint[..., 8:264], joint[..., 4:260], joint.transpose(0, 1)[..., :256]):
        for group in (0, 64):
            # Rows in pieces of 8 and rows value by value sum their squares in another order.
            y8, scales, _ = race.race_add_norm_e4m3(view, group=group)
            assert y8.shape == view.shape and scales.shape == (*view.shape[:-1], 4 if group else 1)
            y = reference(view.reshape(15, 256), torch.ones(256, device=cuda))["y"][0]
            _check_e4m3(y8.view(15, 256), scales.view(15, -1), y, group, BF16)
    y8, scales, s = race.race_add_norm_e4m3(joint[:0], joint[:0])
    assert y8.shape == s.shape == (0, 5, 300) and scales.shape == (0, 5, 1)


def gate_reference(x, z, w, dy):
    """Outputs and bounds of race_gate_norm on streams x [B * H, T, d]."""
    B, T, H, d = z.shape
    x = x.double().view(B, H, T, d).transpose(1, 2)
    z, w, dy = z.double(), w.double(), dy.double()
    r = (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    unit, sig = x * r, torch.sigmoid(z)
    silu, c = z * sig, (48 + 2 * z.abs()) * U
    y = unit * w * silu
    g = dy * silu * w
    dx = r * (g - unit * (g * unit).mean(-1, keepdim=True))
    # Each g carries the gate's own error into the mean.
    ex = r * ((80 * U + c) * g.abs() + unit.abs() * ((80 * U + c) * (g * unit).abs()).mean(-1, keepdim=True))
    slope = sig * (1 + z * (1 - sig))
    # sigma (1 + z (1 - sigma)): both parts by their magnitudes.
    dz, ez = dy * unit * w * slope, (dy * unit * w).abs() * (c + 8 * U) * (sig + (z * sig * (1 - sig)).abs() * 2)
    terms = dy * silu * unit
    rows = terms[..., 0].numel()
    streams = lambda t: t.transpose(1, 2).reshape(B * H, T, d)
    return {"y": (y, c * y.abs()), "dx": (streams(dx), streams(ex)), "dz": (dz, ez),
            "dw": (terms.sum((0, 1, 2)), ((rows + 48) * U + c.amax()) * terms.abs().sum((0, 1, 2)))}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B, T, H, d", [(2, 7, 3, 64), (1, 1, 1, 1), (64, 1, 16, 128), (3, 65, 2, 256), (2, 9, 5, 33), (1, 300, 12, 96),
                                        (2, 40, 4, 40), (1, 2, 3, 8), (2, 3, 2, 255)])
def test_gate_norm_and_gradients(race, cuda, B, T, H, d, dtype):
    x = normal(B * H, T, d, seed=1).to(dtype).requires_grad_(True)
    z = (3 * normal(B, T, H, d, seed=2)).to(dtype).requires_grad_(True)
    w = (1 + 0.3 * normal(d, seed=3)).to(dtype).requires_grad_(True)
    dy = normal(B, T, H, d, seed=4).to(dtype)
    y = race.race_gate_norm(x, z, w, eps=EPS)
    want = gate_reference(x.detach(), z.detach(), w.detach(), dy)
    close("y", y, *want["y"], dtype)
    for name, got in zip(("dx", "dz", "dw"), torch.autograd.grad(y, (x, z, w), dy)):
        close(name, got, *want[name], dtype)
    with torch.no_grad():
        assert torch.equal(race.race_gate_norm(x, z, w, eps=EPS), y)


def test_gate_norm_of_many_rows(race, cuda):
    B, T, H, d = 2, 3001, 8, 64
    x, z = normal(B * H, T, d, seed=1).requires_grad_(True), normal(B, T, H, d, seed=2)
    w = torch.ones(d, device=cuda, requires_grad=True)
    dy = normal(B, T, H, d, seed=4)
    y = race.race_gate_norm(x, z, w, eps=EPS)
    want = gate_reference(x.detach(), z, w.detach(), dy)
    close("y", y, *want["y"], F32)
    for name, got in zip(("dx", "dw"), torch.autograd.grad(y, (x, w), dy)):
        close(name, got, *want[name], F32)


def test_gate_norm_strides_extremes_and_empties(race, cuda):
    B, T, H, d = 2, 5, 3, 64
    streams, joint = normal(B * H, T + 2, 2 * d).to(BF16), normal(B, T, 2 * H, d + 8).to(BF16)
    for x, z in ((streams[:, 1:T + 1, :d], joint[:, :, :H, :d]), (streams[:, :T, 3:d + 3], joint[:, :, ::2, 5:d + 5])):
        assert torch.equal(race.race_gate_norm(x, z), race.race_gate_norm(x.contiguous(), z.contiguous()))
    z = torch.tensor([-1e4, -100.0, 0.0, 100.0, 1e4, 88.0, -88.0, 3.0], device=cuda).repeat(B, T, H, d // 8).requires_grad_(True)
    x = normal(B * H, T, d).requires_grad_(True)
    y = race.race_gate_norm(x, z)
    grads = torch.autograd.grad(y, (x, z), torch.ones_like(y))
    assert torch.isfinite(y).all() and all(torch.isfinite(g).all() for g in grads)
    assert (y[..., 0] == 0).all() and (y[..., 2] == 0).all()
    for shape in ((0, 5, 3), (2, 0, 3)):
        x, z = torch.zeros(shape[0] * 3, shape[1], 8, device=cuda, requires_grad=True), torch.zeros(*shape, 8, device=cuda)
        w = torch.ones(8, device=cuda, requires_grad=True)
        y = race.race_gate_norm(x, z, w)
        dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert y.shape == (*shape, 8) and dx.shape == x.shape and (dw == 0).all()


def test_gradients_of_gradients_and_tangents_are_refused(race, cuda):
    x, z = normal(6, 4, 16).requires_grad_(True), normal(2, 4, 3, 16).requires_grad_(True)
    for run in (lambda t: race.race_gate_norm(t, z), lambda t: race.race_add_norm(t)[0]):
        up = torch.ones_like(run(x)).requires_grad_(True)
        (g,) = torch.autograd.grad(run(x), x, up, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            g.sum().backward()
        with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="jvp"):
            run(torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x)))


@pytest.mark.parametrize("call", [
    lambda race, t: race.race_add_norm(t(3, 4), t(3, 5)), lambda race, t: race.race_add_norm(t(3, 4), t(3, 4).to(BF16)),
    lambda race, t: race.race_add_norm(t(3, 4).half()), lambda race, t: race.race_add_norm(t(3, 16385)),
    lambda race, t: race.race_add_norm(t(3, 4), weight=t(5)), lambda race, t: race.race_add_norm(t(3, 4), weight=t(4).to(BF16)),
    lambda race, t: race.race_add_norm(t(3, 4), weight=t(4).cpu()), lambda race, t: race.race_add_norm(t(3, 4), eps=-1.0),
    lambda race, t: race.race_add_norm(t(3, 4), eps=float("nan")), lambda race, t: race.race_add_norm(t(3, 4)[0, 0]),
    lambda race, t: race.race_add_norm_e4m3(t(3, 64), group=16), lambda race, t: race.race_add_norm_e4m3(t(3, 60), group=32),
    lambda race, t: race.race_add_norm_e4m3(t(3, 64), t(2, 64)),
    lambda race, t: race.race_gate_norm(t(6, 4, 16), t(2, 4, 3, 8)), lambda race, t: race.race_gate_norm(t(6, 4, 16), t(3, 4, 3, 16)),
    lambda race, t: race.race_gate_norm(t(6, 4, 257), t(2, 4, 3, 257)), lambda race, t: race.race_gate_norm(t(6, 4, 16), t(2, 4, 3, 16).to(BF16)),
    lambda race, t: race.race_gate_norm(t(6, 4, 16), t(2, 4, 3, 16), t(15))])
def test_refusals(race, cuda, call):
    with pytest.raises(RuntimeError, match="race_(add|gate)_norm"):
        call(race, lambda *s: torch.zeros(*s, device=cuda))


# Rows in pieces of two values and of one, through every number of pieces a thread holds.
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [2, 126, 130, 514, 1026, 2050, 4098, 5001, 8190, 8194, 8195, 10002, 12287, 16382])
def test_add_norm_of_narrow_pieces(race, cuda, D, dtype):
    test_add_norm_and_gradients(race, cuda, D, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [2, 130, 1002, 5001, 5002, 8195, 10002, 16382])
def test_e4m3_rows_of_narrow_pieces(race, cuda, D, dtype):
    test_e4m3_rows(race, cuda, D, 0, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B, T, H, d", [(2, 5, 3, 2), (1, 9, 2, 6), (2, 7, 3, 50), (3, 5, 2, 66), (1, 11, 4, 130), (2, 3, 2, 254), (2, 5, 3, 17),
                                        (2, 70, 3, 65), (1, 4, 5, 129), (1, 2000, 3, 33)])
def test_gate_norm_of_narrow_pieces(race, cuda, B, T, H, d, dtype):
    test_gate_norm_and_gradients(race, cuda, B, T, H, d, dtype)
