"""The recurrent layer's calls without a derivative of their own: what they do with inputs that
require gradients or carry forward-mode tangents."""
from __future__ import annotations

import pytest
import torch

from test_gpu_delta_rule import F32, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(6, 64), (2, 3, 256)])
@pytest.mark.parametrize("group", [0, 32])
def test_the_residual_stream_keeps_its_gradient_beside_rows_in_8_bits(race, cuda, shape, group):
    g = torch.Generator(device=cuda).manual_seed(51)
    n = lambda *s: torch.randn(*s, generator=g, device=cuda)
    x, res, w, up = n(*shape), n(*shape), n(shape[-1]), n(*shape)
    plain = race.race_add_norm_e4m3(x, res, w, group=group)
    leaves = [t.requires_grad_(True) for t in (x, res, w)]
    y8, scales, total = race.race_add_norm_e4m3(*leaves, group=group)
    for a, b in zip((y8.view(torch.uint8), scales, total), (plain[0].view(torch.uint8), *plain[1:])):
        assert a.shape == b.shape and torch.equal(a, b)
    assert total.requires_grad and not y8.requires_grad and not scales.requires_grad
    dx, dres, dw = torch.autograd.grad(total, leaves, up, allow_unused=True)
    assert torch.equal(dx, up) and torch.equal(dres, up) and dw is None
    # One of the two, a residual that all rows share, and a stream of two layers.
    (only,) = torch.autograd.grad(race.race_add_norm_e4m3(x.detach(), res, w, group=group)[2], res, up)
    assert torch.equal(only, up)
    one = n(shape[-1]).requires_grad_(True)
    (shared,) = torch.autograd.grad(race.race_add_norm_e4m3(x.detach(), one.expand(shape), group=group)[2], one, torch.ones_like(x))
    assert (shared == x.numel() // shape[-1]).all()
    second = race.race_add_norm_e4m3(2 * total.detach(), race.race_add_norm_e4m3(x, res, group=group)[2], group=group)[2]
    assert all(torch.equal(d, up) for d in torch.autograd.grad(second, (x, res), up))
    # Nothing is recorded where nothing is asked for.
    with torch.no_grad():
        assert not race.race_add_norm_e4m3(x, res, w, group=group)[2].requires_grad
    assert race.race_add_norm_e4m3(x, None, w, group=group)[2] is None
    assert not race.race_add_norm_e4m3(x.detach(), res.detach(), w, group=group)[2].requires_grad


def test_the_residual_streams_gradient_in_a_captured_step(race, cuda):
    x, res = (torch.randn(5, 128, device=cuda).requires_grad_(True) for _ in range(2))
    up = torch.randn(5, 128, device=cuda)

    def step():
        y8, scales, total = race.race_add_norm_e4m3(x, res)
        return (y8.view(torch.uint8), scales, *torch.autograd.grad(total * total, (x, res), up))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x)), res.copy_(torch.randn_like(res))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
    alive = race.race_add_norm_e4m3(x, res)[2]
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            up.mul(2)  # something to record
            race.race_add_norm_e4m3(x, res)
    del alive


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(race, cuda, grad):
    *args, _, _ = make(2, 2, 20, 32, 32, F32, seed=52)
    rows = [torch.randn(4, 64, device=cuda), torch.randn(4, 64, device=cuda), torch.randn(64, device=cuda)]
    for call, inputs in ((race.race_delta_rule_carry, args), (race.race_add_norm_e4m3, rows)):
        for i in range(len(inputs)):
            with torch.set_grad_enabled(grad), torch.autograd.forward_ad.dual_level():
                duals = [torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(inputs)]
                with pytest.raises(RuntimeError, match="jvp"):
                    call(*duals)
