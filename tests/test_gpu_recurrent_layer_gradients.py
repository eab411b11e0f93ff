"""The gradient of every leaf of the recurrent layer against the plain layer's in 64 bits.

A gradient goes through the layer's six operators twice, values on the way there and gradients on
the way back, each with the rounding of test_gpu_recurrent_layer.TOL: twice that, of a leaf's
gradient in 2-norm.  test_layer_reference.py holds what is seen at that size."""
from __future__ import annotations

import pytest
import torch

import layer_reference
from gpu_util import say
from test_gpu_recurrent_layer import H, Hk, TOL, Layer, _inputs

pytestmark = pytest.mark.gpu


def test_every_leafs_gradient(race, cuda):
    module = Layer(race, cuda)
    x, residual, state, up = _inputs(cuda)
    leaves = dict(x=x, residual=residual, state=state, **dict(module.named_parameters()))
    leaves = {n: t.requires_grad_(True) for n, t in leaves.items()}
    down = torch.randn(state.shape, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda)
    y, r, s = module(x, residual, state)
    grads = torch.autograd.grad((y, r, s), list(leaves.values()), (up, up, down))
    wide = {n: t.detach().double().requires_grad_(True) for n, t in leaves.items()}
    want = layer_reference.layer(wide, module.unit.double(), module.freq.double(), H, Hk)
    for a, b in zip((y, r, s), want):
        assert (a.double() - b).norm() <= TOL * b.norm()
    exact = torch.autograd.grad(want, list(wide.values()), (up.double(), up.double(), down.double()))
    for name, a, b in zip(leaves, grads, exact):
        err = float((a.double() - b).norm() / b.norm())
        say(name, f"{err:.1e} of {2 * TOL:.1e}")
        assert err <= 2 * TOL, name
