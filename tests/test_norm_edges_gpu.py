"""Calls of the group normalisation that its documentation allows and its own tests do not make.  Tolerances are those of
its own tests (``test_norm_gpu.close``) where nothing else is said."""
import pytest
import torch

import seq_ref
from test_norm_gpu import BF, F32, close
from mamba2d_b200 import group_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("shape,groups", [((1, 128, 64), 8), ((5, 131, 32), 4), ((9, 256, 96), 32)])
def test_clusters_that_begin_at_different_times(shape, groups, dt):
    """Slices of some 16 rows, whose CTAs send their sums to one another as soon as they have begun, launched behind one
    another so that they begin while others end: the same bits every time."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(shape, generator=g, device="cuda").to(dt) for _ in range(2))
    leaf = x.clone().requires_grad_(True)
    ref = x.double().requires_grad_(True)
    want = seq_ref.norm(ref, groups, None, None, 1e-5, "silu")
    grad, = torch.autograd.grad(want, ref, dy.double())
    ys, dxs = [], []
    for _ in range(200):
        ys.append(group_norm(leaf, groups, act="silu"))
        dxs.extend(torch.autograd.grad(ys[-1], leaf, dy))
    close(ys[0], want.detach(), 2e-5)
    close(dxs[0], grad, 1e-4)
    assert all(torch.equal(ys[0], y) for y in ys) and all(torch.equal(dxs[0], d) for d in dxs)
