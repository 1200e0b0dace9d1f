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


# a row a token, clusters, pieces, any shape (rows that are not whole 16-byte pieces)
KINDS = [((300, 256), 4), ((5, 131, 64), 8), ((40, 3136, 64), 16), ((3, 50, 30), 5)]


def dense_and_not(C, dt):
    """(weight, bias) pairs: every second value of a table, one value for all channels, neither."""
    table, gain = (torch.randn(C, 2, device="cuda") * 0.5 + 1).to(dt), torch.full((1,), 0.75, device="cuda", dtype=dt)
    return [(table[:, 0], table[:, 1]), (gain.expand(C), None), (gain.expand(C), table[:, 1]), (table[:, 0], gain.expand(C)), (None, table[:, 1]), (table[:, 0], None)]


@pytest.mark.parametrize("dt,params", [(F32, F32), (BF, F32), (BF, BF)])
@pytest.mark.parametrize("shape,groups", KINDS)
def test_parameters_that_are_not_dense(shape, groups, dt, params):
    """Their gradients are those of dense ones, whichever of the two is wanted."""
    x, dy = torch.randn(shape, device="cuda").to(dt), torch.randn(shape, device="cuda").to(dt)
    for pair in dense_and_not(shape[-1], params):
        for wanted in ((True, True), (True, False), (False, True)):
            if not any(w and t is not None for w, t in zip(wanted, pair)):
                continue

            def call(tensors):
                y = group_norm(x, groups, *tensors, act="silu")
                return torch.autograd.grad(y, [t for t in tensors if t is not None and t.requires_grad], dy, allow_unused=True)
            strided = [t.detach().requires_grad_(w) if t is not None else None for t, w in zip(pair, wanted)]
            dense = [t.detach().contiguous().requires_grad_(w) if t is not None else None for t, w in zip(pair, wanted)]
            assert not all(t.is_contiguous() for t in strided if t is not None)
            got, want = call(strided), call(dense)
            assert len(got) == len(want)
            for a, b in zip(got, want):
                assert a is not None and torch.equal(a, b)


def test_a_gain_that_all_channels_share_gets_its_gradient():
    x = torch.randn(6, 50, 32, device="cuda")
    gain, table = torch.tensor([0.75], device="cuda", requires_grad=True), torch.randn(32, 2, device="cuda", requires_grad=True)
    y = group_norm(x, 4, gain.expand(32), table[:, 1])
    y.square().sum().backward()
    g, t = gain.detach().double().requires_grad_(True), table.detach().double().requires_grad_(True)
    seq_ref.norm(x.double(), 4, g.expand(32), t[:, 1], 1e-5, None).square().sum().backward()
    close(gain.grad, g.grad, 1e-4)
    close(table.grad, t.grad, 1e-4)


@pytest.mark.parametrize("shape,groups,dt", [(s, g, dt) for s, g in (((1, 128, 64), 8), ((9, 300, 96), 32), ((200, 49, 64), 1), ((40, 3136, 64), 16), ((1, 700, 700, 16), 2))
                                             for dt in (F32, BF)] + [((1, 700, 700, 12), 3, F32)])
def test_images_of_one_value(shape, groups, dt):
    """Every value the same, and no power of two: the mean is that value and the result the bias, whatever the number of
    threads, CTAs and pieces that took part in the sum."""
    w, b = torch.full((shape[-1],), 0.5, device="cuda"), torch.full((shape[-1],), 0.25, device="cuda")
    for value in (1000.3, -0.7, 3e-5):
        x = torch.full(shape, value, device="cuda").to(dt)
        assert bool((group_norm(x, groups, w, b) == 0.25).all()), value


# rows that are not whole 16-byte pieces, images of many channels, a tensor that starts at an odd element
ANY = [((1, 700, 700, 12), 3, 0), ((2, 40000, 30), 5, 0), ((3, 30000, 2), 1, 0), ((1, 300, 300, 64), 2, 1), ((1, 3000, 2056), 1, 0)]


def odd_start(x, offset):
    if not offset:
        return x
    flat = torch.empty(x.numel() + offset, dtype=x.dtype, device=x.device)
    flat[offset:] = x.view(-1)
    return flat[offset:].view(x.shape)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("shape,groups,offset", ANY)
def test_large_mean_and_constant_groups_of_any_shape(shape, groups, offset, dt):
    """As ``test_large_mean_and_constant_groups``, by the kernel for any shape."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn(shape, generator=g, device="cuda") + 1000.0).to(dt)
    constant = torch.full(shape, 1000.3, device="cuda").to(dt)
    w, b = torch.full((shape[-1],), 0.5, device="cuda"), torch.full((shape[-1],), 0.25, device="cuda")
    assert bool((group_norm(odd_start(constant, offset), groups, w, b) == 0.25).all())
    y = group_norm(odd_start(x, offset), groups, w, b)
    want = seq_ref.norm(x.double(), groups, w.double(), b.double(), 1e-5, None)
    # the mean is off by up to 2^-24 of 1000, against a deviation of one
    bound = 4e-4 + (want.abs() * 2.0 ** -8 if dt == BF else 0.0)
    assert bool(((y.double() - want).abs() < bound).all())


@pytest.mark.parametrize("shape,groups,offset", ANY)
def test_gradients_that_cancel_in_any_shape(shape, groups, offset):
    """The same dy everywhere: dx is zero, db the number of values.  What is left of dx is h times the mean of dh h, whose
    terms are off by half a step of theirs: 2^-24 times a mean |h| of 0.8, times |h| < 6, below 3e-7; as much again where the
    mean of x lies half a step off."""
    x = odd_start(torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda"), offset).requires_grad_(True)
    b = torch.zeros(shape[-1], device="cuda", requires_grad=True)
    y = group_norm(x, groups, None, b)
    dx, db = torch.autograd.grad(y, (x, b), torch.full_like(y, 1.0003))
    assert float(dx.abs().max()) < 1e-6
    want = 1.0003 * (x.numel() / shape[-1])
    assert float((db.double() / want - 1).abs().max()) < 1e-6


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("shape,groups", KINDS)
def test_activation_at_infinity(shape, groups, act, dt):
    """At +inf it is +inf and its slope one, at -inf both are zero: the gradients are those of biases that are merely
    large.  A NaN stays one."""
    x, dy = torch.randn(shape, device="cuda").to(dt), torch.randn(shape, device="cuda").to(dt)
    C = shape[-1]
    b = torch.randn(C, device="cuda")
    far = b.clone()
    b[3], b[5], far[3], far[5] = float("inf"), -float("inf"), 1e6, -1e6
    results = []
    for bias in (b, far):
        leaves = [x.clone().requires_grad_(True), bias.clone().requires_grad_(True)]
        y = group_norm(leaves[0], groups, None, leaves[1], act=act)
        results.append((y.detach(), *torch.autograd.grad(y, leaves, dy)))
    (y, dx, db), (y_far, dx_far, db_far) = results
    assert bool((y[..., 3] == float("inf")).all()) and not y[..., 5].any()
    assert torch.equal(dx, dx_far) and torch.equal(db, db_far) and bool(torch.isfinite(dx).all())
    keep = [c for c in range(C) if c not in (3, 5)]
    assert torch.equal(y[..., keep], y_far[..., keep])
    w = torch.ones(C, device="cuda")
    w[7] = 3e38                                               # h w beyond the largest float
    y = group_norm(x, groups, w, act=act)
    assert not bool(torch.isnan(y).any()) and bool((y[..., 7] == float("inf")).any())
    b[4] = float("nan")
    leaf = x.clone().requires_grad_(True)
    y = group_norm(leaf, groups, None, b, act=act)
    assert bool(torch.isnan(y[..., 4]).all()) and not bool(torch.isnan(y[..., 3]).any())
    dx, = torch.autograd.grad(y, leaf, dy)
    assert bool(torch.isnan(dx[..., 4]).all())


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("per", [8, 24, 40, 48, 56, 72, 80, 104, 112, 120, 128])
def test_rows_of_one_value(per, dt):
    """As ``test_images_of_one_value``, a group a token: sizes that are a power of two and sizes that are none."""
    C = 4 * per
    w, b = torch.full((C,), 0.5, device="cuda"), torch.full((C,), 0.25, device="cuda")
    for value in (1000.3, -0.7, 3e-5, 12345.67):
        assert bool((group_norm(torch.full((64, C), value, device="cuda").to(dt), 4, w, b) == 0.25).all()), value
