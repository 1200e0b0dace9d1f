"""Group normalisation with an activation (mamba2d_b200.group_norm) against its definition in 64 bits.

Largest errors allowed, relative to the largest result: fp32, 2e-5 forward (statistics to some 2^-22, an activation to
5e-7, both times values of up to 6 deviations) and 1e-4 for gradients (sums of up to 1e5 terms); bf16, one rounding more:
2^-8 of the value.
"""
import pytest
import torch

import seq_ref
from mamba2d_b200 import group_norm

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def close(got, want, tol):
    assert got.shape == want.shape
    bound = tol * float(want.abs().max()) + (want.abs() * 2.0 ** -8 if got.dtype == BF else 0.0) + 1e-30
    worst = float(((got.detach().double() - want).abs() / bound).max())
    assert worst < 1, worst


SHAPES = [((1, 1), 1), ((3, 8), 8), ((2, 7, 5, 12), 3), ((5, 64), 4), ((1, 14, 14, 320), 32), ((4, 196, 96), 1), ((2, 56, 56, 64), 16), ((2049, 256), 2),
          ((3, 1023, 30), 5), ((2, 130, 131, 64), 32), ((1, 300, 300, 128), 8), ((300, 2048), 16), ((70, 4, 576), 9), ((2, 3, 1000), 1), ((40, 33, 192), 192)]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_norm(shape, groups, act, dt):
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    C = shape[-1]
    x = (n(*shape) * 2 + 3 * n(shape[0], *[1] * (len(shape) - 2), C)).to(dt)
    params = (n(C) * 0.3 + 1, n(C) * 0.3)
    for weight, bias in (params, (None, None), (params[0].to(dt), None)):
        leaves = [t.clone().requires_grad_(True) for t in (x, weight, bias) if t is not None]
        it = iter(leaves)
        call = [next(it) if t is not None else None for t in (x, weight, bias)]
        dy = n(*shape).to(dt)
        y = group_norm(call[0], groups, call[1], call[2], eps=1e-3, act=act)
        got = torch.autograd.grad(y, leaves, dy)
        ref = [t.detach().double().requires_grad_(True) if t is not None else None for t in call]
        want = seq_ref.norm(ref[0], groups, ref[1], ref[2], 1e-3, act)
        grads = torch.autograd.grad(want, [t for t in ref if t is not None], dy.double())
        close(y, want.detach(), 2e-5)
        for a, b in zip(got, grads):
            close(a, b, 1e-4)
        with torch.no_grad():
            assert torch.equal(y, group_norm(call[0], groups, call[1], call[2], eps=1e-3, act=act))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("shape,groups", [((2, 1000, 64), 16), ((1000, 256), 4), ((1, 40000, 32), 2)])
def test_large_mean_and_constant_groups(shape, groups, dt):
    """The variance of values far from zero, and a group whose values are all the same: zero, then bias alone."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn(shape, generator=g, device="cuda") + 1000.0).to(dt)
    x[0, ..., :shape[-1] // groups] = 512.0
    w, b = torch.full((shape[-1],), 0.5, device="cuda"), torch.full((shape[-1],), 0.25, device="cuda")
    y = group_norm(x, groups, w, b)
    want = seq_ref.norm(x.double(), groups, w.double(), b.double(), 1e-5, None)
    assert bool((y[0, ..., :shape[-1] // groups] == 0.25).all())
    # the mean is off by up to 2^-24 of 1000, against a deviation of one
    bound = 4e-4 + (want.abs() * 2.0 ** -8 if dt == BF else 0.0)
    assert bool(((y.double() - want).abs() < bound).all())


def test_infinities_stay_in_their_group():
    x = torch.randn(3, 50, 64, device="cuda")
    want = group_norm(x, 4, act="silu")
    x[1, 7, 20] = float("inf")
    x[2, 3, 40] = float("nan")
    y = group_norm(x, 4, act="silu")
    bad = torch.zeros(3, 50, 64, dtype=torch.bool, device="cuda")
    bad[1, :, 16:32] = True
    bad[2, :, 32:48] = True
    assert torch.equal(y[~bad], want[~bad]) and bool(torch.isnan(y[2, :, 32:48]).all())


@pytest.mark.parametrize("act,far", [("silu", 200.0), ("gelu", 60.0)])
def test_activation_far_from_zero(act, far):
    """Arguments of +-far: the value is the argument or zero, its slope one or zero."""
    x = torch.randn(4, 100, 32, device="cuda", requires_grad=True)
    b = torch.tensor([far, -far], device="cuda").repeat(16)
    y = group_norm(x, 1, None, b, act=act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    h = seq_ref.norm(x.detach().double(), 1, None, None, 1e-5, None)
    up, down = (y[..., 0::2].detach().double() - h[..., 0::2] - far).abs().max(), y[..., 1::2].detach().abs().max()
    # the GELU takes erfc at 6 for all that lies beyond: 6 / sqrt 2 * erfc(6) = 4.24 * 2.2e-17 = 1e-16, which stands for zero
    assert float(up) < 1e-4 and float(down) < 1e-15
    ref = x.detach().double().requires_grad_(True)
    want, = torch.autograd.grad(seq_ref.norm(ref, 1, None, b.double(), 1e-5, act), ref, torch.ones_like(ref))
    assert float((dx.double() - want).abs().max()) < 1e-5


def test_layouts_offsets_and_captured_graphs():
    """An image batch in PyTorch's channels_last memory, tensors that start at any element, and a replayed graph with a
    backward pass."""
    img = torch.randn(2, 48, 9, 11, device="cuda").to(memory_format=torch.channels_last)
    y = group_norm(img.permute(0, 2, 3, 1), 6, act="gelu").permute(0, 3, 1, 2)
    want = torch.nn.functional.gelu(torch.nn.functional.group_norm(img, 6))
    assert float((y - want).abs().max()) < 1e-5
    for shape, groups in (((3, 77, 64), 8), ((100, 256), 2)):
        for dt in (F32, BF):
            n = 1
            for s in shape:
                n *= s
            x = torch.randn(n + 1, device="cuda").to(dt)[1:].view(shape)
            assert not x.is_contiguous() or x.data_ptr() % 16
            a, b = group_norm(x, groups, act="silu"), group_norm(x.clone(), groups, act="silu")
            assert float((a.float() - b.float()).abs().max()) < (1e-5 if dt == F32 else 0.05)
    x = torch.randn(4, 500, 64, device="cuda")
    w, b = torch.randn(64, device="cuda"), torch.randn(64, device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    dy = torch.randn_like(x)

    def call():
        y = group_norm(leaves[0], 8, leaves[1], leaves[2], act="gelu")
        return (y, *torch.autograd.grad(y, leaves, dy))
    want = [t.detach().clone() for t in call()]          # (no eager graph of the leaves may live while one is captured)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
