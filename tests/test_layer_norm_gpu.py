"""Layer normalisation against its definition in 64 bits, element by element, within the bounds that ``layer_ref`` derives."""
import pytest
import torch

import layer_ref
from mamba2d_b200 import layer_norm

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16


def rand(*shape, seed=0, dt=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda().to(dt)


def check(x, weight, bias, residual, dy, ds, eps=1e-5):
    """Forward with and without gradients, the sum, and every gradient."""
    d = lambda t: None if t is None else t.detach().double()  # noqa: E731
    total = x.detach() if residual is None else x.detach() + residual.detach()
    t64, w64, b64 = (None if t is None else t.requires_grad_(True) for t in (d(total), d(weight), d(bias)))
    want = layer_ref.norm(t64, w64, b64, eps)
    leaves = [t for t in (t64, w64, b64) if t is not None]
    grads = list(torch.autograd.grad(want, leaves, dy.double()))
    if residual is not None:
        grads[0] = grads[0] + ds.double()
    with torch.no_grad():
        bounds = layer_ref.norm_bounds(t64, w64, b64, dy.double(), eps)
        got = layer_norm(x, weight, bias, residual=residual, eps=eps)
    if residual is not None:
        assert torch.equal(got[1], total)
        got = got[0]
    assert got.dtype == x.dtype and got.shape == x.shape
    assert layer_ref.within(got, want.detach(), bounds[0]) <= 1
    own = [None if t is None else t.detach().requires_grad_(True) for t in (x, weight, bias, residual)]
    out = layer_norm(own[0], own[1], own[2], residual=own[3], eps=eps)
    y = out if residual is None else out[0]
    assert torch.equal(y, got)
    mine = torch.autograd.grad(out, [t for t in own if t is not None], dy if residual is None else (dy, ds))
    if residual is not None:
        assert torch.equal(mine[0], mine[-1])
    want_by, bound_by = [grads[0]], [bounds[1] + (0 if residual is None else 2.0 ** -23 * ds.double().abs())]
    for t, b in ((w64, bounds[2]), (b64, bounds[3])):
        if t is not None:
            want_by.append(grads[len(want_by)])
            bound_by.append(b)
    for a, w, b in zip(mine, want_by, bound_by):
        assert layer_ref.within(a, w, b) <= 1
    return got, mine


SIZES = [(1, 1), (3, 2), (5, 3), (1, 7), (33, 8), (200, 16), (9, 31), (17, 64), (2, 100), (65, 128), (5, 129), (31, 130), (3, 255), (40, 256), (1000, 320), (7, 512), (13, 513), (3, 520),
         (5, 1000), (64, 1024), (2, 2047), (600, 2048), (3, 4096), (2, 4099), (5, 8192), (2, 8193), (3, 8200), (2, 16384), (2, 16392), (3, 20001)]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("N,C", SIZES)
@pytest.mark.parametrize("residual", [False, True])
def test_sizes(N, C, dt, residual):
    x, dy = rand(N, C, seed=1, dt=dt) * 3 + 1, rand(N, C, seed=2, dt=dt)
    check(x, 1 + 0.2 * rand(C, seed=3), rand(C, seed=4), rand(N, C, seed=5, dt=dt) if residual else None, dy, rand(N, C, seed=6, dt=dt))


@pytest.mark.parametrize("N,C", [(20000, 64), (50001, 40), (100352, 320), (3001, 1536), (4000, 33), (700, 5001)])
def test_many_rows(N, C):
    x, dy = rand(N, C, seed=1, dt=BF), rand(N, C, seed=2, dt=BF)
    check(x, 1 + 0.2 * rand(C, seed=3), rand(C, seed=4), None, dy, None)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("N,C", [(50, 320), (9, 1000), (4, 33), (2, 9001)])
def test_parameters(N, C, dt):
    """Neither, one of them, both of x's type, not dense, shared by all channels."""
    x, dy = rand(N, C, seed=1, dt=dt), rand(N, C, seed=2, dt=dt)
    table = (1 + 0.3 * rand(C, 2, seed=3)).to(dt)
    gain = torch.full((1,), 0.75, device="cuda", dtype=dt)
    for w, b in ((None, None), (table[:, 0].float(), None), (None, table[:, 1].float()), (table[:, 0].contiguous(), table[:, 1].contiguous()), (table[:, 0], table[:, 1]),
                 (gain.expand(C), table[:, 1])):
        check(x, w, b, None, dy, None)
    leaf, other = gain.clone().requires_grad_(True), gain.expand(C).contiguous().requires_grad_(True)
    one, = torch.autograd.grad(layer_norm(x, leaf.expand(C)), leaf, dy)
    full, = torch.autograd.grad(layer_norm(x, other), other, dy)
    assert one.shape == (1,) and abs(float(one) - float(full.double().sum())) <= 2.0 ** -7 * float(full.double().abs().sum())


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("C", [64, 320, 1000, 4096, 33])
def test_strides(C, dt):
    """Slices of a wider tensor, more dimensions, transposed ones, expanded rows, odd offsets: the bits of dense ones where the form is the same."""
    wide = rand(4, 6, 3 * C + 8, seed=1, dt=dt)
    w, b = 1 + 0.2 * rand(C, seed=3), rand(C, seed=4)
    x, r, dy = wide[..., :C], wide[..., C:2 * C], wide[..., 2 * C:3 * C]
    for t in (x, x.transpose(0, 1), wide[..., 1:C + 1], x[:, ::2], x[0], x[0, 0], x[:1].expand(4, 6, C), x.transpose(1, 2).contiguous().transpose(1, 2)):
        up = rand(*t.shape, seed=7, dt=dt)
        got, grads = check(t, w, b, None, up, None)
    check(x, w, b, r, dy, wide[..., 5:C + 5])
    one = wide[:1, :1, :C]
    leaf, full = one.detach().clone().requires_grad_(True), one.expand(4, 6, C).contiguous().requires_grad_(True)
    a, = torch.autograd.grad(layer_norm(leaf.expand(4, 6, C), w, b), leaf, dy)
    z, = torch.autograd.grad(layer_norm(full, w, b), full, dy)
    assert float((a.double() - z.double().sum((0, 1), keepdim=True)).abs().max()) <= 2.0 ** -6 * float(z.double().abs().sum((0, 1)).max())


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("C", [3, 64, 320, 1000, 1024, 4096, 20001])
def test_rows_of_one_value(C, dt):
    """The mean is that value and the result the bias, also where C is no power of two and the value far from zero."""
    x = torch.tensor([0.0, 1.1, -1234.56, 3e7, 1e-30], device="cuda").to(dt)[:, None].expand(5, C).contiguous()
    b = rand(C, seed=1)
    assert torch.equal(layer_norm(x, None, b), b.to(dt).expand(5, C))


@pytest.mark.parametrize("C", [64, 1000, 4096])
def test_rows_far_from_zero(C):
    """A deviation of one about 10000, fp32: x itself has 14 bits left, and they count."""
    x = 1e4 + rand(6, C, seed=1)
    check(x, None, None, None, rand(6, C, seed=2), None)
    x[:, 0] = -5e4                       # the value that the mean is taken about lies apart
    check(x, None, None, None, rand(6, C, seed=2), None)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("C", [64, 320, 1000, 4096, 33])
def test_what_is_not_finite_spoils_its_row_alone(C, dt):
    x, dy = rand(40, C, seed=1, dt=dt), rand(40, C, seed=2, dt=dt)
    clean = layer_norm(x)
    x[7, C // 2], x[20, 0], x[39, C - 1] = torch.nan, torch.inf, -torch.inf
    leaf = x.clone().requires_grad_(True)
    y = layer_norm(leaf)
    dx, = torch.autograd.grad(y, leaf, dy)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[7, 20, 39]] = True
    for t in (y, dx):
        assert torch.equal(torch.isnan(t).all(1), bad) and torch.equal(torch.isnan(t).any(1), bad)
    assert torch.equal(y[~bad], clean[~bad])


def test_outputs_that_are_not_used():
    x, r = (rand(10, 64, seed=i).requires_grad_(True) for i in (1, 2))
    w = (1 + 0.1 * rand(64, seed=3)).requires_grad_(True)
    dy = rand(10, 64, seed=4)
    y, s = layer_norm(x, w, residual=r)
    only = torch.autograd.grad(y, (x, r, w), dy, retain_graph=True)
    both = torch.autograd.grad((y, s), (x, r, w), (dy, torch.zeros_like(dy)), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(only, both))
    dx, dr, dw = torch.autograd.grad(s, (x, r, w), dy)
    assert torch.equal(dx, dy) and torch.equal(dr, dy) and bool((dw == 0).all())
    x, w = x.detach(), w.detach().requires_grad_(True)
    got, = torch.autograd.grad(layer_norm(x, w), w, dy)
    assert got.shape == (64,)


@pytest.mark.parametrize("C", [64, 1000, 33])
def test_gradients_against_differences(C):
    """Central differences along random directions, fp32, a step of 2^-5: the third derivative's share is some 1e-3 of the slope."""
    x, w, b, r, dy, ds = rand(8, C, seed=1), 1 + 0.2 * rand(C, seed=2), rand(C, seed=3), rand(8, C, seed=4), rand(8, C, seed=5), rand(8, C, seed=6)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    grads = torch.autograd.grad(layer_norm(*leaves[:3], residual=leaves[3]), leaves, (dy, ds))

    def f(x, w, b, r):
        y, s = layer_norm(x, w, b, residual=r)
        return (y.double() * dy.double()).sum() + (s.double() * ds.double()).sum()
    for i, t in enumerate((x, w, b, r)):
        way, step, args = rand(*t.shape, seed=10 + i), 2.0 ** -5, [x, w, b, r]
        up, down = [*args[:i], t + step * way, *args[i + 1:]], [*args[:i], t - step * way, *args[i + 1:]]
        slope, want = float((f(*up) - f(*down)) / (2 * step)), float((grads[i].double() * way.double()).sum())
        assert abs(slope - want) < 1e-2 * float((grads[i].double() * way.double()).norm())


def test_no_rows_and_no_gradients_of_gradients():
    assert layer_norm(torch.empty(0, 8, device="cuda")).shape == (0, 8)
    y, s = layer_norm(torch.empty(3, 0, device="cuda"), residual=torch.empty(3, 0, device="cuda"))
    assert y.shape == s.shape == (3, 0)
    x = rand(4, 64).requires_grad_(True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(layer_norm(x).sum(), x, create_graph=True)
