"""The distillation loss against its definition in 64 bits, within the bounds that ``layer_ref`` derives."""
import pytest
import torch

import layer_ref
from mamba2d_b200 import distillation_loss
from mamba2d_b200.refmodel import train_step

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16


def inputs(N, V, K, dt, seed=0, labels=True):
    g = torch.Generator().manual_seed(seed)
    z = (3 * torch.randn(N, V, generator=g)).cuda()
    t, index = (z + torch.randn(N, V, generator=g).cuda()).topk(K, -1)
    label = torch.randint(0, V, (N,), generator=g).cuda()
    return z.to(dt), t, index, label if labels else None, torch.randn(N, generator=g).cuda()


def check(z, t, index, labels, up, temperature=1.0, label_weight=0.0):
    """Forward with and without gradients, and the gradient."""
    kw = dict(temperature=temperature, label_weight=label_weight)
    z64 = z.detach().double().requires_grad_(True)
    want = layer_ref.distillation(z64, t, index, labels, **kw)
    grad, = torch.autograd.grad(want, z64, up.double())
    with torch.no_grad():
        bounds = layer_ref.distillation_bounds(z64, t, index, labels, temperature, label_weight, up.double())
        got = distillation_loss(z, t, index, labels, **kw)
    leaf = z.detach().requires_grad_(True)
    loss = distillation_loss(leaf, t, index, labels, **kw)
    assert got.dtype == F32 and torch.equal(loss, got)
    dz, = torch.autograd.grad(loss, leaf, up)
    assert layer_ref.within(got, want.detach(), bounds[0]) <= 1
    assert dz.dtype == z.dtype and layer_ref.within(dz, grad, bounds[1]) <= 1
    return got, dz


SIZES = [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 33, 8), (128, 1000, 16), (9, 1001, 5), (4, 2048, 512), (7, 4097, 33), (3, 8191, 64), (200, 9001, 10), (1, 50001, 100), (8, 131072, 64), (2, 131075, 512),
         (1, 300007, 1), (160, 32000, 20)]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("N,V,K", SIZES)
@pytest.mark.parametrize("temperature,label_weight", [(1.0, 0.0), (2.5, 0.0), (1.0, 0.3), (2.0, 0.5), (2.0, 1.0)])
def test_sizes(N, V, K, dt, temperature, label_weight):
    z, t, index, labels, up = inputs(N, V, K, dt, labels=label_weight > 0)
    check(z, t, index, labels, up, temperature, label_weight)


@pytest.mark.parametrize("V", [1000, 20001])
def test_types(V):
    """Teachers in bfloat16, indices and labels of 32 bits, a single row without a dimension for rows, more dimensions."""
    z, t, index, labels, up = inputs(6, V, 12, BF)
    want, dz = check(z, t.to(BF), index, labels, up, 2.0, 0.5)
    kw = dict(temperature=2.0, label_weight=0.5)
    assert torch.equal(distillation_loss(z, t.to(BF), index.int(), labels.int(), **kw), want)
    assert torch.equal(distillation_loss(z.view(2, 3, V), t.to(BF).view(2, 3, 12), index.view(2, 3, 12), labels.view(2, 3), **kw), want.view(2, 3))
    # (a single row may be read by more CTAs, in another order)
    one = distillation_loss(z[0], t.to(BF)[0], index[0], labels[0], **kw)
    assert one.shape == () and abs(float(one) / float(want[0]) - 1) < 1e-5
    assert distillation_loss(z[:0], t[:0], index[:0]).shape == (0,)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("V", [1000, 9000, 9001, 50001])
def test_strides(V, dt):
    """Rows that lie apart, begin at odd offsets, are one and the same; teachers in slices; an upstream gradient that all rows share."""
    z, t, index, labels, up = inputs(5, V, 9, dt, 1)
    kw = dict(temperature=2.0, label_weight=0.25)
    want, dz = check(z, t, index, labels, up, **kw)

    def same(z, t, index, labels, exact=True):
        leaf = z.detach().requires_grad_(True)
        loss = distillation_loss(leaf, t, index, labels, **kw)
        d, = torch.autograd.grad(loss, leaf, up)
        # (a head of another length gives other threads other values: the same within the bounds)
        bounds = layer_ref.distillation_bounds(z.detach().double(), t, index, labels, 2.0, 0.25, up.double())
        assert float(((loss - want).abs().double() / (2 * bounds[0] + 2.0 ** -24 * want.abs())).max()) <= 1
        assert float(((d.double() - dz.double()).abs() / (2 * bounds[1] + torch.finfo(dt).eps * dz.double().abs() + 1e-30)).max()) <= 1
    wide = torch.zeros(5, V + 11, device="cuda", dtype=dt)
    for o in (0, 1, 3, 8, 11):
        wide[:, o:o + V] = z
        same(wide[:, o:o + V], t, index, labels)
    same(z.t().contiguous().t(), t, index, labels)
    table = torch.cat((t, t), 1)[:, 9:]
    spread = torch.stack((index, index), -1)[..., 0]
    same(z, table, spread, torch.stack((labels, labels), 1)[:, 0])
    check(z[:1].expand(5, V), t[:1].expand(5, 9), index[:1].expand(5, 9), labels[:1].expand(5), up, **kw)
    leaf = z.detach().requires_grad_(True)
    a, = torch.autograd.grad(distillation_loss(leaf, t, index, labels, **kw).sum(), leaf)
    b, = torch.autograd.grad(distillation_loss(leaf, t, index, labels, **kw), leaf, torch.ones(5, device="cuda"))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("V", [50, 1000, 9001, 140000])
def test_entries_that_are_absent_or_twice(V, dt):
    z, t, index, labels, up = inputs(8, V, 12, dt, 2)
    index, t, labels = index.clone(), t.clone(), labels.clone()
    index[0, 4:] = -1                    # a shorter list
    index[1] = -1                        # none
    index[2, ::2] = V                    # beyond the classes
    t[3, 5] = -torch.inf
    t[4] = -torch.inf                    # nothing to learn
    index[5, :] = index[5, 0]            # all the same
    index[6, 7] = index[6, 3]
    labels[6], labels[0], labels[5] = index[6, 3], index[0, 2], index[5, 0]
    labels[1], labels[2], labels[7] = -100, V, V - 1
    index[7, 0], index[7, 1] = 0, V - 1
    for tau, w in ((1.0, 0.0), (2.0, 0.5), (1.0, 0.5), (2.0, 1.0)):
        got, dz = check(z, t, index, labels if w else None, up, tau, w)
        if not w:
            assert float(got[1]) == float(got[4]) == 0 and bool((dz[[1, 4]] == 0).all())
    assert float(got[1]) == 0 and bool((dz[1] == 0).all())
    # the order of a list does not matter beyond rounding, and the same call gives the same bits
    again, dz2 = check(z, t, index, labels, up, 2.0, 0.5)
    other, dz3 = check(z, t, index, labels, up, 2.0, 0.5)
    assert torch.equal(again, other) and torch.equal(dz2, dz3)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("V", [40, 1000, 9001, 140000])
def test_masked_classes(V, dt):
    """Classes masked with -inf or with the type's lowest value, rows with nothing else, rows of one value, large ones."""
    z, t, index, labels, up = inputs(7, V, 8, dt, 3)
    z = z.clone()
    rest = torch.ones(7, V, dtype=torch.bool, device="cuda").scatter_(1, index, False).scatter_(1, labels[:, None], False)
    z[0][rest[0]] = -torch.inf
    z[1][rest[1]] = torch.finfo(dt).min
    z[2] = torch.finfo(dt).min           # all masked: uniform
    z[3] = -7.25
    z[4] = torch.finfo(dt).max
    z[5] = z[5] * 1000
    got, dz = check(z, t, index, labels, up, 2.0, 0.5)
    assert bool(torch.isfinite(dz).all())
    # a class that the teacher wants and the student has masked costs an infinity, and its row alone is spoiled by a NaN or by -inf everywhere
    z[6, index[6, 0]] = -torch.inf
    z[3] = -torch.inf
    z[5, V // 2] = torch.nan
    leaf = z.clone().requires_grad_(True)
    loss = distillation_loss(leaf, t, index, labels, temperature=2.0, label_weight=0.5)
    d, = torch.autograd.grad(loss, leaf, up)
    assert float(loss[6]) == torch.inf and torch.equal(torch.isnan(loss).nonzero()[:, 0].cpu(), torch.tensor([3, 5]))
    assert torch.equal(torch.isnan(d).any(1).nonzero()[:, 0].cpu(), torch.tensor([3, 5]))
    for r in (0, 1, 2, 4):
        assert torch.equal(loss[r], got[r]) and torch.equal(d[r], dz[r])


def test_a_student_like_its_teacher_loses_nothing():
    """All classes given by the teacher: the loss of the same logits is zero and so is the gradient, to the bounds."""
    z = (3 * torch.randn(50, 200, generator=torch.Generator().manual_seed(5))).cuda()
    index = torch.stack([torch.randperm(200, generator=torch.Generator().manual_seed(i)) for i in range(50)]).cuda()
    check(z, z.gather(1, index), index, None, torch.ones(50, device="cuda"), 2.0, 0.0)


@pytest.mark.parametrize("V", [500, 12000])
def test_gradients_against_differences(V):
    """Central differences along random directions in fp32, a step of 2^-6: the third derivative's share is below 1e-3 of the slope."""
    z, t, index, labels, up = inputs(4, V, 10, F32, 6)
    kw = dict(temperature=2.0, label_weight=0.5)
    leaf = z.clone().requires_grad_(True)
    dz, = torch.autograd.grad(distillation_loss(leaf, t, index, labels, **kw), leaf, up)
    f = lambda z: float((distillation_loss(z, t, index, labels, **kw).double() * up.double()).sum())  # noqa: E731
    for seed in range(3):
        way = torch.randn(z.shape, generator=torch.Generator().manual_seed(seed)).cuda()
        slope, want = (f(z + 2.0 ** -6 * way) - f(z - 2.0 ** -6 * way)) * 2.0 ** 5, float((dz.double() * way.double()).sum())
        assert abs(slope - want) < 1e-2 * float((dz.double() * way.double()).norm())


@pytest.mark.parametrize("micro", [3, 8])
def test_a_training_step_with_a_teacher(micro):
    """``refmodel.train_step``: loss and gradients against autograd in 64 bits."""
    g = torch.Generator().manual_seed(7)
    images, labels = torch.randn(8, 30, generator=g).cuda(), torch.randint(0, 40, (8,), generator=g).cuda()
    top, index = torch.randn(8, 40, generator=g).cuda().topk(6, -1)
    for w in (0.0, 0.5):
        torch.manual_seed(1)
        model = torch.nn.Linear(30, 40).cuda()
        weight, bias = (p.detach().double().requires_grad_(True) for p in model.parameters())
        want = layer_ref.distillation(images.double() @ weight.t() + bias, top, index, labels, 2.0, w).mean()
        grads = torch.autograd.grad(want, (weight, bias))
        before = [p.detach().clone() for p in model.parameters()]
        loss = train_step(model, torch.optim.SGD(model.parameters(), lr=0.5), images, labels, micro, autocast_dtype=None, teacher=(top, index), temperature=2.0, label_weight=w)
        assert abs(float(loss) / float(want) - 1) < 1e-5
        for p, old, d in zip(model.parameters(), before, grads):
            assert float((p.detach().double() - (old.double() - 0.5 * d)).abs().max()) < 1e-5


def test_refusals_on_the_device():
    z, t, index, labels, up = inputs(3, 50, 4, F32)
    with pytest.raises(RuntimeError, match="no gradient"):
        distillation_loss(z, t.requires_grad_(True), index)
    with pytest.raises(RuntimeError):
        distillation_loss(z, t.detach(), index.cpu())
    leaf = z.requires_grad_(True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(distillation_loss(leaf, t.detach(), index).sum(), leaf, create_graph=True)
