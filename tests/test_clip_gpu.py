"""Clipping by the global norm (mamba2d_b200.clip_norm_, clip_grad_norm_) against 64 bits.  The norm may be off by 1e-6
(squares are summed in fp32 over at most 64 values, then in fp64), a scaled fp32 value by 2^-22 of itself, a
bf16 value by half a step."""
import pytest
import torch

from mamba2d_b200 import clip_grad_norm_, clip_norm_

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def make(sizes, dt, seed=0, gap=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    flat = torch.randn(sum(sizes) + gap * len(sizes) + 8, generator=g, device="cuda").to(dt)
    out, at = [], gap
    for n in sizes:
        out.append(flat[at:at + n])
        at += n + gap
    return flat, out


def check(tensors, max_norm):
    before = [t.double().clone() for t in tensors]
    want = torch.sqrt(sum((t * t).sum() for t in before))
    norm = clip_norm_(tensors, max_norm)
    assert norm.dtype == F32 and norm.shape == () and abs(float(norm) / float(want) - 1) < 1e-6
    f = min(1.0, max_norm / (float(want) + 1e-6))
    for t, b in zip(tensors, before):
        if f == 1.0:
            assert torch.equal(t.double(), b)
        else:
            assert bool(((t.double() - b * f).abs() <= (b * f).abs() * (1e-6 + (2.0 ** -8 if t.dtype == BF else 2.0 ** -22))).all())
    return norm


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("sizes", [[1], [3, 1, 2], [7, 64, 1023, 5], [8192], [8193, 16384, 16385], [100003, 1, 77], [1 << 20, 3, 1 << 18], list(range(1, 130))])
def test_clip(sizes, dt):
    for gap in (0, 1, 5):
        flat, tensors = make(sizes, dt, gap=gap)
        keep = flat.clone()
        check(tensors, 0.37 * sum(sizes) ** 0.5)
        for t in tensors:
            t.zero_()
        rest = flat != 0                                   # what lies between and behind was not touched
        assert torch.equal(flat[rest], keep[rest])
        check(make(sizes, dt, gap=gap)[1], 1e9)


def test_many_tensors_of_both_types():
    """More than one launch's table."""
    _, a = make([17 + i % 91 for i in range(700)], F32)
    _, b = make([300 + i % 13 for i in range(600)], BF, seed=1)
    mixed = [t for pair in zip(a, b) for t in pair] + a[600:]
    check(mixed, 3.0)
    assert abs(float(clip_norm_(mixed, float("inf"))) - 3.0) < 1e-2


def test_norms_of_zero_and_norms_that_are_not_finite():
    t = [torch.zeros(1000, device="cuda"), torch.zeros(0, device="cuda")]
    assert float(clip_norm_(t, 1.0)) == 0.0 and not t[0].any()
    assert float(clip_norm_([t[1]], 1.0)) == 0.0
    _, g = make([1000, 50], F32)
    check(g, 0.0)
    for bad in (float("inf"), float("nan")):
        _, g = make([1000, 50], F32)
        g[0][17] = bad
        keep = [x.clone() for x in g]
        with pytest.raises(RuntimeError):
            clip_norm_(g, 1.0, error_if_nonfinite=True)
        assert all(torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0)) for x, y in zip(g, keep))
        want = [x.clone() for x in g]
        p = [torch.nn.Parameter(torch.zeros_like(x)) for x in want]
        for x, y in zip(p, want):
            x.grad = y
        torch.nn.utils.clip_grad_norm_(p, 1.0)
        clip_norm_(g, 1.0)
        assert all(torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0)) for x, y in zip(g, want))


def test_gradients_of_parameters_and_layouts():
    model = torch.nn.Sequential(torch.nn.Conv2d(3, 16, 3), torch.nn.Conv2d(16, 8, 3), torch.nn.Flatten(), torch.nn.Linear(512, 10)).cuda().to(memory_format=torch.channels_last)
    model(torch.randn(4, 3, 12, 12, device="cuda").to(memory_format=torch.channels_last)).square().sum().backward()
    model[1].bias.requires_grad_(False)
    model[1].bias.grad = None
    frozen = model[1].bias.clone()
    want = [p.grad.clone() for p in model.parameters() if p.grad is not None]
    total = torch.sqrt(sum(g.double().square().sum() for g in want))
    version = model[0].weight.grad._version
    norm = clip_grad_norm_(model.parameters(), 0.1)
    assert abs(float(norm / total) - 1) < 1e-6 and model[0].weight.grad._version > version and torch.equal(frozen, model[1].bias)
    for g, w in zip([p.grad for p in model.parameters() if p.grad is not None], want):
        assert g.stride() == w.stride() and float((g - w * (0.1 / float(total))).abs().max()) < 1e-6
    assert float(clip_grad_norm_([], 1.0)) == 0.0 and float(clip_grad_norm_(model[1].bias, 1.0)) == 0.0


def test_refusals():
    x = torch.randn(100, device="cuda")
    for bad in ([x, x], [x[:60], x[50:]], [x[::2]], [x.expand(3, 100)], [x.cpu()], [x.half()], [x, torch.randn(3)]):
        keep = x.clone()
        with pytest.raises(RuntimeError):
            clip_norm_(bad, 0.1)
        assert torch.equal(x, keep)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            clip_norm_([x], bad)


def test_captured_and_repeated():
    _, a = make([5000, 33], F32)
    keep = [t.clone() for t in a]
    want = [t.clone() for t in a]
    norm = clip_norm_(want, 2.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = clip_norm_(a, 2.0)
    for _ in range(3):
        for t, k in zip(a, keep):
            t.copy_(k)
        graph.replay()
        assert torch.equal(out, norm) and all(torch.equal(x, y) for x, y in zip(a, want))
