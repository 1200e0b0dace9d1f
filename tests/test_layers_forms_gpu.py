"""Shapes that between them reach every form that a call of the gated recurrence or of the distillation loss can take on a GPU of 148 SMs, against definitions in 64 bits."""
import pytest
import torch

import layer_ref
import test_distillation_gpu
from mamba2d_b200 import gated_recurrence
from test_recurrence_gpu import fast_scan, inputs

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16


def check(x, g, s, dy, ds, form, lengths):
    """``test_recurrence_gpu.test_long_sequences``' comparison, with NaN behind the lengths."""
    T = x.shape[1]
    live = (torch.arange(T, device="cuda") < lengths[:, None])[..., None]
    a, u = layer_ref.terms(x.double(), g.double(), form)
    a, u, up, x64 = torch.where(live, a, 1.0), torch.where(live, u, 0.0), torch.where(live, dy.double(), 0.0), torch.where(live, x.double(), 0.0)
    first = lambda u, s: torch.cat((u[:, :1] + a[:, :1] * s[:, None], u[:, 1:]), 1)  # noqa: E731
    ahead = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), 1).flip(1)
    back = lambda up, s: fast_scan(ahead, torch.cat((up[:, :-1], up[:, -1:] + s[:, None]), 1).flip(1)).flip(1)  # noqa: E731
    bound = lambda a, H: 2.0 ** -17 * H + 1.25 * 2.0 ** -24 * fast_scan(a, H)  # noqa: E731
    prior = lambda h, s: torch.cat((s[:, None], h[:, :-1]), 1)  # noqa: E731
    h, D = fast_scan(a, first(u, s.double())), back(up, ds.double())
    H, E = fast_scan(a, first(u.abs(), s.double().abs())), back(up.abs(), ds.double().abs())
    dh, dD = bound(a, H), bound(ahead, E.flip(1)).flip(1)
    x, g, dy = (torch.where(live, t, torch.full((), torch.nan, dtype=t.dtype, device="cuda")) for t in (x, g, dy))
    leaves = [t.detach().requires_grad_(True) for t in (x, g, s)]
    out = gated_recurrence(leaves[0], leaves[1], form=form, initial_state=leaves[2], lengths=lengths, return_state=True)
    grads = torch.autograd.grad(out, leaves, (dy, ds))
    where = lambda t: torch.where(live, t, 0.0)  # noqa: E731
    assert layer_ref.within(out[0].detach(), where(h), dh) <= 1
    assert layer_ref.within(out[1].detach(), h[:, -1], dh[:, -1]) <= 1
    before, off, size = prior(h, s.double()), prior(dh, torch.zeros_like(s.double())), prior(H, s.double().abs())
    if form == "decay":
        dx, dg, bx, bg = D, a * D * before, dD, a * (dD * size + E * off)
    else:
        rest = torch.where(live, torch.sigmoid(-g.double()), 0.0)
        dx, dg, bx, bg = rest * D, a * rest * D * (before - x64), rest * dD, a * rest * (dD * (size + x64.abs()) + E * off)
    assert layer_ref.within(grads[0], where(dx), bx + 2.0 ** -19 * E) <= 1
    assert layer_ref.within(grads[1], where(dg), bg + 2.0 ** -19 * a * E * (size + x64.abs())) <= 1
    assert layer_ref.within(grads[2], a[:, 0] * D[:, 0], a[:, 0] * (dD[:, 0] + 2.0 ** -19 * E[:, 0])) <= 1


# Lanes of 8, 16 and 32 channels or pairs, by TMA or by plain loads, one CTA a sequence or clusters, one stride of tokens or several: forward, backward, both types.
SHAPES = [(6, 1395, 192), (4, 1225, 512), (15, 562, 128), (24, 319, 64), (44, 3000, 96), (25, 2889, 130), (41, 273, 2), (338, 141, 20), (18, 2164, 18), (330, 68, 1), (322, 265, 8),
          (10, 4319, 24), (49, 139, 2), (204, 65, 34), (22, 1095, 18), (96, 138, 1), (9, 1093, 52), (305, 38, 2), (379, 42, 20), (431, 66, 18), (1, 3192, 2), (45, 141, 4), (51, 274, 40),
          (119, 64, 44)]


@pytest.mark.parametrize("form", ["decay", "forget"])
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,T,C", SHAPES)
def test_forms_of_the_recurrence(B, T, C, dt, form):
    x, g, s, dy, ds = inputs(B, T, C, dt, form, 12, True)
    check(x, g, s, dy, ds, form, torch.full((B,), T, device="cuda"))
    lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(13)).cuda()
    lengths[0] = T - 1
    check(x, g, s, dy, ds, form, lengths)


@pytest.mark.parametrize("temperature,label_weight", [(1.0, 0.0), (2.5, 0.0), (1.0, 0.3), (2.0, 0.5), (2.5, 0.5)])
@pytest.mark.parametrize("N,V,K,dt", [(3600, 7553, 20, BF), (3601, 4099, 12, F32), (3600, 16384, 5, BF), (3600, 2050, 8, F32)])
def test_many_rows_of_the_distillation_loss(N, V, K, dt, temperature, label_weight):
    """Rows of 8 to 32 KB: a warp for each where they are many (3552 on 148 SMs), else shared by CTAs, for the same rows."""
    z, t, index, labels, up = test_distillation_gpu.inputs(N, V, K, dt, 14, label_weight > 0)
    index = index.clone()
    index[5, 1:], index[7], index[9, 1] = -1, -1, index[9, 0]
    if labels is not None:
        labels[11], labels[12] = -100, index[12, 0]
    for n in (N, 3500):
        test_distillation_gpu.check(z[:n], t[:n], index[:n], None if labels is None else labels[:n], up[:n], temperature, label_weight)
