"""Gradients of the linear attention by the form that takes the call: with bf16 tensors q's and k's come from the tcgen05
form only where the decay's is not wanted, so every condition is tested without it too.  Shares of the sum of magnitudes are
those of test_attention_gpu.py: bf16 tensors 2^-7 where a pair's weight or a state is rounded on the way, 2^-16 for the
state's gradient; the decay's gradient, all of whose products are split, has fp32 tensors' 2^-18 with bf16 tensors too
(operands in bf16 are exact in one part, so that fewer products are left out than with fp32 tensors)."""
import pytest
import torch

import seq_ref
from test_attention_gpu import BF, F32, decay_magnitude, make, rounding, share
from mamba2d_b200 import linear_attention

pytestmark = pytest.mark.gpu


def gradients(q, k, v, d, s, lengths, with_state, decay):
    """Of q, k, v, the state, and the decay where ``decay``: checked, and returned in this order."""
    scale = q.shape[-1] ** -0.5
    g = torch.Generator(device="cuda").manual_seed(5)
    d_o = torch.randn(v.shape, generator=g, device="cuda").to(v.dtype)
    d_state = torch.randn(v.shape[0], v.shape[2], q.shape[-1], v.shape[-1], generator=g, device="cuda") if with_state else None
    _, _, want = seq_ref.attention_grads(q, k, v, d, scale, s, lengths, d_o, d_state)
    ab = lambda t: None if t is None else t.abs()  # noqa: E731
    _, _, mag = seq_ref.attention_grads(q.abs(), k.abs(), v.abs(), d, scale, ab(s), lengths, d_o.abs(), ab(d_state))
    if lengths is not None:                                       # rows behind the end may hold anything
        behind = torch.arange(v.shape[1], device="cuda") >= lengths[:, None]
        q, k, v, d_o = (t.masked_fill(behind[..., None, None], float("nan")) for t in (q, k, v, d_o))
        d = d.masked_fill(behind[..., None], float("nan")) if d.dim() == 3 else d
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (q, k, v, s)]
    dd = d.clone().requires_grad_(decay)
    out = linear_attention(*leaves[:3], dd, initial_state=leaves[3], lengths=lengths, return_state=with_state)
    wanted = [t for t in (*leaves, dd) if t is not None and t.requires_grad]
    got = torch.autograd.grad(out, wanted, (d_o, d_state) if with_state else d_o)
    it = iter(got)
    for i, name in ((0, "q"), (1, "k"), (2, "v"), (4, "state"), (3, "decay")):
        if (name == "state" and s is None) or (name == "decay" and not decay):
            continue
        x, m, r = next(it), mag[i], share(v.dtype, i < 3)
        if name == "decay":
            m, r = decay_magnitude(*(torch.nan_to_num(t) for t in (q, k, v)), mag), 2.0 ** -18
            m = m.sum((0, 1)) if want[i].dim() == 1 else m
        ratio = seq_ref.within(x, want[i], m, r, rounding(x))
        assert ratio < 1, (name, ratio)
    if lengths is not None:
        assert not any(x[behind].any() for x in got[:3])
    return got


# one chunk and a row, two segments, three or four (the kernels join them), five (a launch does); heads of both sizes, shared or not
SHAPES = [(2, 129, 2, 2, 64, 64), (3, 1100, 2, 1, 128, 64), (2, 1100, 2, 2, 128, 128), (4, 1500, 1, 1, 64, 128), (3, 2100, 4, 2, 96, 40), (2, 2561, 2, 1, 64, 64), (1, 2100, 3, 3, 48, 128)]


@pytest.mark.parametrize("decay", [False, True])
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,T,H,G,K,V", SHAPES)
def test_lengths_and_the_states_gradient(B, T, H, G, K, V, dt, decay):
    args = make(B, T, H, G, K, V, dt, state=True, ragged=True)
    gradients(*args, True, decay)
    gradients(*args[:5], torch.tensor([T, 0, 1, 513][:B], dtype=torch.int32, device="cuda"), True, decay)
    gradients(*args[:4], None, args[5], False, decay)


@pytest.mark.parametrize("decay", [False, True])
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,T,H,G,K,V", SHAPES)
def test_steep_decays_and_minus_infinity(B, T, H, G, K, V, dt, decay):
    """Chunks that forget more than a factor can hold (tcgen05: weights from differences, not factors), alone and next to
    ordinary ones, and sequences that begin anew inside."""
    q, k, v, d, s, lengths = make(B, T, H, G, K, V, dt, state=True, ragged=B > 1)
    d[:, :, 0] -= 1.5
    d[0, 40:60] = -30.0
    if T > 1000:
        d[0, 700:900] = 0.0
        d[-1, 999] = -200.0
    gradients(q, k, v, d, s, None, True, decay)
    if not decay:                                             # (a sum of 512 dots has no place for the -inf's own gradient of zero)
        d[0, 50], d[0, 51], d[-1, 100, 0], d[-1, T - 1] = (-float("inf"),) * 4
    gradients(q, k, v, d, s, lengths, True, decay)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("decay", [False, True])
def test_fixed_decays(dt, decay):
    for B, T, H, G, K, V in SHAPES[:4]:
        gradients(*make(B, T, H, G, K, V, dt, decay="head", state=True, ragged=True), True, decay)


def test_the_same_bits_every_time():
    for decay in (False, True):
        args = make(3, 2100, 4, 2, 128, 64, BF, state=True, ragged=True)
        a, b = gradients(*args, True, decay), gradients(*args, True, decay)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dt", [F32, BF])
def test_gradient_of_the_decay_against_differences(dt):
    """Central differences of a sum over the outputs from the 64-bit definition, at fp32 tensors' share."""
    q, k, v, d, s, _ = make(1, 90, 2, 1, 32, 32, dt, state=True)
    g = torch.Generator(device="cuda").manual_seed(11)
    w, direction = torch.randn(v.shape, generator=g, device="cuda").to(dt), torch.randn(d.shape, generator=g, device="cuda")
    dd = d.clone().requires_grad_(True)
    slope = float((torch.autograd.grad(linear_attention(q, k, v, dd, initial_state=s), dd, w)[0].double() * direction).sum())
    f = lambda e: float((seq_ref.attention(q.double(), k.double(), v.double(), d.double() + e * direction, 32 ** -0.5, s.double())[0] * w.double()).sum())  # noqa: E731
    h = 1e-5
    _, _, mag = seq_ref.attention_grads(q.abs(), k.abs(), v.abs(), d, 32 ** -0.5, s.abs(), None, w.abs(), None)
    bound = float((decay_magnitude(q, k, v, mag) * direction.abs()).sum()) * 2.0 ** -18
    assert abs(slope - (f(h) - f(-h)) / (2 * h)) < bound + 1e-8 * abs(f(0)) / h
