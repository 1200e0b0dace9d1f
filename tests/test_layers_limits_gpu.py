"""Where the gated recurrence, the norms, linear attention and the distillation loss come to their ends: batches of nothing that are trained on, single
tokens over a long memory, temperatures of any size, losses whose rounding to fp32 is the only one."""
import pytest
import torch

import layer_ref
from mamba2d_b200 import distillation_loss, gated_recurrence, gated_recurrence_step, group_norm, layer_norm, linear_attention, linear_attention_step
from test_recurrence_gpu import fast_scan

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16
FORMS = ("decay", "forget")


def leaf(*shape, dt=F32):
    return torch.full(shape, 0.5, device="cuda", dtype=dt, requires_grad=True)


def zeros_for(out, leaves):
    """Every leaf gets a gradient of its own shape and type, which is zero."""
    out = [t for t in (out if isinstance(out, tuple) else (out,))]
    for t, g in zip(leaves, torch.autograd.grad(out, leaves, [torch.ones_like(t) for t in out])):
        assert g.shape == t.shape and g.dtype == t.dtype and bool((g == 0).all())


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("shape", [(0, 8), (4, 0, 8), (3, 0)])
def test_layer_norm_of_nothing(shape, dt):
    """Parameters get zeros for a share without rows, whether x needs a gradient or not: under DistributedDataParallel none may be left out."""
    C = shape[-1]
    x, r, w, b = leaf(*shape, dt=dt), leaf(*shape, dt=dt), leaf(C), leaf(C, dt=F32)
    zeros_for(layer_norm(x, w, b), (x, w, b))
    zeros_for(layer_norm(x.detach(), w, b), (w, b))
    zeros_for(layer_norm(x.detach(), None, b), (b,))
    y, s = layer_norm(x, w, b, residual=r)
    assert y.shape == s.shape == x.shape and y.dtype == s.dtype == dt
    zeros_for((y, s), (x, r, w, b))
    zeros_for(layer_norm(x, w, b, residual=r)[1], (x, r, w, b))
    assert not layer_norm(x.detach(), w.detach()).requires_grad


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("B,T,C", [(2, 0, 8), (0, 5, 8), (2, 5, 0)])
def test_the_recurrence_of_nothing(B, T, C, form, dt):
    """x and gate get gradients, and the state, which passes through, its own."""
    x, g, s = leaf(B, T, C, dt=dt), leaf(B, T, C, dt=dt), leaf(B, C)
    zeros_for(gated_recurrence(x, g, form=form), (x, g))
    zeros_for(gated_recurrence(x.detach(), g, form=form), (g,))
    part = leaf(1, 1, C, dt=dt)
    zeros_for(gated_recurrence(x, part.expand(B, T, C), form=form), (part,))
    for lengths in (None, torch.zeros(B, dtype=torch.int32, device="cuda")):
        h, last = gated_recurrence(x, g, form=form, initial_state=s, lengths=lengths, return_state=True)
        assert h.shape == x.shape and h.dtype == dt and torch.equal(last, s) and last.data_ptr() != s.data_ptr() or not s.numel()
        up = torch.randn(B, C, device="cuda")
        dx, dg, ds = torch.autograd.grad((h, last), (x, g, s), (torch.ones_like(h), up))
        assert dx.shape == dg.shape == x.shape and torch.equal(ds, up)
        zeros_for(gated_recurrence(x, g, form=form, initial_state=s, lengths=lengths), (x, g, s))
    h, last = gated_recurrence(x, g, form=form, return_state=True)
    assert last.shape == (B, C) and bool((last == 0).all())
    zeros_for((h, last), (x, g))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("shape", [(0, 8), (4, 0, 8), (0, 3, 3, 8)])
def test_group_norm_of_nothing(shape, dt):
    x, w, b = leaf(*shape, dt=dt), leaf(8), leaf(8)
    zeros_for(group_norm(x, 2, w, b, act="silu"), (x, w, b))
    zeros_for(group_norm(x.detach(), 2, w, b), (w, b))
    zeros_for(group_norm(x.detach(), 2, None, b), (b,))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,T", [(2, 0), (0, 5)])
def test_linear_attention_of_nothing(B, T, dt):
    q, k, v, s = leaf(B, T, 1, 16, dt=dt), leaf(B, T, 1, 16, dt=dt), leaf(B, T, 2, 24, dt=dt), leaf(B, 2, 16, 24)
    for g in (leaf(2), leaf(B, T, 2), leaf(2, dt=BF)):
        zeros_for(linear_attention(q, k, v, g), (q, k, v, g))
        o, last = linear_attention(q, k, v, g, initial_state=s, return_state=True)
        up = torch.randn_like(s)
        *rest, ds = torch.autograd.grad((o, last), (q, k, v, g, s), (torch.ones_like(o), up))
        assert torch.equal(last, s) and torch.equal(ds, up) and all(bool((t == 0).all()) for t in rest)
    zeros_for(linear_attention(q, k, v.detach(), leaf(2).detach()), (q, k))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("form", FORMS)
def test_single_tokens_over_a_long_memory(form, dt):
    """A gate that all tokens share and a memory of some 8192 of them, M, for 20000 tokens.  What a token's rounding of its gate is off by has the same sign
    every time and would add up, to M times 2^-25 or more (2.4e-4).  What may be left: each state's own rounding, at most 2^-24 of it and as often up as down (x is
    random), whose share after M tokens has a deviation of 2^-24 (M / 2 / 3)^0.5 = 2.2e-6 at most, of which eight are allowed; and 2^-20, for what 1 - a and the
    weight of x are off by."""
    T, C = 20000, 32
    k = 0.01 * torch.arange(C, device="cuda")
    g = (-2.0 ** -13 * (1 + k) if form == "decay" else 9.01 - k)[None].to(dt)
    x = (1 + 0.5 * torch.randn(1, T, C, generator=torch.Generator().manual_seed(11)).cuda()).to(dt)
    a, u = layer_ref.terms(x.double(), g.double()[:, None].expand(1, T, C), form)
    start = 1.0 if form == "forget" else float(1 / (1 - a).mean())
    state = torch.full((1, C), start, device="cuda")
    want = fast_scan(a, torch.cat((u[:, :1] + a[:, :1] * start, u[:, 1:]), 1))
    allowed = 8 * 2.0 ** -24 * (8192 / 6) ** 0.5 + 2.0 ** -20
    for t in range(T):
        y = gated_recurrence_step(x[:, t], g, state, form=form)
        if t % 2000 == 1999:
            assert float((state.double() / want[:, t] - 1).abs().max()) <= allowed, t
            assert torch.equal(y, state.to(dt))


@pytest.mark.parametrize("form", FORMS)
def test_single_tokens_at_their_ends(form):
    """Resets are exact, a state that nothing forgets stays, values that are not finite are the formula's, and no difference of large values overflows."""
    big = 3e38
    cases = [  # state, x, gate, what becomes of the state
        (5.0, 0.25, -torch.inf, 0.25), (1e30, 0.25, -torch.inf, 0.25 if form == "decay" else None), (-7.5, 0.0, 0.0 if form == "decay" else torch.inf, -7.5), (torch.inf, 1.0, -0.25 if form == "decay" else 3.0, torch.inf),
        (1.0, -torch.inf, -0.25 if form == "decay" else 3.0, -torch.inf), (torch.inf, torch.inf, -0.25 if form == "decay" else 3.0, torch.inf), (torch.nan, 1.0, -0.25, torch.nan), (1.0, torch.nan, -0.25, torch.nan),
        (1.0, 1.0, torch.nan, torch.nan), (-big, big, -0.125 if form == "decay" else 2.0, None), (big, -big, -0.5 if form == "decay" else 0.25, None), (2.0, 3.0, -0.6931472 if form == "decay" else 0.0, None)]
    s, x, g = (torch.tensor([c[k] for c in cases], device="cuda")[None] for k in range(3))
    a, u = layer_ref.terms(x.double(), g.double(), form)
    state = s.clone()
    y = gated_recurrence_step(x, g, state, form=form)
    assert torch.equal(torch.nan_to_num(y, nan=12345.0), torch.nan_to_num(state, nan=12345.0))
    want, size = a * s.double() + u, a * s.double().abs() + u.abs()
    for k, c in enumerate(cases):
        got = float(state[0, k])
        if c[3] is None:                 # (forget gates below -87 count as -87, of which 1.7e-38 of the state is left)
            assert abs(got - float(want[0, k])) <= 2.0 ** -20 * float(size[0, k]) + 1.7e-38 * abs(c[0]), c
        elif c[3] != c[3]:
            assert got != got, c
        else:
            assert got == c[3], c


@pytest.mark.parametrize("V", [2, 20001])
@pytest.mark.parametrize("temperature", [1.0, 2.5, 3.5])
def test_a_loss_is_rounded_once(V, temperature):
    """Rows of two classes far apart (others are masked) whose teacher wants the lower one: temperature times the distance, to what fp32 holds.
    Everything that is computed in 64 bits is off by less than 2^-40 of it."""
    N = 64
    z = torch.full((N, V), -torch.inf, device="cuda")
    far = 150 + 3.7 * torch.arange(N, device="cuda")
    z[:, 0], z[:, 1] = 0.0, -far
    t, index = torch.zeros(N, 1, device="cuda"), torch.ones(N, 1, dtype=torch.long, device="cuda")
    want = temperature * far.double()
    assert layer_ref.within(distillation_loss(z, t, index, temperature=temperature), want, 2.0 ** -40 * want) <= 1


@pytest.mark.parametrize("temperature", [1e-40, 2e-39, 1e-30, 1e4, 3e38])
@pytest.mark.parametrize("V", [50, 20001])
@pytest.mark.parametrize("dt", [F32, BF])
def test_temperatures_of_any_size(V, dt, temperature):
    """The teacher's only entry is the student's largest class, or another one: cold, q is one for the largest and zero for others; hot, it is 1 / V."""
    z = torch.linspace(-3, 3, V, device="cuda").expand(2, V).contiguous().to(dt).requires_grad_(True)
    index = torch.tensor([[V - 1], [0]], device="cuda")
    loss = distillation_loss(z, torch.zeros(2, 1, device="cuda"), index, temperature=temperature)
    assert not bool(torch.isnan(loss).any())
    assert float(loss[0].detach()) == 0.0 or temperature > 1 or dt == BF          # (bf16: several classes are the largest)
    up = 1e-20 if temperature > 1e20 else 1.0          # (a slope is temperature (q - p))
    dz, = torch.autograd.grad(loss, z, torch.full((2,), up, device="cuda"))
    assert bool(torch.isfinite(dz).all())
    ref = z.detach().double()
    q = torch.softmax(ref / temperature, -1)
    p = torch.zeros_like(q).scatter_(1, index, 1.0)
    want = up * temperature * (q - p)
    # (sums of up to 20001 values and exponents near zero: 2^-16; what is below fp32's smallest normal number may be lost)
    assert layer_ref.within(dz, want, 2.0 ** -16 * up * temperature * (q + p)) <= 1


@pytest.mark.parametrize("dt", [F32, BF])
def test_single_tokens_of_linear_attention_over_a_long_memory(dt):
    """The same, for decays that all tokens of a head share: the state against the formula in 64 bits, one token after another."""
    T, H, K, V = 20000, 4, 8, 24
    g = torch.tensor([-2.0 ** -13, -1.1 * 2.0 ** -13, -1.7 * 2.0 ** -13, -2.9 * 2.0 ** -13], device="cuda")
    random = torch.Generator().manual_seed(15)
    k, v = ((1 + 0.5 * torch.randn(T, 1, H, n, generator=random)).cuda().to(dt) for n in (K, V))
    a = g.double().exp()[None, :, None, None]
    state = (1 / (1 - a)).float().expand(1, H, K, V).contiguous()
    want = state.double()
    allowed = 8 * 2.0 ** -24 * (8192 / 6) ** 0.5 + 2.0 ** -20
    for t in range(T):
        linear_attention_step(k[t], k[t], v[t], g, state)
        want = want * a + k[t].double()[..., None] * v[t].double()[..., None, :]
        if t % 2000 == 1999:
            assert float((state.double() / want - 1).abs().max()) <= allowed, t


def test_single_tokens_of_linear_attention_at_their_ends():
    """States of infinity, NaN and next to the largest number under decays that keep all, most and little of them: the formula's."""
    g = torch.tensor([0.0, -2.0 ** -20, -0.1, -0.693, -0.7, -3.0, -80.0, 0.5, 1.0], device="cuda")
    values = torch.tensor([torch.inf, -torch.inf, torch.nan, 3e38, -3e38, 1.0, 0.0, -1e-30], device="cuda")
    H, K, V = len(g), 4, len(values)
    k, v = torch.tensor([[1.0, -2.0, 0.0, 1e-20]], device="cuda").expand(1, H, K), torch.ones(1, H, V, device="cuda")
    state = values.expand(1, H, K, V).contiguous()
    want = state.double() * g.double().exp()[None, :, None, None] + (k[..., None] * v[..., None, :]).double()
    size = state.double().abs() * g.double().exp()[None, :, None, None] + k[..., None].double().abs()
    linear_attention_step(k, k, v, g, state)
    over = want.abs() > torch.finfo(F32).max
    want = torch.where(over & ~torch.isnan(want), want.sign() * torch.inf, want)
    bad = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(state), torch.isnan(want)) and torch.equal(state[bad & ~torch.isnan(want)].double(), want[bad & ~torch.isnan(want)])
    # (-1e-30 under a decay of -80 is -1.8e-65, of which fp32 has nothing: a value near zero is off by its smallest step, 2^-149, whatever its size)
    assert bool(((state.double() - want).abs() <= 2.0 ** -20 * size + 2.0 ** -149)[~bad].all())
