"""The gated recurrence against its definition in 64 bits, element by element, within the bound that ``layer_ref`` derives."""
import ctypes

import pytest
import torch

import layer_ref
from mamba2d_b200 import _lib, gated_recurrence, gated_recurrence_step
from test_layers_host import RecurDesc, RecurTensor

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16
FORMS = ("decay", "forget")


def inputs(B, T, C, dt, form, seed=0, state=False):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    rate = torch.rand(C, generator=g).cuda()
    x = n(B, T, C).to(dt)
    # memories from a token to some thousand, side by side
    gate = (-torch.nn.functional.softplus(n(B, T, C)) * torch.exp(-7 * rate)).to(dt) if form == "decay" else (n(B, T, C) + 10 * rate - 2).to(dt)
    return x, gate, n(B, C) if state else None, n(B, T, C).to(dt), n(B, C)


def check(x, gate, form, state, lengths, dy, d_state):
    """Forward with and without gradients, and the gradients."""
    x64, g64 = (t.double().requires_grad_(True) for t in (x, gate))
    s64 = None if state is None else state.double().requires_grad_(True)
    h, final = layer_ref.recurrence(x64, g64, form, s64, lengths)
    leaves = [t for t in (x64, g64, s64) if t is not None]
    live = None if lengths is None else (torch.arange(x.shape[1], device=x.device) < lengths[:, None])[..., None]
    up = dy.double() if live is None else torch.where(live, dy.double(), 0.0)
    want = torch.autograd.grad((h, final), leaves, (up, d_state.double()))
    with torch.no_grad():
        bounds = layer_ref.recurrence_bounds(x.double(), gate.double(), form, None if state is None else state.double(), lengths, up, d_state.double())
        got, got_final = gated_recurrence(x, gate, form=form, initial_state=state, lengths=lengths, return_state=True)
    assert got.dtype == x.dtype and got_final.dtype == F32
    assert layer_ref.within(got, h.detach(), bounds[0]) <= 1
    assert layer_ref.within(got_final, final.detach(), bounds[1]) <= 1
    own = [t.detach().requires_grad_(True) if t is not None else None for t in (x, gate, state)]
    out = gated_recurrence(own[0], own[1], form=form, initial_state=own[2], lengths=lengths, return_state=True)
    assert torch.equal(out[0], got) and torch.equal(out[1], got_final)
    grads = torch.autograd.grad(out, [t for t in own if t is not None], (dy, d_state))
    for a, w, b in zip(grads, want, bounds[2:]):
        assert layer_ref.within(a, w, b) <= 1
    return got, grads


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,T,C", [(1, 1, 1), (2, 1, 64), (3, 2, 33), (1, 15, 7), (2, 16, 64), (2, 17, 66), (1, 63, 130), (2, 64, 32), (1, 65, 96), (2, 127, 31), (3, 128, 64),
                                   (1, 129, 200), (2, 300, 65), (1, 1025, 48), (5, 777, 130)])
def test_sizes(B, T, C, dt, form):
    check(*(lambda x, g, s, dy, ds: (x, g, form, s, None, dy, ds))(*inputs(B, T, C, dt, form, state=T % 2 == 1)))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dt", [F32, BF])
def test_ragged(dt, form):
    """Lengths of zero, one, in the middle, whole and beyond; rows behind them hold NaN and are not looked at."""
    x, g, s, dy, ds = inputs(7, 200, 70, dt, form, 1, True)
    lengths = torch.tensor([0, 1, 64, 129, 199, 200, 500], dtype=torch.int32, device="cuda")
    behind = (torch.arange(200, device="cuda") >= lengths[:, None])[..., None]
    x, g, dy = (torch.where(behind, torch.nan, t.float()).to(dt) for t in (x, g, dy))
    n = lengths.clamp(max=200)
    got, grads = check(x, g, form, s, n, dy, ds)
    for t in (got, *grads[:2]):
        assert bool((t.masked_select(behind) == 0).all())
    for counts in (lengths, lengths.long(), lengths.long() - 1000 * (lengths == 0)):
        assert torch.equal(gated_recurrence(x, g, form=form, initial_state=s, lengths=counts), got)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dt", [F32, BF])
def test_strides(dt, form):
    """A slice of a wider projection, transposed batches, channels that are not dense, rows at odd offsets, a gate that all tokens (sequences,
    channels) share."""
    B, T, C = 3, 140, 64
    x, g, s, dy, ds = inputs(B, T, C, dt, form, 2, True)
    want, grads = check(x, g, form, s, None, dy, ds)

    def same(x, g, s, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, g, s)]
        h = gated_recurrence(leaves[0], leaves[1], form=form, initial_state=leaves[2])
        assert torch.equal(h, want)
        return torch.autograd.grad(h, leaves, dy)
    plain = same(x, g, s, dy)
    wide = torch.cat((x, g, dy), -1)
    for a, b in zip(plain, same(wide[..., :C], wide[..., C:2 * C], s, wide[..., 2 * C:])):
        assert torch.equal(a, b)
    # (rows at odd offsets are read channel by channel and may be joined elsewhere: within the bounds, not to the bit)
    odd = torch.cat((x[..., :1], x, g[..., :2], g, dy[..., :1], dy), -1)
    check(odd[..., 1:C + 1], odd[..., C + 3:2 * C + 3], form, s, None, odd[..., 2 * C + 4:], ds)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, g, dy)]
    for a, b in zip(plain, same(turned[0], turned[1], s, turned[2])):
        assert torch.equal(a, b)
    apart = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (x, g, dy)]
    for a, b in zip(plain, same(apart[0], apart[1], s.t().contiguous().t(), apart[2])):
        assert torch.equal(a, b)
    for part in (g[:1, :1], g[:, :1], g[:1], g[..., :1]):
        leaf, full = part.detach().clone().requires_grad_(True), part.expand(B, T, C).contiguous().requires_grad_(True)
        one, = torch.autograd.grad(gated_recurrence(x, leaf.expand(B, T, C), form=form), leaf, dy)
        other, = torch.autograd.grad(gated_recurrence(x, full, form=form), full, dy)
        assert one.shape == part.shape
        dims = [d for d in range(3) if part.shape[d] == 1]
        assert float((one.double() - other.double().sum(dims, keepdim=True)).abs().max()) <= 2.0 ** -7 * float(other.abs().double().sum(dims).max())
    up, = torch.autograd.grad(gated_recurrence(x, plain_leaf := g.detach().requires_grad_(True), form=form).sum(), plain_leaf)      # an expanded gradient
    full, = torch.autograd.grad(gated_recurrence(x, plain_leaf, form=form), plain_leaf, torch.ones_like(x))
    assert torch.equal(up, full)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("form", FORMS)
def test_gates_at_their_ends(form, dt):
    """Gates of -inf (and +inf where they forget nothing), far ones, and ones next to zero: a reset is exact, a state that nothing
    forgets stays, and no product of an infinity and a zero appears."""
    x, g, s, dy, ds = inputs(2, 200, 64, dt, form, 3, True)
    g = g.clone()
    g[0, 50] = g[1, 128] = -torch.inf
    g[0, 100:120, 3] = -90.0
    g[0, 60:200, 5] = 0.0 if form == "decay" else torch.inf
    g[1, 0:100, 7] = -1e-6 if form == "decay" else 30.0
    g[1, 130:140] = -20.0
    got, grads = check(x, g, form, s, None, dy, ds)
    assert torch.equal(got[0, 50], x[0, 50])
    fresh = gated_recurrence(x[:1, 50:], torch.cat((torch.full_like(g[:1, :1], -torch.inf), g[:1, 51:]), 1), form=form)
    assert float((fresh[0, :20].float() - got[0, 50:70].float()).abs().max()) <= 2.0 ** -6 * float(got[0, 50:70].abs().max())
    assert bool((grads[2][1] != 0).any())


@pytest.mark.parametrize("form", FORMS)
def test_a_long_memory_in_fp32(form):
    """The same gate at every token, a memory of 8192 of them: errors of a gate's rounding would add up (2^-24 against 2^-13, 5e-4)."""
    T, C = 6000, 32
    x = torch.ones(1, T, C, device="cuda")
    g = torch.full((1, T, C), -2.0 ** -13 if form == "decay" else 9.01, device="cuda") * (1 + 0.01 * torch.arange(C, device="cuda"))
    a, u = layer_ref.terms(x.double(), g.double(), form)
    n = torch.arange(1, T + 1, device="cuda", dtype=torch.float64)[:, None]
    want = u[0] * (-torch.expm1(n * torch.log(a[0])) / (1 - a[0]))       # the geometric sum
    got = gated_recurrence(x, g, form=form)[0]
    assert float(((got.double() - want).abs() / want).max()) < 6000 ** 0.5 * 4 * 2.0 ** -24 + 2.0 ** -18


def test_nan_stays_where_the_formula_has_it():
    x, g, s, dy, ds = inputs(2, 300, 32, F32, "decay", 4, True)
    x = x.clone()
    x[1, 150, 3] = torch.nan
    leaf = x.clone().requires_grad_(True)
    h = gated_recurrence(leaf, g, initial_state=s)
    bad = torch.isnan(h)
    want = torch.zeros_like(bad)
    want[1, 150:, 3] = True
    assert torch.equal(bad, want)
    dy = dy.clone()
    dy[0, 100, 5] = torch.nan
    dx, = torch.autograd.grad(h, leaf, dy)
    want = torch.zeros_like(bad)
    want[0, :101, 5] = True
    assert torch.equal(torch.isnan(dx), want)


@pytest.mark.parametrize("form", FORMS)
def test_gradients_against_differences(form):
    """Central differences of the fp32 forward pass along random directions: with a step of 2^-6 the third derivative's share is some 1e-3 here,
    the rounding's 2^-23 * 2^6 of values near one."""
    x, g, s, dy, ds = inputs(2, 100, 48, F32, form, 5, True)
    leaves = [t.clone().requires_grad_(True) for t in (x, g, s)]
    out = gated_recurrence(leaves[0], leaves[1], form=form, initial_state=leaves[2], return_state=True)
    grads = torch.autograd.grad(out, leaves, (dy, ds))

    def f(x, g, s):
        h, last = gated_recurrence(x, g, form=form, initial_state=s, return_state=True)
        return (h.double() * dy.double()).sum() + (last.double() * ds.double()).sum()
    for i, t in enumerate((x, g, s)):
        way = torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).cuda() * (g.abs().clamp(max=1) if i == 1 else 1)
        step = 2.0 ** -6
        args = [x, g, s]
        up, down = [*args[:i], t + step * way, *args[i + 1:]], [*args[:i], t - step * way, *args[i + 1:]]
        slope, want = float((f(*up) - f(*down)) / (2 * step)), float((grads[i].double() * way.double()).sum())
        assert abs(slope - want) < 5e-3 * float((grads[i].double() * way.double()).norm()) * 3


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,C", [(1, 1), (1, 1024), (3, 33), (70000, 5), (257, 130)])
def test_single_tokens(B, C, dt, form):
    x, g, s, _, _ = inputs(B, 1, C, dt, form, 6, True)
    cache = torch.randn(B, 3, C, device="cuda")
    cache[:, 1] = s
    rest = cache.clone()
    a, u = layer_ref.terms(x[:, 0].double(), g[:, 0].double(), form)
    want, bound = a * s.double() + u, 2.0 ** -20 * (a * s.double().abs() + u.abs())
    y = gated_recurrence_step(x[:, 0], g[:, 0], cache[:, 1], form=form)
    assert y.dtype == dt
    assert layer_ref.within(y, want, bound) <= 1 and layer_ref.within(cache[:, 1], want, bound) <= 1
    assert torch.equal(cache[:, ::2], rest[:, ::2])


@pytest.mark.parametrize("form", FORMS)
def test_a_prompt_and_its_tokens(form):
    x, g, s, _, _ = inputs(2, 90, 40, BF, form, 7, True)
    whole, last = gated_recurrence(x, g, form=form, initial_state=s, return_state=True)
    first, state = gated_recurrence(x[:, :70], g[:, :70], form=form, initial_state=s, return_state=True)
    rows = [first] + [gated_recurrence_step(x[:, t], g[:, t], state, form=form)[:, None] for t in range(70, 90)]
    got = torch.cat(rows, 1)
    assert float((got.float() - whole.float()).abs().max()) <= 2.0 ** -7 * float(whole.abs().max())
    assert float((state - last).abs().max()) <= 2.0 ** -17 * float(last.abs().max()) * 4


def fast_scan(a, u):
    """``layer_ref.scan`` from pairs of tokens."""
    T = u.shape[1]
    if T == 1:
        return u
    odd = fast_scan(a[:, 1::2] * a[:, :T - 1:2], u[:, 1::2] + a[:, 1::2] * u[:, :T - 1:2])
    h = torch.empty_like(u)
    h[:, 1::2], h[:, 0], h[:, 2::2] = odd, u[:, 0], u[:, 2::2] + a[:, 2::2] * odd[:, :(T - 1) // 2]
    return h


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,T,C,ragged", [(1, 40001, 16, False), (1, 9000, 130, False), (2, 5000, 64, True), (1, 30000, 512, False), (3, 2049, 33, True), (9, 3000, 1026, True), (1, 200000, 2, False)])
def test_long_sequences(B, T, C, dt, form, ragged):
    """Sequences that several CTAs share.  The bound is ``layer_ref``'s."""
    x, g, s, dy, ds = inputs(B, T, C, dt, form, 8, True)
    lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(9)).cuda() if ragged else None
    n = torch.full((B,), T, device="cuda") if lengths is None else lengths
    live = (torch.arange(T, device="cuda") < n[:, None])[..., None]
    a, u = layer_ref.terms(x.double(), g.double(), form)
    a, u, up = torch.where(live, a, 1.0), torch.where(live, u, 0.0), torch.where(live, dy.double(), 0.0)
    first = lambda u, s: torch.cat((u[:, :1] + a[:, :1] * s[:, None], u[:, 1:]), 1)  # noqa: E731
    ahead = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), 1).flip(1)
    back = lambda up, s: fast_scan(ahead, torch.cat((up[:, :-1], up[:, -1:] + s[:, None]), 1).flip(1)).flip(1)  # noqa: E731
    bound = lambda a, H: 2.0 ** -17 * H + 1.25 * 2.0 ** -24 * fast_scan(a, H)  # noqa: E731
    h, D = fast_scan(a, first(u, s.double())), back(up, ds.double())
    H, E = fast_scan(a, first(u.abs(), s.double().abs())), back(up.abs(), ds.double().abs())
    dh, dD = bound(a, H), bound(ahead, E.flip(1)).flip(1)
    prior = lambda h, s: torch.cat((s[:, None], h[:, :-1]), 1)  # noqa: E731
    leaves = [t.detach().requires_grad_(True) for t in (x, g, s)]
    out = gated_recurrence(leaves[0], leaves[1], form=form, initial_state=leaves[2], lengths=lengths, return_state=True)
    grads = torch.autograd.grad(out, leaves, (dy, ds))
    assert layer_ref.within(out[0].detach(), torch.where(live, h, 0.0), dh) <= 1
    assert layer_ref.within(out[1].detach(), h[:, -1], dh[:, -1]) <= 1
    before, off = prior(h, s.double()), prior(dh, torch.zeros_like(s.double()))
    size = prior(H, s.double().abs())
    if form == "decay":
        dx, dg, bx, bg = D, a * D * before, dD, a * (dD * size + E * off)
    else:
        rest = torch.sigmoid(-g.double())
        dx, dg, bx, bg = rest * D, a * rest * D * (before - x.double()), rest * dD, a * rest * (dD * (size + x.double().abs()) + E * off)
    where = lambda t: torch.where(live, t, 0.0)  # noqa: E731
    assert layer_ref.within(grads[0], where(dx), bx + 2.0 ** -19 * E) <= 1
    assert layer_ref.within(grads[1], where(dg), bg + 2.0 ** -19 * a * E * (size + x.double().abs())) <= 1
    assert layer_ref.within(grads[2], a[:, 0] * D[:, 0], a[:, 0] * (dD[:, 0] + 2.0 ** -19 * E[:, 0])) <= 1
    again = gated_recurrence(x, g, form=form, initial_state=s, lengths=lengths)
    assert torch.equal(again, out[0])


@pytest.mark.parametrize("B,T,C", [(2, 30000, 128), (64, 3000, 512)])
def test_a_wait_that_gives_up(monkeypatch, B, T, C):
    """The first CTA asks for nothing: its results are NaN, and those of tokens behind its own, the next call raises, and the one after is right.
    Sequences of several CTAs and of one."""
    monkeypatch.setenv("M2D_TEST_HOOKS", "1")
    L = _lib.lib()
    x, g, s, dy, ds = inputs(B, T, C, BF, "decay", 10, True)
    want, last = gated_recurrence(x, g, initial_state=s, return_state=True)
    y, out, marks = torch.empty_like(x), torch.empty_like(s), torch.zeros(B, -(-T // 64), C, device="cuda")
    dx, dg, d0 = torch.empty_like(x), torch.empty_like(x), torch.empty_like(s)
    d = RecurDesc(struct_bytes=ctypes.sizeof(RecurDesc), dtype=1, B=B, T=T, C=C, form=0, flags=0x100)
    for name, t in (("x", x), ("gate", g), ("d_y", dy)):
        setattr(d, name, RecurTensor(t.data_ptr(), t.stride(0), t.stride(1)))
    for name, t in (("state", s), ("state_out", out), ("y", y), ("marks", marks), ("d_state_out", ds), ("d_x", dx), ("d_gate", dg), ("d_state", d0)):
        setattr(d, name, t.data_ptr())
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for call, first, others in ((L.m2d_recur_fwd, (y[0], out[0]), (y[1], out[1])), (L.m2d_recur_bwd, (dx[0], dg[0], d0[0]), (dx[1], dg[1], d0[1]))):
        assert call(ctypes.byref(d), stream) == 0
        torch.cuda.synchronize()
        assert all(bool(torch.isnan(t).any()) for t in first) and not any(bool(torch.isnan(t).any()) for t in others)
        with pytest.raises(RuntimeError, match="timed out"):
            gated_recurrence_step(x[:, 0], g[:, 0], s.clone())
        d.flags = 0                      # (marks for the backward pass)
        assert L.m2d_recur_fwd(ctypes.byref(d), stream) == 0
        assert torch.equal(y, want) and torch.equal(out, last)
        d.flags = 0x100
    assert torch.equal(gated_recurrence(x, g, initial_state=s), want)
