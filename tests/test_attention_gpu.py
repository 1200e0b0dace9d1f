"""Linear attention with a decay per head (mamba2d_b200.linear_attention, linear_attention_step) against its definition
in 64 bits.

Shares of the sum of magnitudes that a result may be off by (see seq_ref): fp32 tensors, 2^-18: the products of split
operands leave out 3 * 2^-22 of each term, three products follow one another, and sums of some hundred fp32 terms are off
by a few times 2^-24 of theirs.  bf16 tensors: pairs' products and states are rounded to bf16 before the second product, 2^-8 (half a step)
each, and only one of the two lies on a term's way; outputs are rounded once more, 2^-8 of their value.  States and the
decay's gradient are float32 and stay at 2^-16 with bf16 tensors (two bf16 parts for what is rounded; sums over a run of tokens).
"""
import pytest
import torch

import seq_ref
from mamba2d_b200 import linear_attention, linear_attention_step

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def make(B, T, H, G, K, V, dt, decay="token", state=False, ragged=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + T + 7 * K + V)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    u = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    q, k, v = n(B, T, G, K).to(dt), (n(B, T, G, K) * K ** -0.5).to(dt), n(B, T, H, V).to(dt)
    d = -0.3 * u(H) if decay == "head" else -u(B, T, H) * torch.exp(3 * u(H) - 3)
    s = n(B, H, K, V) if state else None
    lengths = (u(B) * (T + 1)).int().clamp(max=T) if ragged else None
    return q, k, v, d, s, lengths


def share(dt, rounded):
    return 2.0 ** -18 if dt == F32 else 2.0 ** -7 if rounded else 2.0 ** -16


def rounding(t):
    return torch.finfo(t.dtype).eps / 2


def forward(q, k, v, d, s, lengths, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    o, final = linear_attention(q, k, v, d, scale=scale, initial_state=s, lengths=lengths, return_state=True)
    ab = [t.double().abs() if t is not None else None for t in (q, k, v)]
    want, wfinal = seq_ref.attention(q.double(), k.double(), v.double(), d.double(), scale, None if s is None else s.double(), lengths)
    mag, mfinal = seq_ref.attention(*ab, d.double(), abs(scale), None if s is None else s.double().abs(), lengths)
    assert o.dtype == v.dtype and o.shape == v.shape and final.dtype == F32
    assert seq_ref.within(o, want, mag, share(v.dtype, True), rounding(o)) < 1
    assert seq_ref.within(final, wfinal, mfinal, share(v.dtype, False), rounding(final)) < 1
    return o, final


SHAPES = [(1, 1, 1, 1, 1, 1), (2, 1, 3, 1, 64, 64), (1, 2, 2, 2, 16, 8), (3, 63, 4, 2, 64, 64), (1, 64, 2, 2, 128, 128), (2, 65, 5, 5, 33, 47),
          (1, 127, 3, 3, 128, 64), (2, 128, 4, 1, 64, 128), (1, 129, 2, 1, 96, 80), (2, 300, 3, 3, 128, 128), (1, 513, 2, 2, 64, 64), (1, 700, 1, 1, 256, 200),
          (1, 1100, 2, 1, 128, 128), (1, 640, 1, 1, 24, 256)]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,T,H,G,K,V", SHAPES)
def test_forward(B, T, H, G, K, V, dt):
    forward(*make(B, T, H, G, K, V, dt))
    forward(*make(B, T, H, G, K, V, dt, decay="head", state=True, ragged=B > 1))


def decay_magnitude(q, k, v, mag):
    """Of the decay's gradient: a suffix sum over up to 512 tokens of q.dq - k.dk, and a product of states; `mag`: the
    gradients for the magnitudes of all inputs."""
    per = lambda t: (t.double().sum(-1) if t.shape[2] == v.shape[2] else t.double().sum(-1).repeat_interleave(v.shape[2] // t.shape[2], 2))  # noqa: E731
    dots = per(q.abs().double() * mag[0]) + per(k.abs().double() * mag[1])
    B, T, H = dots.shape
    runs = -(-T // 512)
    pad = torch.nn.functional.pad(dots, (0, 0, 0, runs * 512 - T)).view(B, runs, 512, H)
    return pad.flip(2).cumsum(2).flip(2).reshape(B, runs * 512, H)[:, :T] + (mag[3] if mag[3].dim() == 3 else mag[3].expand(B, T, H))


def backward(q, k, v, d, s, lengths, with_state):
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (q, k, v, d, s)]
    scale = q.shape[-1] ** -0.5
    g = torch.Generator(device="cuda").manual_seed(5)
    d_o = torch.randn(v.shape, generator=g, device="cuda").to(v.dtype)
    d_state = torch.randn(v.shape[0], v.shape[2], q.shape[-1], v.shape[-1], generator=g, device="cuda") if with_state else None
    out = linear_attention(*leaves[:4], initial_state=leaves[4], lengths=lengths, return_state=with_state)
    got = torch.autograd.grad(out, [t for t in leaves if t is not None], (d_o, d_state) if with_state else d_o)
    _, _, want = seq_ref.attention_grads(q, k, v, d, scale, s, lengths, d_o, d_state)
    ab = lambda t: None if t is None else t.abs()  # noqa: E731
    _, _, mag = seq_ref.attention_grads(q.abs(), k.abs(), v.abs(), d, scale, ab(s), lengths, d_o.abs(), ab(d_state))
    it = iter(got)
    for i, (name, w, m) in enumerate(zip(("q", "k", "v", "decay", "state"), want, mag)):
        if w is None:
            continue
        x = next(it)
        if name == "decay":
            m = decay_magnitude(q, k, v, mag)
            if w.dim() == 1:
                m = m.sum((0, 1))
        ratio = seq_ref.within(x, w, m, share(v.dtype, name in ("q", "k", "v")), rounding(x))
        assert ratio < 1, (name, ratio)
    return got


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,T,H,G,K,V", SHAPES)
def test_backward(B, T, H, G, K, V, dt):
    backward(*make(B, T, H, G, K, V, dt), False)
    backward(*make(B, T, H, G, K, V, dt, decay="head", state=True, ragged=B > 1), True)


@pytest.mark.parametrize("dt", [F32, BF])
def test_decays_of_zero_of_nothing_left_and_of_minus_infinity(dt):
    q, k, v, d, s, _ = make(2, 200, 3, 3, 64, 64, dt, state=True)
    d[0] = 0.0                                                  # nothing is forgotten
    d[1, 50], d[1, 51], d[1, 130, 1], d[1, 131] = -float("inf"), -float("inf"), -float("inf"), -200.0
    d[1, 140:] = -30.0                                          # hardly anything is left of the token before
    o, final = forward(q, k, v, d, s, None)
    # behind a -inf the sequence starts again
    alone, last = forward(q[1:, 51:], k[1:, 51:], v[1:, 51:], d[1:, 51:], None, None)
    assert torch.equal(final[1, 0], last[0, 0]) or float((final[1, 0] - last[0, 0]).abs().max()) < 1e-5
    backward(q, k, v, d, s, None, True)


@pytest.mark.parametrize("dt", [F32, BF])
def test_gradient_of_the_decay_against_differences(dt):
    """Central differences of a sum over the outputs, in one direction of the decays, from the 64-bit definition.  The
    slope is a sum of gradients, and may be off by the sum of what each of them may be off by (``decay_magnitude``):
    with bf16 tensors 2^-16 of some hundreds, times 180 tokens and heads."""
    q, k, v, d, s, _ = make(1, 90, 2, 1, 32, 32, dt, state=True)
    g = torch.Generator(device="cuda").manual_seed(11)
    w, direction = torch.randn(v.shape, generator=g, device="cuda").to(dt), torch.randn(d.shape, generator=g, device="cuda")
    dd = d.clone().requires_grad_(True)
    o = linear_attention(q, k, v, dd, initial_state=s)
    slope = float((torch.autograd.grad(o, dd, w)[0].double() * direction).sum())
    f = lambda e: float((seq_ref.attention(q.double(), k.double(), v.double(), d.double() + e * direction, 32 ** -0.5, s.double())[0] * w.double()).sum())  # noqa: E731
    h = 1e-5
    want = (f(h) - f(-h)) / (2 * h)
    _, _, mag = seq_ref.attention_grads(q.abs(), k.abs(), v.abs(), d, 32 ** -0.5, s.abs(), None, w.abs(), None)
    bound = float((decay_magnitude(q, k, v, mag) * direction.abs()).sum()) * share(dt, False)
    assert abs(slope - want) < bound + 1e-8 * abs(f(0)) / h


@pytest.mark.parametrize("dt", [F32, BF])
def test_rows_behind_a_length_are_not_read(dt):
    q, k, v, d, s, _ = make(4, 333, 3, 3, 64, 64, dt, state=True)
    lengths = torch.tensor([0, 1, 200, 333], dtype=torch.int32, device="cuda")
    want = backward(q, k, v, d, s, lengths, True)
    o, final = linear_attention(q, k, v, d, initial_state=s, lengths=lengths, return_state=True)
    for b, n in enumerate(lengths.tolist()):
        for t in (q, k, v, d):
            t[b, n:] = float("nan")
    o2, final2 = linear_attention(q, k, v, d, initial_state=s, lengths=lengths, return_state=True)
    assert torch.equal(o, o2) and torch.equal(final, final2)
    assert torch.equal(final[0], s[0])
    for b, n in enumerate(lengths.tolist()):
        assert not o[b, n:].any()
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, d, s)]
    out = linear_attention(*leaves[:4], initial_state=leaves[4], lengths=lengths, return_state=True)
    g = torch.Generator(device="cuda").manual_seed(5)
    d_o = torch.randn(v.shape, generator=g, device="cuda").to(v.dtype)
    d_state = torch.randn(final.shape, generator=g, device="cuda")
    for b, n in enumerate(lengths.tolist()):
        d_o[b, n:] = float("inf")
    for x, y in zip(torch.autograd.grad(out, leaves, (d_o, d_state)), want):
        assert torch.equal(x, y)
    # beyond the range: clamped; 64-bit integers
    far = torch.tensor([-5, 1, 200, 2 ** 40], device="cuda")
    for b in (0, 3):
        for t in (q, k, v, d):
            t[b] = 0.5 if t is not d else -0.5
    x = linear_attention(q, k, v, d, initial_state=s, lengths=far)
    y = linear_attention(q, k, v, d, initial_state=s, lengths=lengths)
    assert torch.equal(x, y)


@pytest.mark.parametrize("dt", [F32, BF])
def test_strides_and_alignment(dt):
    B, T, H, G, K, V = 2, 150, 4, 2, 64, 64
    q, k, v, d, s, _ = make(B, T, H, G, K, V, dt, state=True)
    want = linear_attention(q, k, v, d, initial_state=s)
    packed = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1)                     # one projection's output
    a, b, c = packed.split([G * K, G * K, H * V], -1)
    views = [a.view(B, T, G, K), b.view(B, T, G, K), c.view(B, T, H, V)]
    assert torch.equal(want, linear_attention(*views, d, initial_state=s))
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(want, linear_attention(*heads_first, d.transpose(1, 2).contiguous().transpose(1, 2), initial_state=s))

    def odd(t):                                                                             # rows that start anywhere
        w = torch.empty(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device="cuda")
        w[..., 1:-2] = t
        return w[..., 1:-2]
    near = linear_attention(odd(q), odd(k), odd(v), d, initial_state=s)
    assert float((near.float() - want.float()).norm() / want.float().norm()) < (1e-5 if dt == F32 else 8e-3)
    last = [t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in (q, k, v)]           # copied
    assert torch.equal(want, linear_attention(*last, d, initial_state=s))
    forward(odd(q), k, odd(v), d.expand(B, T, H), s, None)


def test_prompts_in_pieces_and_by_single_tokens():
    """A prompt in two pieces, and token by token, carries the same state."""
    for dt in (F32, BF):
        q, k, v, d, s, _ = make(2, 140, 4, 2, 64, 48, dt, state=True)
        o, final = linear_attention(q, k, v, d, initial_state=s, return_state=True)
        o1, mid = linear_attention(q[:, :77], k[:, :77], v[:, :77], d[:, :77], initial_state=s, return_state=True)
        o2, end = linear_attention(q[:, 77:], k[:, 77:], v[:, 77:], d[:, 77:], initial_state=mid, return_state=True)
        state = s.clone()
        single = torch.stack([linear_attention_step(q[:, t], k[:, t], v[:, t], d[:, t], state) for t in range(140)], 1)
        tol = 2e-5 if dt == F32 else 1e-2
        for x in (torch.cat([o1, o2], 1), single):
            assert float((x.float() - o.float()).norm() / o.float().norm()) < tol
        for x in (end, state):
            assert float((x - final).norm() / final.norm()) < 2e-5


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,H,G,K,V", [(1, 1, 1, 1, 1), (3, 4, 2, 64, 64), (2, 3, 3, 33, 47), (5, 2, 1, 128, 128), (1, 2, 2, 256, 256), (70, 3, 1, 130, 132), (2, 1, 1, 7, 200)])
def test_step(B, H, G, K, V, dt):
    q, k, v, d, s, _ = make(B, 1, H, G, K, V, dt, state=True)
    for decay in (d[:, 0], d[0, 0]):
        state = s.clone()
        o = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, state, scale=0.7)
        dd = (decay if decay.dim() == 2 else decay.expand(B, H))[:, None].double()
        want, wstate = seq_ref.attention(q.double(), k.double(), v.double(), dd, 0.7, s.double())
        mag, mstate = seq_ref.attention(q.double().abs(), k.double().abs(), v.double().abs(), dd, 0.7, s.double().abs())
        assert seq_ref.within(o, want[:, 0], mag[:, 0], 2.0 ** -20, rounding(o)) < 1
        assert seq_ref.within(state, wstate, mstate, 2.0 ** -21, 2.0 ** -24) < 1


def test_step_of_a_slice_of_a_cache_leaves_the_rest():
    B, H, K, V = 3, 4, 64, 48
    q, k, v, d, s, _ = make(B, 1, H, H, K, V, BF, state=True)
    want = s.clone()
    o = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], d[:, 0], want)
    cache = torch.full((H + 2, B + 1, 2, K, V), 7.0, device="cuda")
    view = cache[1:H + 1, :B, 1].transpose(0, 1)                       # heads far apart, sequences near
    view.copy_(s)
    version = cache._version
    assert torch.equal(o, linear_attention_step(q[:, 0], k[:, 0], v[:, 0], d[:, 0], view))
    assert cache._version > version and torch.equal(view, want)
    mask = torch.ones_like(cache, dtype=torch.bool)
    mask[1:H + 1, :B, 1] = False
    assert bool((cache[mask] == 7.0).all())


def test_empty_sequences():
    q, k, v, d, s, _ = make(2, 5, 2, 2, 16, 16, F32, state=True)
    o, final = linear_attention(q[:, :0], k[:, :0], v[:, :0], d[:, :0], initial_state=s, return_state=True)
    assert o.shape == (2, 0, 2, 16) and torch.equal(final, s) and final.data_ptr() != s.data_ptr()
    o, final = linear_attention(q[:0], k[:0], v[:0], d[:0], return_state=True)
    assert o.shape == (0, 5, 2, 16) and final.shape == (0, 2, 16, 16)
    assert linear_attention_step(q[:0, 0], k[:0, 0], v[:0, 0], d[:0, 0], s[:0]).shape == (0, 2, 16)


def test_gradients_through_the_state_alone_and_through_nothing():
    q, k, v, d, s, _ = make(2, 70, 2, 2, 32, 32, F32, state=True)
    vv, ss = v.clone().requires_grad_(True), s.clone().requires_grad_(True)
    o, final = linear_attention(q, k, vv, d, initial_state=ss, return_state=True)
    dv, ds = torch.autograd.grad(final.sum(), [vv, ss])
    c = d.double().cumsum(1)
    left = torch.exp(c[:, -1:] - c)
    want = left * k.double().sum(-1)
    assert float((dv.double() - want[..., None]).abs().max()) < 1e-5
    assert float((ds.double() - torch.exp(c[:, -1])[..., None, None]).abs().max()) < 1e-6
    with pytest.raises(RuntimeError):
        linear_attention_step(q[:, 0], k[:, 0], vv[:, 0], d[:, 0], s)


@pytest.mark.parametrize("dt", [F32, BF])
def test_streams_threads_and_captured_graphs(dt):
    """Two graphs of the same call, replayed in turn with other inputs, and a call on another stream."""
    args = make(2, 700, 2, 1, 64, 64, dt, state=True)
    other = make(2, 700, 2, 1, 64, 64, dt, state=True, seed=9)
    call = lambda a: linear_attention(*a[:4], initial_state=a[4], return_state=True)  # noqa: E731
    want, want2 = call(args), call(other)
    static = [t.clone() if t is not None else None for t in args]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = call(static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(on_side, want))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(call(static))
    for turn in range(2):
        for src, expect in ((other, want2), (args, want)):
            for t, x in zip(static, src):
                if t is not None:
                    t.copy_(x)
            for g in graphs:
                g.replay()
            for o in outs:
                assert all(torch.equal(x, y) for x, y in zip(o, expect))


def test_repeated_calls_give_the_same_bits():
    args = make(3, 900, 4, 2, 128, 64, BF, state=True)
    a, b = backward(*args, True), backward(*args, True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
