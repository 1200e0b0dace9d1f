"""Calls of the sequence operators that their documentation allows and ordinary use seldom makes: long sequences in few
and in many segments, heads shared without a decay's gradient, expanded inputs, offsets beyond 32 bits, captured backward
passes, two streams at once, gradients of gradients.  Tolerances are those of the operators' own tests."""
import copy

import pytest
import torch

import seq_ref
from test_attention_gpu import BF, F32, backward, forward, make, rounding, share
from mamba2d_b200 import clip_norm_, group_norm, linear_attention, linear_attention_step, refmodel

pytestmark = pytest.mark.gpu


# bf16: two segments, three and four (the kernels join them), five (a launch does), a tail of one token
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,T,H,G,K,V", [(3, 1100, 2, 1, 128, 64), (2, 2700, 1, 1, 64, 128), (1, 2561, 2, 2, 128, 128), (4, 1500, 1, 1, 64, 64), (1, 2100, 2, 1, 96, 64)])
def test_segments(B, T, H, G, K, V, dt):
    args = make(B, T, H, G, K, V, dt, state=True, ragged=B > 1)
    forward(*args)
    backward(*args, True)
    if B > 1:                                                  # whole segments behind the end, and nothing at all
        lengths = torch.tensor([0, 300, T, 513][:B], dtype=torch.int32, device="cuda")
        forward(*args[:5], lengths)
        backward(*args[:5], lengths, False)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,T,H,G,K,V", [(2, 300, 4, 2, 64, 64), (1, 1100, 6, 1, 128, 64), (2, 129, 2, 2, 64, 128)])
def test_gradients_without_that_of_the_decay(B, T, H, G, K, V, dt):
    q, k, v, d, s, _ = make(B, T, H, G, K, V, dt, state=True)
    scale = K ** -0.5
    d_o = torch.randn(v.shape, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(dt)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, s)]
    got = torch.autograd.grad(linear_attention(*leaves[:3], d, initial_state=leaves[3]), leaves, d_o)
    _, _, want = seq_ref.attention_grads(q, k, v, d, scale, s, None, d_o, None)
    _, _, mag = seq_ref.attention_grads(q.abs(), k.abs(), v.abs(), d, scale, s.abs(), None, d_o.abs(), None)
    for i, x in zip((0, 1, 2, 4), got):
        assert seq_ref.within(x, want[i], mag[i], share(dt, i < 3), rounding(x)) < 1, i


@pytest.mark.parametrize("dt", [F32, BF])
def test_expanded_inputs(dt):
    """Batch, tokens and heads that share memory; their gradients are sums."""
    q, k, v, d, s, _ = make(1, 200, 2, 1, 64, 64, dt, state=True)
    B = 3
    wide = [q.expand(B, -1, -1, -1), k[:, :1].expand(B, 200, 1, 64), v[:, :, :1].expand(B, 200, 2, 64), d.expand(B, -1, -1), s.expand(B, -1, -1, -1)]
    forward(*wide, None)
    leaf = q.clone().requires_grad_(True)
    dense = wide[0].clone().requires_grad_(True)
    d_o = torch.randn(B, 200, 2, 64, device="cuda").to(dt)
    a, = torch.autograd.grad(linear_attention(leaf.expand(B, -1, -1, -1), *wide[1:4], initial_state=wide[4]), leaf, d_o)
    b, = torch.autograd.grad(linear_attention(dense, *[t.contiguous() for t in wide[1:4]], initial_state=wide[4]), dense, d_o)
    b = b.double().sum(0, keepdim=True)
    assert float((a.double() - b).norm() / b.norm()) < (1e-5 if dt == F32 else 8e-3)
    # the gradient of a sum is one value, expanded
    x, = torch.autograd.grad(linear_attention(dense, *wide[1:4]).sum(), dense)
    y, = torch.autograd.grad(linear_attention(dense, *wide[1:4]), dense, torch.ones(B, 200, 2, 64, device="cuda", dtype=dt))
    assert torch.equal(x, y)


@pytest.mark.parametrize("dt", [F32, BF])
def test_offsets_beyond_32_bits(dt):
    """Sequences 2^31 elements apart, in tokens and in a cache of states."""
    B, T, H, K, V = 2, 130, 2, 64, 64
    q, k, v, d, s, _ = make(B, T, H, H, K, V, dt, state=True)
    want, final = linear_attention(q, k, v, d, initial_state=s, return_state=True)
    n = T * H * K
    buffer = torch.empty(2 ** 31 + 3 * n, dtype=dt, device="cuda")
    far = []
    for i, t in enumerate((q, k, v)):
        view = buffer.as_strided((B, T, H, K), (2 ** 31, H * K, K, 1), i * n)
        view.copy_(t)
        far.append(view)
    o, end = linear_attention(*far, d, initial_state=s, return_state=True)
    assert torch.equal(o, want) and torch.equal(end, final)
    del buffer, far
    cache = torch.empty(2 ** 31 + H * K * V, device="cuda").as_strided((B, H, K, V), (2 ** 31, K * V, V, 1))
    cache.copy_(s)
    dense = s.clone()
    x = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], d[:, 0], dense)
    y = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], d[:, 0], cache)
    assert torch.equal(x, y) and torch.equal(cache, dense)


def test_norm_and_clipping_beyond_32_bits():
    N, C = 2 ** 24 + 3, 128
    x = torch.empty(N, C, dtype=BF, device="cuda")
    x[:1000].normal_()
    x[1000:-1000] = 1.0
    x[-1000:].normal_()
    w = torch.randn(C, device="cuda")
    y = group_norm(x, 4, w, act="silu")
    assert torch.equal(y[-1000:], group_norm(x[-1000:].clone(), 4, w, act="silu")) and torch.equal(y[:1000], group_norm(x[:1000].clone(), 4, w, act="silu"))
    del y
    # two images of 2^30 elements: the second as it is alone (but for a step of bf16 where the last bit of a sum differs)
    a = torch.empty(2, 2 ** 24, 64, dtype=BF, device="cuda").normal_()
    leaf = a.detach().requires_grad_(True)
    y = group_norm(leaf, 8, eps=0.0)
    alone = group_norm(a[1:], 8, eps=0.0)
    assert float((y[1, -2000:].detach().float() - alone[0, -2000:].float()).abs().max()) < 0.05
    dy = torch.zeros_like(y)
    dy[1, -1] = 1.0
    dx, = torch.autograd.grad(y, leaf, dy)
    assert not dx[0].any() and bool(dx[1, -1].any())
    del y, dy, dx, alone, leaf
    flat = x.view(-1)
    total = torch.sqrt(sum(c.double().square().sum() for c in flat.split(2 ** 26)))
    head, tail = flat[:100].clone(), flat[-100:].clone()
    norm = clip_norm_(x, 0.25 * float(total))
    assert abs(float(norm / total) - 1) < 1e-6
    for got, was in ((flat[:100], head), (flat[-100:], tail)):
        assert float((got.double() - 0.25 * was.double()).abs().max()) <= 2.0 ** -8 * 0.25 * float(was.double().abs().max())


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("T,G", [(300, 2), (1100, 1)])
def test_captured_backward(dt, T, G):
    """Forward and backward in two graphs, replayed in turn with other inputs (workspaces are each graph's own)."""
    first, second = make(2, T, 2, G, 64, 128, dt, state=True), make(2, T, 2, G, 64, 128, dt, state=True, seed=4)
    d_o = torch.randn(first[2].shape, device="cuda").to(dt)

    def call(leaves):
        o, final = linear_attention(*leaves[:4], initial_state=leaves[4], return_state=True)
        grads = torch.autograd.grad((o, final), leaves, (d_o, torch.ones_like(final)))
        return [o.detach(), final.detach(), *grads]
    leaf = lambda args: [t.clone().requires_grad_(True) for t in args[:5]]  # noqa: E731
    want = [call(leaf(first)), call(leaf(second))]
    static = leaf(first)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    torch.cuda.synchronize()
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(call(static))
    for args, expect in ((second, want[1]), (first, want[0]), (second, want[1])):
        with torch.no_grad():
            for t, x in zip(static, args):
                t.copy_(x)
        for g in graphs:
            g.replay()
        for o in outs:
            assert all(torch.equal(x, y) for x, y in zip(o, expect))


def test_two_streams_at_once():
    """Calls of all operators under way on two streams beside each other."""
    args = [make(2, 1100, 2, 2, 128, 64, BF, state=True, seed=i) for i in range(2)]
    x = [torch.randn(8, 900, 64, device="cuda") for _ in range(2)]

    def call(i):
        leaves = [t.clone().requires_grad_(True) for t in args[i][:5]] + [x[i].clone().requires_grad_(True)]
        o = linear_attention(*leaves[:4], initial_state=leaves[4])
        y = group_norm(leaves[5], 8, act="gelu")
        grads = torch.autograd.grad((o, y), leaves, (torch.ones_like(o), x[i]))
        norm = clip_norm_([g.contiguous() for g in grads], 1.0)
        return [o.detach(), y.detach(), norm, *grads]
    want = [call(0), call(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[i]))


def test_gradients_of_gradients_are_refused():
    q, k, v, d, _, _ = make(1, 20, 2, 2, 16, 16, F32)
    q.requires_grad_(True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(linear_attention(q, k, v, d).sum(), q, create_graph=True)
    x = torch.randn(2, 10, 16, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(group_norm(x, 4).square().sum(), x, create_graph=True)


def test_a_training_step_with_clipped_gradients():
    """``train_step(max_grad_norm=...)`` is a step without it whose gradients are scaled in between."""
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Flatten(), torch.nn.Linear(48, 32), torch.nn.GELU(), torch.nn.Linear(32, 5)).cuda()
    x, labels = torch.randn(6, 3, 4, 4, device="cuda"), torch.randint(5, (6,), device="cuda")
    nets = [copy.deepcopy(model) for _ in range(2)]
    opts = [torch.optim.SGD(n.parameters(), lr=0.5) for n in nets]
    losses = [refmodel.train_step(nets[0], opts[0], x, labels, 3, autocast_dtype=None, max_grad_norm=0.05),
              refmodel.train_step(nets[1], opts[1], x, labels, 3, autocast_dtype=None)]
    assert torch.equal(*losses)
    grads = [p.grad for p in nets[1].parameters()]
    total = float(torch.sqrt(sum(g.double().square().sum() for g in grads)))
    assert total > 0.05
    for old, p, g in zip(model.parameters(), nets[0].parameters(), grads):
        want = old.detach().double() - 0.5 * (0.05 / (total + 1e-6)) * g.double()
        assert float((p.detach().double() - want).abs().max()) < 1e-6


@pytest.mark.parametrize("dt", [F32, BF])
def test_a_thread_that_has_not_used_the_gpu(dt):
    """A call that allocates nothing new is the first thing a thread does with the device (an autograd thread's first
    backward pass, a server's worker)."""
    import threading
    args = make(2, 700, 2, 1, 64, 64, dt, state=True)
    run = lambda: linear_attention(*args[:4], initial_state=args[4], return_state=True)  # noqa: E731
    want = [t.clone() for t in run()]
    got = []
    thread = threading.Thread(target=lambda: got.extend(run()))
    thread.start()
    thread.join()
    assert len(got) == 2 and all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("B,T,H,G,K,V", [(2, 1000, 4, 4, 128, 128), (2, 1500, 4, 1, 48, 64)])
def test_the_decays_gradient_of_bf16_tensors_has_fp32s_precision(B, T, H, G, K, V):
    """It is float32: 1e-5 of its 2-norm (split products leave 2^-21 of each of up to 512 dots, whose sum is some tenth of
    their magnitude), whatever the tensors are rounded to."""
    q, k, v, d, s, _ = make(B, T, H, G, K, V, BF, state=True)
    d_o = torch.randn(v.shape, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(BF)
    leaf = d.clone().requires_grad_(True)
    got, = torch.autograd.grad(linear_attention(q, k, v, leaf, initial_state=s), leaf, d_o)
    _, _, want = seq_ref.attention_grads(q, k, v, d, K ** -0.5, s, None, d_o, None)
    assert float((got.double() - want[3]).norm() / want[3].norm()) < 1e-5
