"""Calls of the gated recurrence, the layer norm and the distillation loss that their documentation allows and ordinary use seldom makes: captured
calls, two streams at once, offsets beyond 32 bits, the same tensor twice, gradients of some inputs only, changed inputs, repeated calls."""
import pytest
import torch

import layer_ref
from mamba2d_b200 import distillation_loss, gated_recurrence, gated_recurrence_step, layer_norm

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16


def rand(*shape, seed=0, dt=F32):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dt)


def calls(seed, dt=BF):
    """name -> (function of its tensors, tensors of which the first two get gradients where there are two, upstream gradient's shape)."""
    x, g = rand(2, 3000, 128, seed=seed, dt=dt), (rand(2, 3000, 128, seed=seed + 1) + 3).to(dt)
    y, r, w = rand(700, 1000, seed=seed + 2, dt=dt), rand(700, 1000, seed=seed + 3, dt=dt), 1 + 0.1 * rand(1000, seed=seed + 4)
    z, index = rand(5, 30001, seed=seed + 5, dt=dt), torch.randint(0, 30001, (5, 16), generator=torch.Generator().manual_seed(seed)).cuda()
    t = rand(5, 16, seed=seed + 6)
    short, s_index = rand(50, 600, seed=seed + 7, dt=dt), index[:, :8].repeat(10, 1) % 600
    return {"recurrence": (lambda a, b: gated_recurrence(a, b, form="forget"), [x, g]), "norm": (lambda a, b, r: layer_norm(a, b, residual=r)[0], [y, w, r]),
            "distill": (lambda a: distillation_loss(a, t, index, temperature=1.5), [z]),
            "distill_short": (lambda a: distillation_loss(a, t.repeat(10, 1)[:, :8], s_index, index[:, 0].repeat(10), temperature=2.0, label_weight=0.5), [short])}


@pytest.mark.parametrize("name", ["recurrence", "norm", "distill", "distill_short"])
@pytest.mark.parametrize("dt", [F32, BF])
def test_captured_calls(name, dt):
    """Forward and backward passes in two graphs that share a pool and are replayed in turn, with new inputs: the bits of eager calls."""
    f, tensors = calls(0, dt)[name]
    _, others = calls(50, dt)[name]

    def once(f, leaves, up):
        leaves = [t.detach().clone().requires_grad_(True) for t in leaves]
        out = f(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, up)]
    up = rand(*f(*tensors).shape, seed=9, dt=f(*tensors).dtype)
    want, wanted = once(f, tensors, up), once(f, others, up)
    pool, made = None, []
    for _ in range(2):
        static = [t.clone() for t in tensors]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            once(f, static, up)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs = once(f, static, up)
        pool = graph.pool()
        made.append((graph, static, outs))
    for turn in range(3):
        for k, (graph, static, outs) in enumerate(made):
            source, expected = ((tensors, want), (others, wanted))[(turn + k) % 2]
            for a, b in zip(static, source):
                a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, expected)), (turn, k)


def test_a_captured_token():
    x, g, s = rand(3, 100, seed=1), rand(3, 100, seed=2), rand(3, 100, seed=3)
    eager, state = s.clone(), s.clone()
    graph = torch.cuda.CUDAGraph()
    gated_recurrence_step(x, g, s.clone(), form="forget")
    with torch.cuda.graph(graph):
        out = gated_recurrence_step(x, g, state, form="forget")
    state.copy_(s)
    for k in range(4):
        x.normal_()
        want = gated_recurrence_step(x, g, eager, form="forget")
        graph.replay()
        assert torch.equal(out, want) and torch.equal(state, eager)


def test_two_streams_at_once():
    """Different calls side by side, many times over: the bits of calls one after another."""
    work = [(*calls(k)[n], n) for k, n in ((0, "recurrence"), (20, "norm"), (40, "distill"), (60, "recurrence"))]

    def once(f, tensors):
        leaves = [t.detach().requires_grad_(True) for t in tensors]
        out = f(*leaves)
        return [out.detach(), *torch.autograd.grad(out.float().sum(), leaves)]
    want = [once(f, t) for f, t, _ in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [[] for _ in work]
    for _ in range(5):
        for k, (f, t, _) in enumerate(work):
            with torch.cuda.stream(streams[k]):
                got[k].append(once(f, t))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for one in a for x, y in zip(one, b))


@pytest.mark.parametrize("name", ["recurrence", "norm", "distill", "distill_short"])
def test_the_same_bits_every_time(name):
    f, tensors = calls(3)[name]
    first = None
    for _ in range(10):
        leaves = [t.detach().requires_grad_(True) for t in tensors]
        out = f(*leaves)
        now = [out.detach(), *torch.autograd.grad(out.float().square().sum(), leaves)]
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


@pytest.mark.parametrize("dt", [F32, BF])
def test_offsets_beyond_32_bits(dt):
    """Sequences, rows and states 2^31 elements apart: the bits of neighbouring ones (the recurrence by TMA and by plain loads)."""
    far = 2 ** 31
    buffer = torch.empty(far + 3 * 2 ** 20, dtype=dt, device="cuda")
    for T, C in ((5000, 64), (700, 63)):
        x, g, dy = rand(2, T, C, seed=1, dt=dt), (rand(2, T, C, seed=2) + 2).to(dt), rand(2, T, C, seed=3, dt=dt)
        views = []
        for i, t in enumerate((x, g, dy)):
            view = buffer.as_strided((2, T, C), (far, C, 1), i * 2 ** 20)
            view.copy_(t)
            views.append(view)
        assert torch.equal(gated_recurrence(views[0], views[1], form="forget"), gated_recurrence(x, g, form="forget"))
        a, b = (torch.autograd.grad(gated_recurrence(*leaves, form="forget"), leaves, up) for leaves, up in
                (([t.detach().requires_grad_(True) for t in views[:2]], views[2]), ([t.detach().requires_grad_(True) for t in (x, g)], dy)))
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    for C in (320, 1001, 9000):
        x, dy = rand(2, C, seed=4, dt=dt), rand(2, C, seed=5, dt=dt)
        views = [buffer.as_strided((2, C), (far, 1), 2 ** 20 * i) for i in range(2)]
        views[0].copy_(x)
        views[1].copy_(dy)
        one, two = views[0].detach().requires_grad_(True), x.detach().requires_grad_(True)
        y, w = layer_norm(one), layer_norm(two)
        assert torch.equal(y, w) and torch.equal(torch.autograd.grad(y, one, views[1])[0], torch.autograd.grad(w, two, dy)[0])
    for V in (1000, 40000):
        z, t, index = rand(2, V, seed=6, dt=dt), rand(2, 9, seed=7), torch.randint(0, V, (2, 9)).cuda()
        view = buffer.as_strided((2, V), (far, 1), 0)
        view.copy_(z)
        one, two = view.detach().requires_grad_(True), z.detach().requires_grad_(True)
        a, b = distillation_loss(one, t, index), distillation_loss(two, t, index)
        assert torch.equal(a, b) and torch.equal(torch.autograd.grad(a.sum(), one)[0], torch.autograd.grad(b.sum(), two)[0])
    del buffer, views, view, one
    cache = torch.empty(far + 64, device="cuda").as_strided((2, 64), (far, 1), 0)
    s = rand(2, 64, seed=8)
    cache.copy_(s)
    x, g = rand(2, 64, seed=9), rand(2, 64, seed=10)
    assert torch.equal(gated_recurrence_step(x, g, cache, form="forget"), gated_recurrence_step(x, g, s, form="forget")) and torch.equal(cache, s)


def test_outputs_beyond_32_bits():
    """More than 2^31 values in one call, forward and backward; the last rows against 64 bits."""
    N, C = 300000, 7200
    x = torch.empty(N, C, dtype=BF, device="cuda").normal_()
    leaf = x.requires_grad_(True)
    y = layer_norm(leaf)
    last = x[-3:].detach().double()
    assert layer_ref.within(y[-3:].detach(), layer_ref.norm(last, None, None), layer_ref.norm_bounds(last, None, None)) <= 1
    dx, = torch.autograd.grad(y, leaf, x.detach())
    _, bound, _, _ = layer_ref.norm_bounds(last, None, None, last)
    ref = last.clone().requires_grad_(True)
    want, = torch.autograd.grad(layer_ref.norm(ref, None, None), ref, last)
    assert layer_ref.within(dx[-3:], want, bound) <= 1
    del x, y, dx, leaf
    N, V = 20000, 110001
    z = torch.empty(N, V, dtype=BF, device="cuda").normal_().requires_grad_(True)
    t, index, up = rand(N, 4, seed=1), torch.randint(0, V, (N, 4)).cuda(), torch.ones(N, device="cuda")
    loss = distillation_loss(z, t, index)
    dz, = torch.autograd.grad(loss, z, up)
    ref = z[-3:].detach().double().requires_grad_(True)
    want = layer_ref.distillation(ref, t[-3:], index[-3:])
    grad, = torch.autograd.grad(want, ref, up[-3:].double())
    bounds = layer_ref.distillation_bounds(ref.detach(), t[-3:], index[-3:], None, 1.0, 0.0, up[-3:].double())
    assert layer_ref.within(loss[-3:].detach(), want.detach(), bounds[0]) <= 1 and layer_ref.within(dz[-3:], grad, bounds[1]) <= 1
    del z, dz
    x = torch.ones(1, 40000, 56000, dtype=BF, device="cuda")
    h = gated_recurrence(x, torch.full((1,), -torch.log(torch.tensor(2.0)).item(), device="cuda", dtype=BF).expand_as(x))
    a = torch.exp(torch.full((), -torch.log(torch.tensor(2.0)).item()).bfloat16().double())
    assert float((h[0, -1].double() - 1 / (1 - a).cuda()).abs().max()) <= 2.0 ** -7 and bool((h[0, 0] == 1).all())


def test_the_same_tensor_twice():
    x = rand(2, 300, 64, seed=1).clamp(max=0)
    leaf, a, b = (x.clone().requires_grad_(True) for _ in range(3))
    dy = rand(2, 300, 64, seed=2)
    both, = torch.autograd.grad(gated_recurrence(leaf, leaf), leaf, dy)
    da, db = torch.autograd.grad(gated_recurrence(a, b), (a, b), dy)
    assert torch.equal(both, da + db)
    y, s = layer_norm(leaf, residual=leaf)
    dx, = torch.autograd.grad(y, leaf, dy)
    y2, _ = layer_norm(a, residual=b)
    da, db = torch.autograd.grad(y2, (a, b), dy)
    assert torch.equal(y, y2) and torch.equal(dx, da + db)


def test_some_gradients_and_none():
    x, g, s, dy = rand(2, 300, 64, seed=1), rand(2, 300, 64, seed=2), rand(2, 64, seed=3), rand(2, 300, 64, seed=4)
    leaves = [t.clone().requires_grad_(True) for t in (x, g, s)]
    whole = torch.autograd.grad(gated_recurrence(leaves[0], leaves[1], form="forget", initial_state=leaves[2]), leaves, dy)
    for k in range(3):
        args = [t.clone() for t in (x, g, s)]
        args[k].requires_grad_(True)
        h, last = gated_recurrence(args[0], args[1], form="forget", initial_state=args[2], return_state=True)
        assert torch.equal(torch.autograd.grad(h, args[k], dy, retain_graph=True)[0], whole[k])
        via_state, = torch.autograd.grad(last, args[k], rand(2, 64, seed=5))       # no gradient of h at all
        # (of the first state 300 gates of about a half leave nothing: 2^-300 is below fp32's smallest number)
        assert bool(torch.isfinite(via_state).all()) and (k == 2 or bool((via_state != 0).any()))
    with torch.inference_mode():
        h = gated_recurrence(x, g, form="forget")
        state = torch.zeros(2, 64, device="cuda")
        assert torch.equal(gated_recurrence_step(x[:, 0], g[:, 0], state, form="forget"), h[:, 0]) and layer_norm(x).shape == x.shape
    with torch.no_grad():
        assert not gated_recurrence(*leaves[:2]).requires_grad
    with pytest.raises(RuntimeError, match="no gradients"):
        gated_recurrence_step(leaves[0][:, 0], g[:, 0], s.clone())


def test_inputs_that_change_before_the_backward_pass_are_found():
    x, g = (rand(2, 100, 64, seed=k).requires_grad_(True) for k in (1, 2))
    for f in (lambda: gated_recurrence(x, g, form="forget"), lambda: layer_norm(x), lambda: distillation_loss(x, rand(2, 100, 3), torch.zeros(2, 100, 3, dtype=torch.long, device="cuda"))):
        out = f()
        with torch.no_grad():
            x.mul_(1.5)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()
    y, s = layer_norm(x, residual=x.detach())
    s.detach().add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_of_gradients_are_refused():
    x, g = (rand(1, 70, 64, seed=k).requires_grad_(True) for k in (1, 2))
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(gated_recurrence(x, g).sum(), x, create_graph=True)


def test_a_thread_that_has_not_used_the_gpu():
    import threading
    x, g = rand(2, 3000, 128, seed=1, dt=BF), rand(2, 3000, 128, seed=2, dt=BF)
    want = gated_recurrence(x, g, form="forget")
    got = []
    thread = threading.Thread(target=lambda: got.append((gated_recurrence(x, g, form="forget"), layer_norm(x), distillation_loss(x[0], rand(3000, 3), torch.zeros(3000, 3, dtype=torch.long, device="cuda")))))
    thread.start()
    thread.join()
    assert torch.equal(got[0][0], want)
