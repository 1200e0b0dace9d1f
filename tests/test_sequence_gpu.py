"""The sequence operators as they are used together: a layer (projections, linear attention, norm over the heads with SiLU,
output projection) trained for a step with clipped gradients, and the same layer serving a prompt and single tokens."""
import pytest
import torch

import seq_ref
from mamba2d_b200 import clip_grad_norm_, group_norm, linear_attention, linear_attention_step

pytestmark = pytest.mark.gpu
H, G, D, E = 4, 2, 32, 64


def params(seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"qkv": n(G * D * 2 + H * D, E) * E ** -0.5, "rate": n(H) * 0.3 - 2, "step": n(H, E) * E ** -0.5, "w": 1 + 0.1 * n(H * D), "b": 0.1 * n(H * D),
            "out": n(E, H * D) * (H * D) ** -0.5}


def layer(p, x, attention, norm):
    B, T, _ = x.shape
    q, k, v = (x @ p["qkv"].t()).split([G * D, G * D, H * D], -1)
    decay = -torch.nn.functional.softplus(x @ p["step"].t()) * torch.exp(p["rate"])
    o = attention(q.view(B, T, G, D), k.view(B, T, G, D), v.view(B, T, H, D), decay)
    return norm(o.reshape(B * T, H * D), p["w"], p["b"]).view(B, T, H * D) @ p["out"].t()


def exact_layer(p, x):
    return layer(p, x, lambda q, k, v, d: seq_ref.attention(q, k, v, d, D ** -0.5)[0], lambda o, w, b: seq_ref.norm(o, H, w, b, 1e-5, "silu"))


def own_layer(p, x):
    return layer(p, x, linear_attention, lambda o, w, b: group_norm(o, H, w, b, act="silu"))


def test_a_training_step():
    """fp32: loss, gradients, norm and the clipped update against autograd in 64 bits; 1e-4 of the largest value, a hundred
    times what single operators are off by and what a norm of small values amplifies."""
    x, y = torch.randn(3, 200, E, generator=torch.Generator().manual_seed(1)).cuda(), torch.randn(3, 200, E, generator=torch.Generator().manual_seed(2)).cuda()
    own = {k: torch.nn.Parameter(v.cuda()) for k, v in params().items()}
    ref = {k: v.cuda().double().requires_grad_(True) for k, v in params().items()}
    loss = (own_layer(own, x) - y).square().mean()
    loss.backward()
    want = (exact_layer(ref, x.double()) - y.double()).square().mean()
    grads = torch.autograd.grad(want, list(ref.values()))
    assert abs(float(loss) / float(want) - 1) < 1e-5
    for p, g in zip(own.values(), grads):
        assert float((p.grad.double() - g).abs().max() / g.abs().max()) < 1e-4
    total = torch.sqrt(sum(g.square().sum() for g in grads))
    bound = 0.5 * float(total)
    norm = clip_grad_norm_(own.values(), bound)
    assert abs(float(norm) / float(total) - 1) < 1e-4
    for p, g in zip(own.values(), grads):
        assert float((p.grad.double() - 0.5 * g).abs().max() / g.abs().max()) < 1e-4
    torch.optim.AdamW(own.values(), lr=1e-3).step()
    assert all(bool(torch.isfinite(p).all()) for p in own.values())


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_a_prompt_and_the_tokens_behind_it(dt):
    p = {k: v.cuda() for k, v in params().items()}
    cast = {k: v.to(dt) if k in ("qkv", "out") else v for k, v in p.items()}
    x = torch.randn(2, 150, E, generator=torch.Generator().manual_seed(3)).cuda().to(dt)
    rounded = {k: v.double() for k, v in cast.items()}
    want = exact_layer(rounded, x.double())
    state = None
    outs = []

    def project(x):
        q, k, v = (x @ cast["qkv"].t()).split([G * D, G * D, H * D], -1)
        decay = -torch.nn.functional.softplus(x.float() @ p["step"].t()) * torch.exp(p["rate"])
        return q.unflatten(-1, (G, D)), k.unflatten(-1, (G, D)), v.unflatten(-1, (H, D)), decay

    def finish(o):
        return group_norm(o.reshape(-1, H * D), H, p["w"], p["b"], act="silu").view(*o.shape[:-2], H * D) @ cast["out"].t()

    with torch.no_grad():
        o, state = linear_attention(*project(x[:, :120]), return_state=True)
        outs.append(finish(o))
        for t in range(120, 150):
            outs.append(finish(linear_attention_step(*project(x[:, t]), state))[:, None])
    got = torch.cat(outs, 1)
    # bf16: projections, attention, norm and output are rounded one after another; the norm amplifies what is small
    assert float((got.double() - want).norm() / want.norm()) < (1e-5 if dt == torch.float32 else 4 * 2.0 ** -8)
