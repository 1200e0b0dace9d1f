"""The operators as they are used together: a model of pre-norm recurrent layers (residual sum and layer norm, projections, gated recurrence) and
a head, trained for a step against a teacher's top logits and the labels, and the same model serving a prompt and single tokens."""
import pytest
import torch

import layer_ref
from mamba2d_b200 import clip_grad_norm_, distillation_loss, gated_recurrence, gated_recurrence_step, layer_norm

pytestmark = pytest.mark.gpu
E, LAYERS, CLASSES = 64, 3, 300


def params(seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    p = {"head": n(CLASSES, E) * E ** -0.5, "w": 1 + 0.1 * n(E), "b": 0.1 * n(E)}
    for k in range(LAYERS):
        p.update({f"in{k}": n(2 * E, E) * E ** -0.5, f"gate{k}": 6 * torch.rand(E, generator=g) - 1, f"out{k}": n(E, E) * E ** -0.5, f"w{k}": 1 + 0.1 * n(E), f"b{k}": 0.1 * n(E)})
    return p


def model(p, x, norm, recurrence):
    """x (..., E); norm(h, w, b, stream) gives the normalised and the new stream, recurrence(layer, u, gate) all states."""
    stream, h = torch.zeros_like(x), x
    for k in range(LAYERS):
        y, stream = norm(h, p[f"w{k}"], p[f"b{k}"], stream)
        u, gate = (y @ p[f"in{k}"].t()).split(E, -1)
        h = recurrence(k, u, gate + p[f"gate{k}"]) @ p[f"out{k}"].t()
    y, _ = norm(h, p["w"], p["b"], stream)
    return y @ p["head"].t()


def exact_model(p, x):
    return model(p, x, lambda h, w, b, s: (layer_ref.norm(h + s, w, b), h + s), lambda k, u, g: layer_ref.recurrence(u, g, "forget")[0])


def own_model(p, x):
    return model(p, x, lambda h, w, b, s: layer_norm(h, w, b, residual=s), lambda k, u, g: gated_recurrence(u, g, form="forget"))


def test_a_training_step():
    """fp32: loss and every gradient against autograd in 64 bits; 1e-4 of the largest value, a hundred times what single operators are off by, for
    what three layers and a norm of small values amplify."""
    g = torch.Generator().manual_seed(1)
    x, teacher, labels = torch.randn(3, 200, E, generator=g).cuda(), torch.randn(3, 200, CLASSES, generator=g).cuda(), torch.randint(-1, CLASSES, (3, 200), generator=g).cuda()
    top, index = teacher.topk(12, -1)
    own = {k: torch.nn.Parameter(v.cuda()) for k, v in params().items()}
    ref = {k: v.cuda().double().requires_grad_(True) for k, v in params().items()}
    loss = distillation_loss(own_model(own, x), top, index, labels, temperature=2.0, label_weight=0.5).mean()
    loss.backward()
    want = layer_ref.distillation(exact_model(ref, x.double()).flatten(0, 1), top.flatten(0, 1), index.flatten(0, 1), labels.flatten(), 2.0, 0.5).mean()
    grads = torch.autograd.grad(want, list(ref.values()))
    assert abs(float(loss.detach()) / float(want.detach()) - 1) < 1e-5
    for p, d in zip(own.values(), grads):
        assert float((p.grad.double() - d).abs().max() / d.abs().max()) < 1e-4
    assert abs(float(clip_grad_norm_(own.values(), 1e-3)) / float(torch.sqrt(sum(d.square().sum() for d in grads))) - 1) < 1e-4
    torch.optim.AdamW(own.values(), lr=1e-3).step()
    assert all(bool(torch.isfinite(p).all()) for p in own.values())


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_a_prompt_and_the_tokens_behind_it(dt):
    """bf16: four roundings a layer (norm, projections, recurrence), 13 in all, each half a step of 2^-8 of its values, and three norms that keep their scale."""
    p = {k: v.cuda().to(dt) if v.dim() == 2 or k.startswith("gate") else v.cuda() for k, v in params().items()}
    x = torch.randn(2, 90, E, generator=torch.Generator().manual_seed(3)).cuda().to(dt)
    want = exact_model({k: v.double() for k, v in p.items()}, x.double())
    states = [None] * LAYERS

    def prompt(k, u, gate):
        h, states[k] = gated_recurrence(u, gate, form="forget", return_state=True)
        return h
    norm = lambda h, w, b, s: layer_norm(h, w, b, residual=s)  # noqa: E731
    with torch.no_grad():
        outs = [model(p, x[:, :70], norm, prompt)]
        for t in range(70, 90):
            outs.append(model(p, x[:, t], norm, lambda k, u, gate: gated_recurrence_step(u, gate, states[k], form="forget"))[:, None])
    got = torch.cat(outs, 1)
    assert float((got.double() - want).norm() / want.norm()) < (1e-5 if dt == torch.float32 else 13 * 2.0 ** -8)
