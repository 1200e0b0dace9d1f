"""The sequence operators' definitions in 64 bits, and how far a result may be from them.

For attention the bound is taken element by element.  A product of two values, each off by a share r of itself, is off by
2 r of its magnitude, so a sum of products is off by at most 2 r times the sum of the magnitudes, and that sum is what the
same operator gives for the magnitudes of its inputs (all of its weights are positive).
"""
import torch


def attention(q, k, v, g, scale, state=None, lengths=None):
    """(o, final state) as one product over pairs of tokens; float64 throughout."""
    B, T, H, V = v.shape
    q, k = (t.repeat_interleave(H // t.shape[2], 2).transpose(1, 2) for t in (q, k))
    v, g = v.transpose(1, 2), g.expand(B, T, H).transpose(1, 2)
    live = torch.ones(B, 1, T, dtype=torch.bool, device=v.device)
    if lengths is not None:
        live = (torch.arange(T, device=v.device) < lengths[:, None])[:, None]
    q, k, v = (torch.where(live[..., None], t, 0.0) for t in (q, k, v))
    g = torch.where(live, g.clamp(min=-1e4), 0.0)
    c = g.cumsum(-1)
    later = torch.ones(T, T, dtype=torch.bool, device=v.device).triu(1)
    D = torch.exp((c[..., :, None] - c[..., None, :]).masked_fill(later, -torch.inf))
    o = ((q @ k.transpose(-1, -2)) * D) @ v
    end = c[..., -1:]
    final = (k * torch.exp(end - c)[..., None]).transpose(-1, -2) @ v
    if state is not None:
        o = o + torch.exp(c)[..., None] * (q @ state)
        final = final + torch.exp(end)[..., None] * state
    return (scale * o).transpose(1, 2), final


def attention_grads(q, k, v, g, scale, state, lengths, d_o, d_state):
    leaves = [t.detach().double().requires_grad_(True) if t is not None else None for t in (q, k, v, g, state)]
    o, final = attention(*leaves[:4], scale, leaves[4], lengths)
    outs, ups = [o], [d_o.double()]
    if d_state is not None:
        outs.append(final)
        ups.append(d_state.double())
    if lengths is not None:
        ups[0] = torch.where((torch.arange(v.shape[1], device=v.device) < lengths[:, None])[:, :, None, None], ups[0], 0.0)
    grads = torch.autograd.grad(outs, [t for t in leaves if t is not None], ups)
    it = iter(grads)
    return o.detach(), final.detach(), [next(it) if t is not None else None for t in leaves]


def within(got, want, magnitude, share, rounding):
    """Largest (error / bound): ``share`` of the sum of magnitudes, and the result's own rounding."""
    if not bool(torch.isfinite(got).all()):
        return float("inf")
    bound = share * magnitude.double() + rounding * want.double().abs() + 1e-30
    return float(((got.double() - want.double()).abs() / bound).max())


def norm(x, groups, weight, bias, eps, act):
    N, C = x.shape[0], x.shape[-1]
    f = x.reshape(N, -1, groups, C // groups)
    d = f - f.mean((1, 3), keepdim=True)
    y = (d / (d.square().mean((1, 3), keepdim=True) + eps).sqrt()).reshape(x.shape)
    if weight is not None:
        y = y * weight
    if bias is not None:
        y = y + bias
    return y * torch.sigmoid(y) if act == "silu" else y * torch.special.ndtr(y) if act == "gelu" else y
