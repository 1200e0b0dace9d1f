"""Definitions in 64 bits of the gated recurrence, the layer norm and the distillation loss, and bounds on what their results may be off by.

The recurrence's weights are all positive, so what rounding does to h_t is bounded by the same operator on magnitudes, H_t = a_t H_{t-1} + |u_t|:
  - a run's tokens (up to 16) are weighted by products of up to 16 gates, each off by 2^-22 of itself (the approximate exponential's and
    reciprocal's error, and the gate's own rounding), and what is carried from run to run by the sum of their logarithms: 2^-17 of H_t covers
    both, twice;
  - every token's state is rounded once, and twice more where runs are joined: 1.25 * 2^-24 of H_t, each carried on like a state.
"""
import torch


def terms(x, gate, form):
    return (gate.exp(), x) if form == "decay" else (gate.sigmoid(), x * (-gate).sigmoid())


def scan(a, u, state=None, lengths=None):
    """(h, final state), token by token."""
    B, T, C = u.shape
    h = torch.zeros(B, C, dtype=u.dtype, device=u.device) if state is None else state
    out = []
    for t in range(T):
        new = a[:, t] * h + u[:, t]
        if lengths is not None:
            inside = (lengths > t)[:, None]
            h = torch.where(inside, new, h)
            out.append(torch.where(inside, new, 0.0))
        else:
            h = new
            out.append(new)
    return torch.stack(out, 1), h


def recurrence(x, gate, form, state=None, lengths=None):
    if lengths is not None:              # rows behind a sequence may hold anything
        live = (torch.arange(x.shape[1], device=x.device) < lengths[:, None])[..., None]
        x, gate = torch.where(live, x, 0.0), torch.where(live, gate, 0.0)
    return scan(*terms(x, gate, form), state, lengths)


def rounded(a, H, lengths=None):
    """The bound above, for states of magnitude H."""
    return 2.0 ** -17 * H + 1.25 * 2.0 ** -24 * scan(a, H, None, lengths)[0]


def recurrence_bounds(x, gate, form, state, lengths, dy=None, d_state=None):
    """Bounds on h (and, with dy, on dx, dgate and the state's gradient), in the order of ``h, final, dx, dgate, dstate``."""
    if lengths is not None:
        live = (torch.arange(x.shape[1], device=x.device) < lengths[:, None])[..., None]
        x, gate = torch.where(live, x, 0.0), torch.where(live, gate, 0.0)
        dy = None if dy is None else torch.where(live, dy, 0.0)
    a, u = terms(x, gate, form)
    state = torch.zeros_like(x[:, 0]) if state is None else state.abs()
    H, last = scan(a, u.abs(), state, lengths)
    h = rounded(a, H, lengths)
    n = torch.full((x.shape[0],), x.shape[1], device=x.device) if lengths is None else lengths
    final = torch.where((n > 0)[:, None], h[torch.arange(len(h), device=h.device), (n - 1).clamp(min=0)], 0.0)
    if dy is None:
        return h, final
    if lengths is not None:              # (rows behind a sequence pass the state's gradient on)
        a = torch.where(live, a, 1.0)
    D = scan(torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), 1).flip(1), torch.cat((dy[:, :-1].abs(), dy[:, -1:].abs() + (0 if d_state is None else d_state.abs()[:, None])), 1).flip(1))[0].flip(1)
    dD = rounded(torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), 1).flip(1), D.flip(1)).flip(1)
    before, dbefore = torch.cat((state[:, None], H[:, :-1]), 1), torch.cat((torch.zeros_like(h[:, :1]), h[:, :-1]), 1)
    if form == "decay":
        dx, dg = dD, a * (dD * before + D * dbefore)
    else:
        rest = (-gate).sigmoid()
        dx, dg = rest * dD, a * rest * (dD * (before + x.abs()) + D * dbefore)
    # (the gates' own factors: four of them, each off by 2^-21 at most)
    dx = dx + 2.0 ** -19 * D
    dg = dg + 2.0 ** -19 * a * D * (before + x.abs())
    return h, final, dx, dg, a[:, 0] * (dD[:, 0] + 2.0 ** -19 * D[:, 0])


def within(got, want, bound):
    """Largest error over (bound + the result's own rounding); infinite where one is not finite and the other is."""
    assert got.shape == want.shape, (got.shape, want.shape)
    if not got.numel():
        return 0.0
    if not bool(torch.isfinite(got).all()):
        return float("inf")
    allowed = bound + torch.finfo(got.dtype).eps / 2 * want.abs() + 1e-36
    return float(((got.double() - want).abs() / allowed).max())


def norm(x, weight, bias, eps=1e-5):
    d = x - x.mean(-1, keepdim=True)
    h = d / (d.square().mean(-1, keepdim=True) + eps).sqrt()
    return (h if weight is None else h * weight) + (0.0 if bias is None else bias)


def norm_bounds(x, weight, bias, dy=None, eps=1e-5):
    """What (y, dx, dw, db) may be off by before their own rounding, in steps e = 2^-24.  A sum of C values has k = 64 + C / 512 roundings on a
    value's way (a thread's share, then a tree); the mean is taken about the first value, so its error is that of a mean of
    distances from it; h is off by the mean's error and by some 3 k / 2 steps of its own."""
    e, C, N = 2.0 ** -24, x.shape[-1], x.numel() // x.shape[-1]
    k = 64 + C / 512
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = 1 / (d.square().mean(-1, keepdim=True) + eps).sqrt()
    w = torch.ones_like(x[..., :1]) if weight is None else weight
    off_mean = k * e * (x - x[..., :1]).abs().mean(-1, keepdim=True) + 2 * e * mean.abs()
    h = d * rstd
    dh = rstd * off_mean + 2 * k * e * h.abs()
    y = w.abs() * dh + 4 * e * ((h * w).abs() + (0.0 if bias is None else bias.abs()))
    if dy is None:
        return y
    g = dy * w
    m0, m1 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    off0 = k * e * g.abs().mean(-1, keepdim=True)
    off1 = k * e * (g * h).abs().mean(-1, keepdim=True) + (g.abs() * dh).mean(-1, keepdim=True)
    dx = rstd * (off0 + h.abs() * off1 + dh * m1.abs()) + (k + 8) * e * rstd * (g.abs() + m0.abs() + (h * m1).abs())
    rows = 64 + N / 32                   # (a thread's rows one after another, then CTAs in turn)
    over = lambda t: t.reshape(-1, C).sum(0)  # noqa: E731
    return y, dx, over(dy.abs() * dh) + rows * e * over((dy * h).abs()), rows * e * over(dy.abs())


def distillation(z, t, index, labels=None, temperature=1.0, label_weight=0.0):
    """A loss a row, z (N, V) in 64 bits."""
    tau, w, V = temperature, label_weight, z.shape[-1]
    there = (index >= 0) & (index < V)
    at = torch.where(there, index, 0).long()
    t = torch.where(there, t.double(), -torch.inf)
    teaches = (t > -torch.inf).any(-1) | torch.isnan(t).any(-1)
    log_p = torch.log_softmax(torch.where(teaches[:, None], t, 0.0) / tau, -1)
    log_q = torch.log_softmax(z / tau, -1).gather(-1, at)
    p = torch.where(there, log_p.exp(), 0.0)
    kl = torch.where(p != 0, p * (torch.where(p != 0, log_p, 0.0) - torch.where(p != 0, log_q, 0.0)), 0.0).sum(-1)
    loss = (1 - w) * tau ** 2 * torch.where(teaches, kl, 0.0) if w < 1 else torch.zeros_like(kl)
    if w > 0:
        counted = (labels >= 0) & (labels < V)
        label = torch.where(counted, labels, 0).long()
        loss = loss - w * torch.where(counted, torch.log_softmax(z, -1).gather(-1, label[:, None])[:, 0], 0.0)
    return loss


def distillation_bounds(z, t, index, labels, temperature, label_weight, up):
    """What (loss, dz) may be off by.  An exponential's argument (z - max) c is rounded twice and c = log2(e) / tau once, so it is off by
    2^-22 of itself at most, the approximate exponential by 2^-22, and a row's sum by k more steps of 2^-24, k the values that a thread adds and
    a tree above it."""
    tau, w, V = temperature, label_weight, z.shape[-1]
    k = 32 + max(V / 256, min(V, 4096) / 32)
    base = 2.0 ** -21 + k * 2.0 ** -24
    far = torch.where(torch.isfinite(z), z.max(-1, keepdim=True).values - z, 0.0).clamp(max=2e3)
    there = (index >= 0) & (index < V)
    at = torch.where(there, index, 0).long()
    p = torch.nan_to_num(torch.softmax(torch.where(there, t.double(), -1e30) / tau, -1)) * there         # (of a list of -inf: nothing)
    spread = 2.0 ** -22 * (far.gather(-1, at) * there).max(-1).values / tau + 2.0 ** -22 * torch.where(there & torch.isfinite(t), t.double().abs(), 0.0).max(-1).values / tau
    loss = (1 - w) * tau ** 2 * (base + spread) + w * (base + 2.0 ** -22 * (0 if labels is None else far.gather(-1, labels.clamp(0, V - 1).long()[:, None])[:, 0]))
    q, s = torch.softmax(z / tau, -1), torch.softmax(z, -1)
    dz = (1 - w) * tau * q * (2 * base + 2.0 ** -21 * far / tau) + w * s * (2 * base + 2.0 ** -21 * far)
    take = torch.zeros_like(z).scatter_add_(-1, at, p * (8 * 2.0 ** -22 + 2.0 ** -21 * torch.where(there & torch.isfinite(t), (t.double().max() - t.double()).abs().clamp(max=2e3), 0.0) / tau))
    dz = dz + (1 - w) * tau * take + 2.0 ** -22 * (w + tau * (1 - w)) * (q + s) + 2.0 ** -23 * (torch.zeros_like(z).scatter_add_(-1, at, (1 - w) * tau * p))
    if labels is not None:
        inside = (labels >= 0) & (labels < V)
        dz.scatter_add_(-1, labels.clamp(0, V - 1).long()[:, None], (2.0 ** -22 * w * inside)[:, None].double())
    return loss, up.abs()[:, None] * dz
