"""The gated recurrence per channel (prompts, training, single tokens), layer normalisation with a residual sum, and the
distillation loss against a teacher's top logits, as they are measured.

``run`` computes them in plain form (elementary torch operations in 32 bits, a row's final sums of the loss in 64), or, where
``own`` is set, by the calls that a user makes of this package.  ``exact`` follows the definitions in 64 bits.
"""
import math

import torch

own = False

SCAN_WIDTHS = (64, 96, 128, 192, 320, 384, 512, 576)     # stage widths of the shipped models


def listed():
    def recur(name, kind, B, T, C, dtype, form, state=False, ragged=False):
        return dict(name=name, op="recur", kind=kind, B=B, T=T, C=C, dtype=dtype, form=form, state=state, ragged=ragged)

    def norm(name, kind, N, C, dtype, residual):
        return dict(name=name, op="norm", kind=kind, N=N, C=C, dtype=dtype, residual=residual)

    def distill(name, kind, N, V, K, dtype, temperature, label_weight):
        return dict(name=name, op="distill", kind=kind, N=N, V=V, K=K, dtype=dtype, temperature=temperature, label_weight=label_weight)

    return [
        # one token of one sequence: what a single user's next token waits for
        recur("step_1x1024_bf16", "step", 1, 1, 1024, "bf16", "forget"),
        # four prompts, the state kept for the tokens that follow
        recur("prefill_4x4096x2048_bf16", "prefill", 4, 4096, 2048, "bf16", "forget", state=True),
        # one long prompt of few channels
        recur("prefill_1x65536x512_bf16", "prefill", 1, 65536, 512, "bf16", "decay", state=True),
        # ragged sequences of up to 45x31 pixels, 192 channels, fp32
        recur("train_6x1395x192_f32", "train", 6, 1395, 192, "f32", "decay", ragged=True),
        # a training step's share of one GPU
        recur("train_8x4096x2048_bf16", "train", 8, 4096, 2048, "bf16", "forget"),
        # the tokens of one 14x14 map of 320 channels
        norm("norm_196x320_f32", "infer", 196, 320, "f32", False),
        # batched training, the tokens of 128 maps of 28x28, 320 channels
        norm("norm_100352x320_bf16", "train", 100352, 320, "bf16", False),
        # a wide layer's tokens, with the residual stream
        norm("norm_8192x4096_bf16", "train", 8192, 4096, "bf16", True),
        # a classifier's training batch of 1000 classes, with its labels
        distill("distill_128x1000_f32", "train", 128, 1000, 16, "f32", 2.0, 0.5),
        # eight tokens and a large vocabulary: the loss alone
        distill("distill_8x131072_bf16", "eval", 8, 131072, 64, "bf16", 1.0, 0.0),
        # rows of an odd length, labels beside the teacher
        distill("distill_2047x50001_bf16", "train", 2047, 50001, 20, "bf16", 2.0, 0.25),
        # a training step's tokens with a large vocabulary
        distill("distill_2048x131072_bf16", "train", 2048, 131072, 64, "bf16", 1.0, 0.0),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    kind, dtype = rng.choice(("step", "prefill", "train", "prefill", "train", "norm", "norm", "distill", "distill")), rng.choice(("f32", "bf16"))
    if kind in ("step", "prefill", "train"):
        form = rng.choice(("decay", "forget"))
        C = rng.choice((rng.choice(SCAN_WIDTHS), log_int(16, 4096), 8 * log_int(2, 512)))
        if kind == "step":
            return dict(op="recur", kind=kind, B=log_int(1, 1024), T=1, C=C, dtype=dtype, form=form, state=False, ragged=False)
        B = log_int(1, 64)
        most = (1 << 25) if dtype == "f32" else (1 << 26)          # the listed training step's values
        T = log_int(1, max(1, min(65536, most // (B * C))))
        return dict(op="recur", kind=kind, B=B, T=T, C=C, dtype=dtype, form=form, state=rng.random() < 0.4, ragged=B > 1 and rng.random() < 0.4)
    if kind == "norm":
        C = rng.choice((rng.choice(SCAN_WIDTHS), log_int(16, 8192), 8 * log_int(2, 1024)))
        most = (1 << 24) if dtype == "f32" else (1 << 25)
        return dict(op="norm", kind=rng.choice(("infer", "train", "train")), N=log_int(1, min(1 << 17, most // C)), C=C, dtype=dtype, residual=rng.random() < 0.5)
    V = rng.choice((log_int(10, 131072), 64 * log_int(1, 2048)))
    most = (1 << 27) if dtype == "f32" else (1 << 28)
    weight = rng.choice((0.0, 0.0, 0.25, 0.5, 0.9))
    return dict(op="distill", kind=rng.choice(("eval", "train", "train")), N=log_int(1, min(8192, most // V)), V=V, K=log_int(1, min(V, 128)), dtype=dtype,
                temperature=rng.choice((1.0, 1.0, 2.0, 3.5)), label_weight=weight)


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=g, device="cuda") * (hi - lo) + lo

    return {"case": dict(case), **{"recur": _prepare_recur, "norm": _prepare_norm, "distill": _prepare_distill}[case["op"]](case, normal, uniform)}


def _prepare_recur(case, normal, uniform):
    B, T, C, dt = case["B"], case["T"], case["C"], _dtype(case)
    tokens = (B,) if case["kind"] == "step" else (B, T)
    s = {"x": normal(*tokens, C).to(dt)}
    if case["form"] == "decay":          # a step size for each token, a rate for each channel
        s["gate"] = -(torch.nn.functional.softplus(normal(*tokens, C) * 0.5 - 3.0) * torch.exp(uniform(math.log(0.1), math.log(16.0), C))).to(dt)
    else:                                # channels from a memory of a token to one of some thousand
        s["gate"] = (normal(*tokens, C) + uniform(-2.0, 8.0, C)).to(dt)
    s["state"] = normal(B, C) if case["kind"] == "step" or case["state"] else None
    s["lengths"] = (uniform(0.3, 1.0, B) * T).ceil().to(torch.int32) if case["ragged"] else None
    if case["kind"] == "train":
        s["d_out"] = normal(*tokens, C).to(dt)
        s["d_state"] = normal(B, C) if case["state"] else None
        for n in ("x", "gate", "state"):
            if s[n] is not None:
                s[n].requires_grad_(True)
    return s


def _prepare_norm(case, normal, uniform):
    N, C, dt = case["N"], case["C"], _dtype(case)
    s = {"x": (normal(N, C) * torch.exp(0.5 * normal(N, 1)) + normal(N, 1)).to(dt),      # tokens differ in scale and offset
         "residual": normal(N, C).to(dt) if case["residual"] else None, "weight": 1.0 + 0.1 * normal(C), "bias": 0.1 * normal(C)}
    if case["kind"] == "train":
        s["d_out"] = normal(N, C).to(dt)
        s["d_sum"] = normal(N, C).to(dt) if case["residual"] else None
        for n in ("x", "residual", "weight", "bias"):
            if s[n] is not None:
                s[n].requires_grad_(True)
    return s


def _prepare_distill(case, normal, uniform):
    N, V, K = case["N"], case["V"], case["K"]
    logits = normal(N, V).mul_(2.0)
    teacher = normal(N, V).add_(logits, alpha=0.7)
    top, index = teacher.topk(K, dim=-1)
    del teacher
    # a teacher's list may be shorter than others (its first entries are always there)
    count = (uniform(0.4, 1.4, N) * K).ceil()[:, None]
    index = torch.where(torch.arange(K, device="cuda") < count, index, -1)
    s = {"logits": logits.to(_dtype(case)), "top": top.to(_dtype(case)), "index": index, "labels": None}
    if case["label_weight"] > 0:         # one row in eight has none
        s["labels"] = torch.where(uniform(0, 1, N) < 0.125, -100, (uniform(0, V, N)).long().clamp(max=V - 1))
    if case["kind"] == "train":
        s["logits"].requires_grad_(True)
        s["d_loss"] = torch.full((N,), 1.0 / N, device="cuda") * uniform(0.5, 1.5, N)
    return s


def run(state):
    return {"recur": _run_recur, "norm": _run_norm, "distill": _run_distill}[state["case"]["op"]](state)


def _run_recur(s):
    case = s["case"]
    if case["kind"] == "step":
        if own:
            import mamba2d_b200
            return mamba2d_b200.gated_recurrence_step(s["x"], s["gate"], s["state"], form=case["form"]), s["state"]
        a, u = _plain_terms(s["x"].float(), s["gate"].float(), case["form"])
        s["state"].mul_(a).add_(u)
        return s["state"].to(s["x"].dtype), s["state"]
    if own:
        import mamba2d_b200
        out = mamba2d_b200.gated_recurrence(s["x"], s["gate"], form=case["form"], initial_state=s["state"], lengths=s["lengths"], return_state=case["state"])
        if case["kind"] != "train":
            return out
        leaves = [s[n] for n in ("x", "gate", "state") if s[n] is not None]
        if case["state"]:
            return (*out, *torch.autograd.grad(out, leaves, (s["d_out"], s["d_state"])))
        return (out, *torch.autograd.grad(out, leaves, s["d_out"]))
    with torch.no_grad():
        return _plain_recur(s)


def _plain_terms(x, gate, form):
    """a and u of h_t = a_t h_{t-1} + u_t."""
    if form == "decay":
        return torch.exp(gate), x
    return 1 / (1 + torch.exp(-gate)), x / (1 + torch.exp(gate))


def _scan(a, u):
    """All h_t of h_t = a_t h_{t-1} + u_t along the second dimension: pairs of tokens make one, whose scan gives every second h."""
    T = u.shape[1]
    if T == 1:
        return u
    odd = _scan(a[:, 1::2] * a[:, :T - 1:2], torch.addcmul(u[:, 1::2], a[:, 1::2], u[:, :T - 1:2]))
    h = torch.empty_like(u)
    h[:, 1::2] = odd
    h[:, 0] = u[:, 0]
    h[:, 2::2] = torch.addcmul(u[:, 2::2], a[:, 2::2], odd[:, :(T - 1) // 2])
    return h


def _plain_recur(s):
    case, x, gate, state = s["case"], s["x"].float(), s["gate"].float(), s["state"]
    a, u = _plain_terms(x, gate, case["form"])
    if s["lengths"] is not None:         # behind a sequence nothing changes the state
        live = (torch.arange(case["T"], device=x.device) < s["lengths"][:, None])[..., None]
        a, u = torch.where(live, a, 1.0), torch.where(live, u, 0.0)
    else:
        live = None
    first = u if state is None else torch.cat((torch.addcmul(u[:, :1], a[:, :1], state[:, None]), u[:, 1:]), 1)
    h = _scan(a, first)
    y = (h if live is None else torch.where(live, h, 0.0)).to(s["x"].dtype)
    out = (y, h[:, -1].clone()) if case["state"] else (y,)
    if case["kind"] != "train":
        return out if case["state"] else y
    dy = s["d_out"].float() if live is None else torch.where(live, s["d_out"].float(), 0.0)
    last = dy if not case["state"] else torch.cat((dy[:, :-1], dy[:, -1:] + s["d_state"][:, None]), 1)
    # D_t = dy_t + a_{t+1} D_{t+1}
    ahead = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), 1)
    D = _scan(ahead.flip(1), last.flip(1)).flip(1)
    before = torch.cat((torch.zeros_like(h[:, :1]) if state is None else state[:, None], h[:, :-1]), 1)
    if case["form"] == "decay":
        dx, dgate = D, D * a * before
    else:
        rest = 1 / (1 + torch.exp(gate))
        dx, dgate = D * rest, D * a * rest * (before - x)
    if live is not None:
        dx, dgate = torch.where(live, dx, 0.0), torch.where(live, dgate, 0.0)
    return (*out, dx.to(s["x"].dtype), dgate.to(s["x"].dtype), *([a[:, 0] * D[:, 0]] if case["state"] else []))


def _run_norm(s):
    case = s["case"]
    if own:
        import mamba2d_b200
        out = mamba2d_b200.layer_norm(s["x"], s["weight"], s["bias"], residual=s["residual"])
        if case["kind"] != "train":
            return out
        leaves = [s[n] for n in ("x", "residual", "weight", "bias") if s[n] is not None]
        if case["residual"]:
            return (*out, *torch.autograd.grad(out, leaves, (s["d_out"], s["d_sum"])))
        return (out, *torch.autograd.grad(out, leaves, s["d_out"]))
    with torch.no_grad():
        return _plain_norm(s)


def _plain_norm(s, eps=1e-5):
    case, weight = s["case"], s["weight"]
    total = s["x"] if not case["residual"] else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    f = total.float()
    d = f - f.mean(-1, keepdim=True)
    inv = torch.rsqrt((d * d).mean(-1, keepdim=True) + eps)
    h = d * inv
    y = (h * weight + s["bias"]).to(total.dtype)
    out = (y, total) if case["residual"] else (y,)
    if case["kind"] != "train":
        return out if case["residual"] else y
    dy = s["d_out"].float()
    dh = dy * weight
    dx = inv * (dh - dh.mean(-1, keepdim=True) - h * (dh * h).mean(-1, keepdim=True))
    if case["residual"]:
        dx = dx + s["d_sum"].float()
    dx = dx.to(total.dtype)
    return (*out, dx, *([dx] if case["residual"] else []), (dy * h).sum(0), dy.sum(0))


def _run_distill(s):
    case = s["case"]
    if own:
        import mamba2d_b200
        loss = mamba2d_b200.distillation_loss(s["logits"], s["top"], s["index"], s["labels"], temperature=case["temperature"], label_weight=case["label_weight"])
        return (loss, *torch.autograd.grad(loss, s["logits"], s["d_loss"])) if case["kind"] == "train" else loss
    with torch.no_grad():
        return _plain_distill(s)


def _plain_distill(s):
    case = s["case"]
    tau, w = case["temperature"], case["label_weight"]
    z = s["logits"].float()
    m = z.max(-1, keepdim=True).values
    e = torch.exp((z - m) / tau)
    q = e.sum(-1, keepdim=True)
    there = s["index"] >= 0
    at = s["index"].clamp(min=0)
    t = torch.where(there, s["top"].float(), -math.inf)
    t = (t - t.max(-1, keepdim=True).values).double() / tau
    p = torch.exp(t)
    total = p.sum(-1, keepdim=True)
    p = p / total
    log_q = (z.gather(-1, at) - m).double() / tau - torch.log(q.double())
    loss = (1 - w) * tau * tau * torch.where(there, p * (t - torch.log(total) - log_q), 0.0).sum(-1)
    if w > 0:
        e1 = e if tau == 1 else torch.exp(z - m)
        one = e1.sum(-1, keepdim=True)
        label, counted = s["labels"].clamp(min=0)[:, None], (s["labels"] >= 0)[:, None]
        nll = torch.log(one.double()) - (z.gather(-1, label) - m).double()
        loss = loss + w * torch.where(counted, nll, 0.0)[:, 0]
    loss = loss.float()
    if case["kind"] != "train":
        return loss
    up = s["d_loss"][:, None]
    dz = e * ((1 - w) * tau / q * up)
    dz.scatter_add_(-1, at, (torch.where(there, p, 0.0) * (-(1 - w) * tau)).float() * up)
    if w > 0:
        live = torch.where(counted, w * up, 0.0)
        dz += e1 * (live / one)
        dz.scatter_add_(-1, label, -live)
    return loss, dz.to(s["logits"].dtype)


def work(case):
    """Bytes: inputs once, outputs once.  Operations: a handful for each value."""
    s, train = 4 if case["dtype"] == "f32" else 2, case["kind"] == "train"
    if case["op"] == "recur":
        n = case["B"] * case["T"] * case["C"] * (0.65 if case["ragged"] else 1)
        state = 4 * case["B"] * case["C"] * (2 if case["kind"] == "step" or case["state"] else 0)
        return {"bytes": n * s * (6 if train else 3) + state * (2 if train else 1), "flops": n * (28 if train else 8)}
    if case["op"] == "norm":
        n, extra = case["N"] * case["C"], 2 if case["residual"] else 0
        return {"bytes": n * s * ((4 if train else 2) + extra * (2 if train else 1)) + 8 * case["C"] * (2 if train else 1), "flops": n * (24 if train else 8)}
    n, rows = case["N"] * case["V"], case["N"] * (case["K"] * (8 + s) + 4 + (8 if case["label_weight"] else 0) + (4 if train else 0))
    return {"bytes": n * s * (2 if train else 1) + rows, "flops": n * (8 if train else 4) * (2 if case["label_weight"] and case["temperature"] != 1 else 1)}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"recur": _exact_recur, "norm": _exact_norm, "distill": _exact_distill}[case["op"]](case, s)


def _exact_recur(case, s):
    """Token by token, forwards for the states and backwards for what flows through them."""
    step, form, train = case["kind"] == "step", case["form"], case["kind"] == "train"
    x, g = (s[n].detach().double() for n in ("x", "gate"))
    if step:
        x, g = x[:, None], g[:, None]
    B, T, C = x.shape
    f = torch.exp(g) if form == "decay" else torch.sigmoid(g)
    rest = torch.sigmoid(-g) if form == "forget" else None
    h = s["state"].detach().double() if s["state"] is not None else torch.zeros(B, C, dtype=x.dtype, device=x.device)
    lengths = s["lengths"].long() if s["lengths"] is not None else None
    before, y = torch.empty_like(x) if train else None, torch.zeros_like(x)
    for t in range(T):
        if train:
            before[:, t] = h
        new = f[:, t] * h + (x[:, t] if form == "decay" else rest[:, t] * x[:, t])
        if lengths is not None:
            inside = (lengths > t)[:, None]
            y[:, t] = new * inside
            h = torch.where(inside, new, h)
        else:
            y[:, t] = h = new
    if step:
        return y[:, 0], h
    if not train:
        return (y, h) if case["state"] else y
    final, dy = h, s["d_out"].double()
    R = s["d_state"].double() if case["state"] else torch.zeros_like(h)
    dx, dg = torch.zeros_like(x), torch.zeros_like(x)
    for t in reversed(range(T)):
        D = dy[:, t] + R
        if form == "decay":
            dxt, dgt = D, D * f[:, t] * before[:, t]
        else:
            dxt, dgt = D * rest[:, t], D * f[:, t] * rest[:, t] * (before[:, t] - x[:, t])
        if lengths is not None:
            inside = (lengths > t)[:, None]
            dx[:, t], dg[:, t], R = dxt * inside, dgt * inside, torch.where(inside, f[:, t] * D, R)
        else:
            dx[:, t], dg[:, t], R = dxt, dgt, f[:, t] * D
    return (y, final, dx, dg, R) if case["state"] else (y, dx, dg)


def _exact_norm(case, s, eps=1e-5):
    x = s["x"].detach().double()
    if case["residual"]:                 # the stream holds the sum in its own type
        x = (x + s["residual"].detach().double()).to(s["x"].dtype).double()
    C = x.shape[1]
    mean = x.sum(1, keepdim=True) / C
    var = ((x - mean) ** 2).sum(1, keepdim=True) / C
    rstd = 1 / (var + eps).sqrt()
    h = (x - mean) * rstd
    w, b = s["weight"].detach().double(), s["bias"].detach().double()
    y = h * w + b
    if case["kind"] != "train":
        return (y, x) if case["residual"] else y
    dy = s["d_out"].double()
    dh = dy * w
    dx = rstd * (dh - dh.sum(1, keepdim=True) / C - h * ((dh * h).sum(1, keepdim=True) / C))
    if case["residual"]:
        dx = dx + s["d_sum"].double()
        return y, x, dx, dx, (dy * h).sum(0), dy.sum(0)
    return y, dx, (dy * h).sum(0), dy.sum(0)


def _exact_distill(case, s):
    tau, w, N = case["temperature"], case["label_weight"], case["N"]
    z = s["logits"].detach().double()
    log_q = torch.log_softmax(z / tau, -1)
    loss = torch.zeros(N, dtype=torch.float64, device=z.device)
    dz = torch.exp(log_q).mul_((1 - w) * tau) if case["kind"] == "train" else None
    rows = torch.arange(N, device=z.device)
    there = s["index"] >= 0
    log_p = torch.log_softmax(torch.where(there, s["top"].double() / tau, -math.inf), -1)
    for k in range(case["K"]):
        live, at = there[:, k], s["index"][:, k].clamp(min=0)
        p = torch.where(live, torch.exp(log_p[:, k]), 0.0)
        loss += (1 - w) * tau ** 2 * torch.where(live, p * (log_p[:, k] - log_q[rows, at]), 0.0)
        if dz is not None:
            dz[rows, at] -= (1 - w) * tau * p
    del log_q
    if w > 0:
        has, at = s["labels"] >= 0, s["labels"].clamp(min=0)
        log_1 = torch.log_softmax(z, -1)
        loss -= w * torch.where(has, log_1[rows, at], 0.0)
        if dz is not None:
            dz += w * torch.exp(log_1) * has[:, None]
            dz[rows, at] -= w * has
    return loss if dz is None else (loss, dz * s["d_loss"].double()[:, None])
