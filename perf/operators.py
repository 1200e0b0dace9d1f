"""The sequence operators next to the 2-D scan, as they are measured: linear attention with a decay per head (prompts,
training, single tokens), group normalisation with an activation on channels-last tensors, and clipping of gradients by
their global norm.

``run`` computes them in plain form (elementary torch operations in 32 bits, decays and long sums in 64), or, where
``own`` is set, by the calls that a user makes of this package.  ``exact`` follows the definitions token by token in
64 bits.
"""
import math

import torch

own = False

SCAN_WIDTHS = (64, 96, 128, 192, 320, 384, 512, 576)     # stage widths of the shipped models


def listed():
    def attention(name, kind, B, T, H, G, K, V, dtype, decay, state=False, ragged=False):
        return dict(name=name, op="attention", kind=kind, B=B, T=T, H=H, G=G, K=K, V=V, dtype=dtype, decay=decay, state=state, ragged=ragged)

    def norm(name, kind, N, S, C, groups, dtype, act):
        return dict(name=name, op="norm", kind=kind, N=N, S=S, C=C, groups=groups, dtype=dtype, act=act)

    return [
        # one token of one sequence: what a single user's next token waits for
        attention("step_1x8x64x64_bf16", "step", 1, 1, 8, 8, 64, 64, "bf16", "token"),
        # one token of 256 sequences served together, queries and keys shared by four heads
        attention("step_256x16x128x128_bf16", "step", 256, 1, 16, 4, 128, 128, "bf16", "token"),
        # the tokens of one 14x14 map of 320 channels in heads of 64
        attention("prefill_1x196x5x64_f32", "prefill", 1, 196, 5, 5, 64, 64, "f32", "token"),
        # four prompts, fixed decays, the state kept for the tokens that follow
        attention("prefill_4x4096x16x128_bf16", "prefill", 4, 4096, 16, 16, 128, 128, "bf16", "head", state=True),
        # one long prompt; one query and key for all heads
        attention("prefill_1x65536x8x64_bf16", "prefill", 1, 65536, 8, 1, 128, 64, "bf16", "token", state=True),
        # ragged sequences of up to 45x31 pixels, 192 channels, fp32
        attention("train_6x1395x3x64_f32", "train", 6, 1395, 3, 3, 64, 64, "f32", "token", ragged=True),
        # a training step's share of one GPU
        attention("train_8x2048x16x128_bf16", "train", 8, 2048, 16, 16, 128, 128, "bf16", "token"),
        # one image, third stage
        norm("norm_1x14x14x320_f32", "infer", 1, 196, 320, 32, "f32", "silu"),
        # batched training, first stage
        norm("norm_128x56x56x64_bf16", "train", 128, 3136, 64, 16, "bf16", "gelu"),
        # every head of a token normalised for itself, as after the attention of the training case
        norm("norm_16384x16x128_bf16", "train", 16384, 1, 2048, 16, "bf16", "silu"),
        # the gradients of a model of the shipped tiny widths and depths
        dict(name="clip_tiny_f32", op="clip", widths="64,128,320,512", blocks="3,3,9,3", dtype="f32"),
        # a large model's, in bf16
        dict(name="clip_wide_bf16", op="clip", widths="2048", blocks="16", dtype="bf16"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    kind = rng.choice(("step", "prefill", "train", "prefill", "train", "norm", "norm", "clip"))
    dtype = rng.choice(("f32", "bf16"))
    if kind in ("step", "prefill", "train"):
        K, V = rng.choice((32, 48, 64, 64, 96, 128, 128)), rng.choice((32, 64, 64, 80, 128, 128))
        H = rng.choice((1, 2, 3, 4, 5, 8, 12, 16))
        G = rng.choice([d for d in range(1, H + 1) if H % d == 0])
        if kind == "step":
            B, T = log_int(1, 256), 1
        else:
            # up to the listed training step's tokens (prompts: the listed long prompt's)
            most = 32768 if kind == "train" else 65536
            cost = H * (K + V) / 256 * (4 if dtype == "f32" else 1)
            B = log_int(1, 16)
            T = log_int(1, max(1, min(8192 if kind == "train" else 32768, int(most * 4 / (B * cost)))))
        return dict(op="attention", kind=kind, B=B, T=T, H=H, G=G, K=K, V=V, dtype=dtype, decay=rng.choice(("head", "token", "token")),
                    state=kind != "step" and rng.random() < 0.4, ragged=kind != "step" and B > 1 and rng.random() < 0.4)
    if kind == "norm":
        act = rng.choice(("", "silu", "gelu"))
        train = rng.choice(("infer", "train"))
        if rng.random() < 0.4:       # heads of tokens
            groups, per = rng.choice((1, 2, 3, 4, 8, 16)), rng.choice((32, 48, 64, 96, 128))
            return dict(op="norm", kind=train, N=log_int(1, 16384), S=1, C=groups * per, groups=groups, dtype=dtype, act=act)
        C = rng.choice(SCAN_WIDTHS)
        groups = rng.choice([g for g in (1, 4, 8, 16, 32) if C % g == 0])
        side = log_int(5, 128)
        S = side * max(3, int(side * math.exp(rng.uniform(-0.5, 0.5))))
        return dict(op="norm", kind=train, N=log_int(1, max(1, min(128, (1 << 24) // (S * C)))), S=S, C=C, groups=groups, dtype=dtype, act=act)
    level = [str(rng.choice(SCAN_WIDTHS[2 * i:2 * i + 2])) for i in range(4)]
    return dict(op="clip", widths=",".join(level), blocks=",".join(str(rng.randint(1, 12)) for _ in range(4)), dtype=dtype)


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=g, device="cuda") * (hi - lo) + lo

    return {"case": dict(case), **{"attention": _prepare_attention, "norm": _prepare_norm, "clip": _prepare_clip}[case["op"]](case, normal, uniform)}


def _prepare_attention(case, normal, uniform):
    B, T, H, G, K, V = (case[k] for k in ("B", "T", "H", "G", "K", "V"))
    dt = _dtype(case)
    tokens = (B,) if case["kind"] == "step" else (B, T)
    s = {"q": normal(*tokens, G, K).to(dt), "k": (normal(*tokens, G, K) * K ** -0.5).to(dt), "v": normal(*tokens, H, V).to(dt)}
    if case["decay"] == "head":          # fixed, from a memory of 16 tokens to one of 4096
        s["decay"] = torch.log1p(-torch.exp2(-4 - 8 * torch.arange(H, device="cuda", dtype=torch.float32) / max(1, H - 1)))
    else:                                # a step size for each token, a rate for each head
        step = torch.nn.functional.softplus(normal(*tokens, H) * 0.5 - 3.0)
        s["decay"] = -step * torch.exp(uniform(math.log(0.1), math.log(16.0), H))
    s["scale"] = K ** -0.5
    s["state"] = normal(B, H, K, V) if case["kind"] == "step" or case["state"] else None
    s["lengths"] = (uniform(0.3, 1.0, B) * T).ceil().to(torch.int32) if case["ragged"] else None
    if case["kind"] == "train":
        s["d_out"] = normal(*tokens, H, V).to(dt)
        s["d_state"] = normal(B, H, K, V) if case["state"] else None
        for n in ("q", "k", "v", "decay", "state"):
            if s[n] is not None and not (n == "decay" and case["decay"] == "head"):
                s[n].requires_grad_(True)
    return s


def _prepare_norm(case, normal, uniform):
    N, S, C, dt = case["N"], case["S"], case["C"], _dtype(case)
    scale = torch.exp(0.5 * normal(N, 1, 1))              # images differ in contrast and brightness
    s = {"x": (normal(N, S, C) * scale + normal(N, 1, C)).to(dt), "weight": 1.0 + 0.1 * normal(C), "bias": 0.1 * normal(C)}
    if S == 1:
        s["x"] = s["x"].view(N, C)
    if case["kind"] == "train":
        s["d_out"] = normal(*s["x"].shape).to(dt)
        for n in ("x", "weight", "bias"):
            s[n].requires_grad_(True)
    return s


def _shapes(case):
    """The parameters of a model of these stages: norms, projections, scan parameters, depthwise convolution, MLP."""
    out = []
    for E, n in zip(map(int, case["widths"].split(",")), map(int, case["blocks"].split(","))):
        R = math.ceil(E / 16)
        block = [(E,), (E,), (E, E), (2 * R + 48, E), (E, R), (E,), (E, R), (E,), (E, 16), (E, 16), (E,), (E, E), (E, 1, 3, 3), (4 * E, E), (4 * E,), (E, 4 * E), (E,)]
        out += block * n
    return out + [(1000, E), (1000,)]


def _prepare_clip(case, normal, uniform):
    # gradients as data-parallel training holds them: views of one buffer, neighbours without gaps
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    flat = (normal(sum(sizes)) * 1e-3).to(_dtype(case))
    return {"flat": flat, "grads": [f.view(s) for f, s in zip(flat.split(sizes), shapes)], "max_norm": 0.5e-3 * sum(sizes) ** 0.5}


def run(state):
    return {"attention": _run_attention, "norm": _run_norm, "clip": _run_clip}[state["case"]["op"]](state)


def _run_attention(s):
    kind = s["case"]["kind"]
    if kind == "step":
        if own:
            import mamba2d_b200
            return mamba2d_b200.linear_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"], scale=s["scale"]), s["state"]
        return _plain_step(s)
    if own:
        import mamba2d_b200
        o = mamba2d_b200.linear_attention(s["q"], s["k"], s["v"], s["decay"], scale=s["scale"], initial_state=s["state"], lengths=s["lengths"],
                                          return_state=s["case"]["state"])
    else:
        o = _plain_attention(s)
    if kind != "train":
        return o
    return _with_grads(s, o)


def _with_grads(s, o):
    leaves = [s[n] for n in ("q", "k", "v", "decay", "state") if s[n] is not None and s[n].requires_grad]
    if s["case"]["state"]:
        return (*o, *torch.autograd.grad(o, leaves, (s["d_out"], s["d_state"])))
    return (o, *torch.autograd.grad(o, leaves, s["d_out"]))


def _plain_step(s):
    heads = s["v"].shape[1] // s["q"].shape[1]
    q, k = (s[n].float().repeat_interleave(heads, 1) for n in ("q", "k"))
    s["state"].mul_(torch.exp(s["decay"])[..., None, None]).add_(k[..., :, None] * s["v"].float()[..., None, :])
    return (s["scale"] * (q[..., :, None] * s["state"]).sum(-2)).to(s["v"].dtype), s["state"]


def _plain_attention(s, chunk=64):
    """Chunks of 64 tokens: products of pairs inside a chunk, a state of (K, V) between chunks."""
    B, T, H, V = s["v"].shape
    G, K = s["q"].shape[2:]
    N = -(-T // chunk)

    def tiles(x, n, fill=0.0):           # (B, T, heads, n) -> (B, H, N, chunk, n)
        if x.shape[2] != H:
            x = x.repeat_interleave(H // x.shape[2], 2)
        if s["lengths"] is not None:
            x = torch.where(inside, x, fill)
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, N * chunk - T))
        return x.view(B, N, chunk, H, n).permute(0, 3, 1, 2, 4)

    if s["lengths"] is not None:
        inside = (torch.arange(T, device=s["v"].device) < s["lengths"][:, None])[:, :, None, None]
    q, k, v = tiles(s["q"].float(), K), tiles(s["k"].float(), K), tiles(s["v"].float(), V)
    g = tiles(s["decay"].expand(B, T, H)[..., None], 1)[..., 0].double()
    c = g.cumsum(-1)                                                            # (B, H, N, chunk)
    later = torch.ones(chunk, chunk, dtype=torch.bool, device=v.device).triu(1)
    pairs = torch.exp((c[..., :, None] - c[..., None, :]).masked_fill(later, -math.inf)).float()
    o = ((q @ k.transpose(-1, -2)) * pairs) @ v
    delta = (k * torch.exp(c[..., -1:] - c).float()[..., None]).transpose(-1, -2) @ v      # what each chunk adds to the state
    ends = torch.nn.functional.pad(c[..., -1].cumsum(-1), (1, 0))               # decay up to the start of chunk n (and the end)
    after = torch.ones(N + 1, N, dtype=torch.bool, device=v.device).triu(0)     # chunk m adds to the states before chunks n > m
    between = torch.exp((ends[..., :, None] - ends[..., None, 1:]).masked_fill(after, -math.inf)).float()
    states = (between @ delta.reshape(B, H, N, K * V)).view(B, H, N + 1, K, V)
    if s["state"] is not None:
        states = states + torch.exp(ends).float()[..., None, None] * s["state"][:, :, None]
    o = o + (q * torch.exp(c).float()[..., None]) @ states[:, :, :N]
    o = (s["scale"] * o).permute(0, 2, 3, 1, 4).reshape(B, N * chunk, H, V)[:, :T].to(s["v"].dtype)
    if s["lengths"] is not None:
        o = torch.where(inside, o, 0.0)
    return (o, states[:, :, N]) if s["case"]["state"] else o


def _run_norm(s):
    case = s["case"]
    if own:
        import mamba2d_b200
        y = mamba2d_b200.group_norm(s["x"], case["groups"], s["weight"], s["bias"], act=case["act"] or None)
    else:
        y = _plain_norm(s["x"], s["weight"], s["bias"], case)
    if case["kind"] != "train":
        return y
    return (y, *torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["d_out"]))


def _plain_norm(x, weight, bias, case):
    C, groups = case["C"], case["groups"]
    f = x.float().reshape(x.shape[0], -1, groups, C // groups)
    d = f - f.mean((1, 3), keepdim=True)
    y = d * torch.rsqrt((d * d).mean((1, 3), keepdim=True) + 1e-5)
    y = y.reshape(x.shape) * weight + bias
    if case["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif case["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y.to(x.dtype)


def _run_clip(s):
    # the bound tightens a little with every step, so that every pass clips
    s["max_norm"] *= 0.999
    if own:
        import mamba2d_b200
        return mamba2d_b200.clip_norm_(s["grads"], s["max_norm"]), s["flat"]
    total = torch.sqrt(sum(g.float().square().sum().double() for g in s["grads"])).float()
    factor = torch.clamp(s["max_norm"] / (total + 1e-6), max=1.0)
    [g.copy_(g.float() * factor) for g in s["grads"]]
    return total, s["flat"]


def work(case):
    """Bytes: inputs once, outputs once.  Operations: the recurrences' own (4 KV a token and head forward, three times that
    with the backward pass), whatever more a chunked form computes."""
    s = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        n, train = case["N"] * case["S"] * case["C"], case["kind"] == "train"
        return {"bytes": n * s * (4 if train else 2) + 8 * case["C"] * (2 if train else 1), "flops": n * (30 if train else 10)}
    if case["op"] == "clip":
        n = sum(math.prod(x) for x in _shapes(case))
        return {"bytes": 2 * n * s, "flops": 3 * n}
    B, T, H, G, K, V = (case[k] for k in ("B", "T", "H", "G", "K", "V"))
    T = T * 0.65 if case["ragged"] else T
    tokens = s * B * T * (2 * G * K + 2 * H * V) + (4 * B * T * H if case["decay"] == "token" else 4 * H)
    state = 4 * B * H * K * V
    if case["kind"] == "step":
        return {"bytes": tokens + 2 * state, "flops": 5 * B * H * K * V}
    if case["kind"] == "train":
        return {"bytes": tokens * 2 + (4 * state if case["state"] else 0), "flops": 12 * B * T * H * K * V}
    return {"bytes": tokens + (2 * state if case["state"] else 0), "flops": 4 * B * T * H * K * V}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "norm": _exact_norm, "clip": _exact_clip}[case["op"]](case, s)


def _exact_attention(case, s):
    """S_t = exp(g_t) S_{t-1} + k_t v_t^T, o_t = scale q_t^T S_t, and backwards through the tokens D_t = exp(g_{t+1}) D_{t+1} +
    scale q_t do_t^T for the gradients."""
    B, T, H, G, K, V = (case[k] for k in ("B", "T", "H", "G", "K", "V"))
    dt, scale = torch.float64, s["scale"]
    step = case["kind"] == "step"

    def each(x):                          # (B, T, heads, n), a head's own copy of what it shares
        x = x.detach().to(dt)
        x = x[:, None] if step else x
        return x.repeat_interleave(H // x.shape[2], 2)

    q, k, v = each(s["q"]), each(s["k"]), each(s["v"])
    g = s["decay"].detach().to(dt)
    g = (g[:, None] if step else g) if g.dim() > 1 else g.expand(B, T, H)
    live = torch.ones(B, T, 1, dtype=dt, device=v.device)
    if s["lengths"] is not None:
        live = (torch.arange(T, device=v.device) < s["lengths"][:, None]).to(dt)[..., None]
    a = torch.exp(g * live)
    k, q = k * live[..., None], q * live[..., None]
    S = torch.zeros(B, H, K, V, dtype=dt, device=v.device) if s["state"] is None else s["state"].detach().to(dt)
    train, every = case["kind"] == "train", 64
    o, kept = torch.empty(B, T, H, V, dtype=dt, device=v.device), []
    for t in range(T):
        if train and t % every == 0:
            kept.append(S)
        S = S * a[:, t, :, None, None] + k[:, t, :, :, None] * v[:, t, :, None, :]
        o[:, t] = scale * (q[:, t, :, None, :] @ S)[:, :, 0]
    if step:
        return o[:, 0], S
    if not train:
        return (o, S) if case["state"] else o
    do, final = s["d_out"].to(dt), S
    D = s["d_state"].to(dt) if case["state"] else torch.zeros_like(S)
    dq, dk, dv, dg = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(a)
    for n in reversed(range(len(kept))):
        S, before = kept[n], []
        for t in range(n * every, min(T, n * every + every)):
            before.append(S)
            S = S * a[:, t, :, None, None] + k[:, t, :, :, None] * v[:, t, :, None, :]
        for t in reversed(range(n * every, min(T, n * every + every))):
            D = D + scale * q[:, t, :, :, None] * do[:, t, :, None, :]
            dq[:, t] = scale * live[:, t, :, None] * (S @ do[:, t, :, :, None])[..., 0]
            dk[:, t] = live[:, t, :, None] * (D @ v[:, t, :, :, None])[..., 0]
            dv[:, t] = (k[:, t, :, None, :] @ D)[:, :, 0]
            S = before[t - n * every]
            dg[:, t] = live[:, t] * a[:, t] * (S * D).sum((-1, -2))
            D = D * a[:, t, :, None, None]
    dq, dk = (x.view(B, T, G, H // G, K).sum(3) for x in (dq, dk))
    return (o, *([final] if case["state"] else []), dq, dk, dv, *([dg] if case["decay"] == "token" else []), *([D] if case["state"] else []))


def _exact_norm(case, s):
    """Every group by its own sums; the gradients by the derivative of a normalised value with respect to its group."""
    G, Cg, N, S = case["groups"], case["C"] // case["groups"], case["N"], case["S"]
    x = s["x"].detach().double().view(N, S, G, Cg).transpose(1, 2).reshape(N * G, S * Cg)
    n = x.shape[1]
    mean = x.sum(1, keepdim=True) / n
    inv = 1 / ((x * x).sum(1, keepdim=True) / n - mean * mean + 1e-5).sqrt()
    h = (x - mean) * inv
    w, b = (s[k].detach().double().view(1, G, 1, Cg).expand(N, G, S, Cg).reshape(N * G, S * Cg) for k in ("weight", "bias"))
    z = h * w + b
    if case["act"] == "silu":
        sg = torch.sigmoid(z)
        y, slope = z * sg, sg * (1 + z * (1 - sg))
    elif case["act"] == "gelu":
        cdf = torch.special.ndtr(z)
        y, slope = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        y, slope = z, torch.ones_like(z)

    def back(t):
        return t.view(N, G, S, Cg).transpose(1, 2).reshape(s["x"].shape)

    if case["kind"] != "train":
        return back(y)
    dz = s["d_out"].double().view(N, S, G, Cg).transpose(1, 2).reshape(N * G, S * Cg) * slope
    dh = dz * w
    dx = inv * (dh - dh.sum(1, keepdim=True) / n - h * (dh * h).sum(1, keepdim=True) / n)
    per_channel = lambda t: t.view(N, G, S, Cg).sum((0, 2)).reshape(-1)  # noqa: E731
    return back(y), back(dx), per_channel(dz * h), per_channel(dz)


def _exact_clip(case, s):
    f = s["flat"].double()
    total = f.norm()
    return total, f * min(1.0, float(s["max_norm"] * 0.999 / (total + 1e-6)))
