"""Calls of the linear attention that its documentation allows and its own tests do not make.  Tolerances are those of its
own tests (see test_attention_gpu.py) where nothing else is said."""
import collections
import ctypes

import pytest
import torch

from test_attention_gpu import BF, make
from test_sequence_host import AttnDesc, Tensor
from mamba2d_b200 import _lib, linear_attention, linear_attention_step

pytestmark = pytest.mark.gpu


def test_as_many_tokens_as_there_may_be():
    """Just below 2^31 tokens, in segments whose last would end behind 2^31.  All tokens are the same one: o is the geometric
    series, 2 - 2^-t, which bf16 cannot tell from 2 after ten tokens."""
    T = 2 ** 31 - 2049
    one = torch.ones(1, 1, 1, 1, dtype=BF, device="cuda").expand(1, T, 1, 1)
    decay = torch.full((1,), 0.5, device="cuda").log()
    o, state = linear_attention(one, one, one, decay, scale=1.0, return_state=True)
    assert abs(float(state) - 2) < 1e-5
    assert abs(float(o[0, 0]) - 1) < 1e-2 and abs(float(o[0, 1]) - 1.5) < 1e-2
    for part in o.view(-1).split(2 ** 28):
        low, high = torch.aminmax(part[10:])
        assert float(low) == float(high) == 2.0
    del o
    lengths = torch.tensor([T - 5000], dtype=torch.int32, device="cuda")
    o = linear_attention(one, one, one, decay, scale=1.0, lengths=lengths).view(-1)
    assert not o[T - 5000:].any() and bool((o[T - 2 ** 20:T - 5000] == 2).all())


def _tensor(t):
    return Tensor(t.data_ptr(), *t.stride()[:3])


def _through_the_library(q, k, v, d, s, flags, d_o=None):
    """m2d_attn_fwd, or m2d_attn_bwd where d_o is given, with these descriptor flags: (o, state) or (dq, dk, dv, ds)."""
    B, T, H, V = v.shape
    G, K = q.shape[2:]
    desc = AttnDesc(struct_bytes=ctypes.sizeof(AttnDesc), dtype=_lib.M2D_BF16, B=B, T=T, H=H, G=G, K=K, V=V, flags=flags, scale=K ** -0.5, q=_tensor(q), k=_tensor(k), v=_tensor(v),
                    log_decay=d.data_ptr(), g_batch=d.stride(0), g_token=d.stride(1), g_head=d.stride(2), state=s.data_ptr())
    L = ctypes.CDLL(_lib.LIB_PATH)
    if d_o is None:
        outs = [torch.empty_like(v), torch.empty_like(s)]
        desc.o, desc.state_out = (t.data_ptr() for t in outs)
        query, call = L.m2d_attn_fwd_workspace, L.m2d_attn_fwd
    else:
        outs = [torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(s)]
        desc.d_q, desc.d_k, desc.d_v, desc.d_state = (t.data_ptr() for t in outs)
        desc.d_o = _tensor(d_o)
        query, call = L.m2d_attn_bwd_workspace, L.m2d_attn_bwd
    query.restype = ctypes.c_uint64
    need = query(ctypes.byref(desc))
    ws = torch.zeros(max(need, 1), dtype=torch.uint8, device="cuda")
    desc.workspace, desc.workspace_bytes = ws.data_ptr(), need
    assert call(ctypes.byref(desc), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    return outs


# two segments, four, five (a launch joins them)
@pytest.mark.parametrize("B,T,H,K,V", [(2, 1100, 2, 64, 64), (1, 2100, 2, 128, 64), (1, 2561, 3, 64, 128)])
def test_a_wait_that_gives_up_leaves_nothing_that_looks_right(B, T, H, K, V, monkeypatch):
    """What depends on a CTA that gave up is NaN, be it through the state of a segment; all else is as ever, and the next
    call tells."""
    monkeypatch.setenv("M2D_TEST_HOOKS", "1")
    _lib.lib()
    q, k, v, d, s, _ = make(B, T, H, H, K, V, BF, state=True)
    d_o = torch.randn(v.shape, device="cuda").to(BF)
    want, grads = _through_the_library(q, k, v, d, s, 0), _through_the_library(q, k, v, d, s, 0, d_o)
    assert not _lib.take_wait_failure()

    def check(got, want, spoilt):
        """Bits as ever or NaN; NaN in head 0 of sequence 0 alone, and in all of ``spoilt`` there."""
        for name, x, y in zip(got._fields, got, want):
            nan = torch.isnan(x)
            assert torch.equal(x[~nan], y[~nan]) and not bool(torch.isnan(y).any()), name
            inside = nan[:1, :1] if name in ("state", "ds") else nan[:1, :, :1]
            assert int(inside.sum()) == int(nan.sum()), name
            if name in spoilt:
                rows = inside.flatten(1).all(1) if name in ("state", "ds") else inside[0, :, 0].all(-1)
                assert bool(rows[spoilt[name]].all()), name

    Out, Grads = collections.namedtuple("Out", "o state"), collections.namedtuple("Grads", "dq dk dv ds")
    hook = 0x100                                             # what comes after the first segment comes of the first CTA's state
    check(Out(*_through_the_library(q, k, v, d, s, hook)), want, {"o": slice(T - 128, T), "state": slice(None)})
    assert _lib.take_wait_failure()
    check(Grads(*_through_the_library(q, k, v, d, s, hook, d_o)), grads, {"dq": slice(T - 128, T)})
    with pytest.raises(RuntimeError, match="earlier launch timed out"):
        linear_attention(q, k, v, d)
    assert not _lib.take_wait_failure()
    check(Out(*_through_the_library(q, k, v, d, s, 0)), want, {})


def test_a_token_behind_a_prompt_that_went_wrong_tells(monkeypatch):
    monkeypatch.setenv("M2D_TEST_HOOKS", "1")
    _lib.lib()
    q, k, v, d, s, _ = make(2, 1100, 2, 2, 64, 64, BF, state=True)
    _, state = _through_the_library(q, k, v, d, s, 0x100)
    with pytest.raises(RuntimeError, match="linear_attention_step: a wait inside an earlier launch timed out"):
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], d[:, 0], state)
    assert not _lib.take_wait_failure()
    assert bool(torch.isfinite(linear_attention_step(q[:, 0], k[:, 0], v[:, 0], d[:, 0], s)).all())      # told once


@pytest.mark.parametrize("exponent", [-57, 57])
@pytest.mark.parametrize("rate", [0.3, 0.55, 0.65, 0.8])
def test_small_and_large_values_with_steep_decays(rate, exponent):
    """v, and the gradient of the output, times a power of two, which changes no rounding: 2^-57 is 7e-18.  Everything that
    is a product of them is that many times what it was, in every bit.  (Decays of 16 to 46 in a chunk's 128 tokens from its
    middle, as powers of two 25 to 74: the tcgen05 form holds a pair's weight as a product of factors that large.)"""
    q, k, v, _, s, _ = make(2, 1100, 2, 1, 64, 128, BF, state=True)
    d = -rate * (0.9 + 0.2 * torch.rand(2, 1100, 2, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"))
    d_o = torch.randn(v.shape, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(BF)

    def call(scale):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v * scale, s * scale)]
        o, final = linear_attention(*leaves[:3], d, initial_state=leaves[3], return_state=True)
        _, _, dv, ds = torch.autograd.grad(o, leaves, d_o * scale, retain_graph=True)
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v, s)]
        dq, dk = torch.autograd.grad(linear_attention(*leaves[:3], d, initial_state=leaves[3]), leaves[:2], d_o * scale)
        return [t.detach() / scale for t in (o, final, dv, ds, dq, dk)]
    for name, x, y in zip(("o", "state", "dv", "ds", "dq", "dk"), call(2.0 ** exponent), call(1.0)):
        assert bool(torch.isfinite(x).all()), name
        # (results that are themselves below the smallest normal float, or their parts, may differ)
        assert torch.equal(x, y) or float((x.double() - y.double()).abs().max()) <= 1e-6 * float(y.abs().max()), name
