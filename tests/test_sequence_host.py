"""Sequence operators without a device: refusals of the Python entry points and of the C ABI, and workspace planning."""
import ctypes

import pytest
import torch

import mamba2d_b200
from mamba2d_b200 import _lib, clip_grad_norm_, clip_norm_, group_norm, linear_attention, linear_attention_step


class Tensor(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("batch", ctypes.c_int64), ("token", ctypes.c_int64), ("head", ctypes.c_int64)]


class AttnDesc(ctypes.Structure):
    """Mirror of ``m2d_attn_desc``."""
    _fields_ = [("struct_bytes", ctypes.c_uint32), ("dtype", ctypes.c_int32), *[(n, ctypes.c_int32) for n in "BTHGKV"], ("flags", ctypes.c_uint32),
                ("scale", ctypes.c_float), ("q", Tensor), ("k", Tensor), ("v", Tensor), ("log_decay", ctypes.c_void_p),
                *[(n, ctypes.c_int64) for n in ("g_batch", "g_token", "g_head")],
                *[(n, ctypes.c_void_p) for n in ("lengths", "state", "state_out", "o")], ("d_o", Tensor),
                *[(n, ctypes.c_void_p) for n in ("d_state_out", "d_q", "d_k", "d_v", "d_log_decay", "d_state", "workspace")], ("workspace_bytes", ctypes.c_uint64)]


class NormDesc(ctypes.Structure):
    """Mirror of ``m2d_norm_desc``."""
    _fields_ = [("struct_bytes", ctypes.c_uint32), ("dtype", ctypes.c_int32), ("N", ctypes.c_int64), ("S", ctypes.c_int64),
                *[(n, ctypes.c_int32) for n in ("C", "groups", "act", "params_f32")], ("eps", ctypes.c_float),
                *[(n, ctypes.c_void_p) for n in ("x", "weight", "bias", "y", "stats", "d_y", "d_x", "d_weight", "d_bias", "workspace")],
                ("workspace_bytes", ctypes.c_uint64)]


class ClipTensor(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("elements", ctypes.c_int64), ("dtype", ctypes.c_int32)]


@pytest.fixture(scope="module")
def L():
    from mamba2d_b200 import build
    build.build()
    raw = ctypes.CDLL(_lib.LIB_PATH)
    for n in ("m2d_attn_fwd_workspace", "m2d_attn_bwd_workspace", "m2d_norm_fwd_workspace", "m2d_norm_bwd_workspace", "m2d_clip_workspace"):
        getattr(raw, n).restype = ctypes.c_uint64
    return raw


def attn(**kw):
    d = AttnDesc(struct_bytes=ctypes.sizeof(AttnDesc), dtype=_lib.M2D_BF16, B=2, T=1000, H=4, G=2, K=64, V=128, scale=1.0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


OK, NULL, DTYPE, SHAPE, WORKSPACE, ABI, LARGE, FLAGS, PITCH = 0, -1, -2, -3, -6, -8, -9, -10, -5


def test_attention_descriptors(L):
    for kw, rc in (({}, NULL), ({"struct_bytes": 8}, ABI), ({"dtype": 7}, DTYPE), ({"flags": 1 << 20}, FLAGS), ({"G": 3}, SHAPE), ({"K": 257}, SHAPE), ({"V": 0}, SHAPE),
                   ({"T": 0}, SHAPE), ({"B": 1 << 23}, LARGE), ({"B": 1, "H": 1, "G": 1, "T": (1 << 31) - 1}, LARGE)):
        for fn in (L.m2d_attn_fwd, L.m2d_attn_bwd):
            assert fn(ctypes.byref(attn(**kw)), None) == rc, kw
    assert L.m2d_attn_fwd(None, None) == NULL
    t = Tensor(256, 0, 0, 0)
    full = dict(q=t, k=t, v=t, log_decay=256)
    assert L.m2d_attn_step(ctypes.byref(attn(**full)), ctypes.c_int64(0), ctypes.c_int64(0), None) == SHAPE      # T is not 1
    assert L.m2d_attn_step(ctypes.byref(attn(T=1, **full)), ctypes.c_int64(0), ctypes.c_int64(0), None) == NULL  # no state
    assert L.m2d_attn_fwd(ctypes.byref(attn(**full)), None) == NULL                                                # no output
    assert L.m2d_attn_bwd(ctypes.byref(attn(**full)), None) == NULL
    grads = dict(d_o=t, d_q=256, d_k=256, d_v=256, d_log_decay=256, **full)
    assert L.m2d_attn_bwd(ctypes.byref(attn(**grads)), None) == WORKSPACE
    need = L.m2d_attn_bwd_workspace(ctypes.byref(attn(**grads)))
    assert need and L.m2d_attn_bwd(ctypes.byref(attn(workspace=256, workspace_bytes=need - 1, **grads)), None) == WORKSPACE
    assert L.m2d_attn_bwd(ctypes.byref(attn(workspace=128, workspace_bytes=need, **grads)), None) == WORKSPACE
    assert L.m2d_attn_fwd_workspace(ctypes.byref(attn(G=3))) == 0


def test_attention_workspace_grows_with_what_is_asked(L):
    size = lambda **kw: L.m2d_attn_bwd_workspace(ctypes.byref(attn(B=64, H=16, G=16, **kw)))  # noqa: E731
    assert size() == 0                                           # the GPU is full without segments, nothing is shared
    assert size(d_log_decay=256) > 0
    assert L.m2d_attn_bwd_workspace(ctypes.byref(attn(B=64, H=16, G=4))) >= 2 * 4 * 64 * 1000 * 16 * 64
    assert L.m2d_attn_fwd_workspace(ctypes.byref(attn(B=1, T=65536, H=8))) > 0            # segments of a long sequence
    assert L.m2d_attn_fwd_workspace(ctypes.byref(attn(B=1, T=60, H=8))) == 0


def test_norm_and_clip_descriptors(L):
    def norm(**kw):
        d = NormDesc(struct_bytes=ctypes.sizeof(NormDesc), dtype=0, N=2, S=100, C=64, groups=4, eps=1e-5)
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)
    for kw, rc in (({}, NULL), ({"struct_bytes": 4}, ABI), ({"dtype": 3}, DTYPE), ({"act": 3}, FLAGS), ({"groups": 5}, SHAPE), ({"S": 0}, SHAPE), ({"N": 1 << 30}, LARGE), ({"C": 1 << 30, "groups": 1}, LARGE)):
        assert L.m2d_norm_fwd(norm(**kw), None) == rc and L.m2d_norm_bwd(norm(**kw), None) == rc
    p = dict(x=256, d_y=256, d_x=256, stats=256)
    assert L.m2d_norm_bwd(norm(d_weight=256, **p), None) == NULL                          # one of the two gradients
    assert L.m2d_norm_bwd(norm(d_weight=256, d_bias=256, **p), None) == WORKSPACE
    assert L.m2d_norm_bwd_workspace(norm(d_weight=256, d_bias=256)) > 0

    def clip(t, n=1, ws=256, size=1 << 20, norm=256):
        return L.m2d_clip_grad_norm(ctypes.byref(t), n, ctypes.c_float(1.0), ctypes.c_void_p(norm), ctypes.c_void_p(ws), ctypes.c_uint64(size), None)
    assert clip(ClipTensor(256, 10, 5)) == DTYPE and clip(ClipTensor(256, -1, 0)) == SHAPE and clip(ClipTensor(None, 3, 0)) == NULL
    assert clip(ClipTensor(258, 3, 0)) == PITCH and clip(ClipTensor(256, 3, 0), size=0) == WORKSPACE and clip(ClipTensor(256, 3, 0), norm=None) == NULL
    assert clip(ClipTensor(256, 3, 0), n=-1) == SHAPE


def test_refusals_of_the_python_entry_points():
    q, k, v, g, s = torch.randn(2, 5, 2, 8), torch.randn(2, 5, 2, 8), torch.randn(2, 5, 4, 6), -torch.rand(2, 5, 4), torch.zeros(2, 4, 8, 6)
    with pytest.raises(RuntimeError, match="CUDA device"):
        linear_attention(q, k, v, g)
    for args in ((q[:, :4], k, v, g), (q[..., :7], k, v, g), (q, k, v[0], g), (q.repeat(1, 1, 2, 1)[:, :, :3], k.repeat(1, 1, 2, 1)[:, :, :3], v, g),
                 (q, k, v, g[..., :2]), (q, k, v, g[0]), (q, k, v, g.long()), (q.double(), k, v, g), (q.half(), k.half(), v.half(), g),
                 (torch.randn(2, 5, 2, 300), torch.randn(2, 5, 2, 300), v, g), (q[..., :0], k[..., :0], v, g)):
        with pytest.raises(RuntimeError):
            linear_attention(*args)
    for state in (s[:1], s.double(), s.transpose(2, 3)):
        with pytest.raises(RuntimeError):
            linear_attention(q, k, v, g, initial_state=state)
    with pytest.raises(RuntimeError):
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], None)
    x = torch.randn(3, 7, 12)
    for kw in ({"groups": 5}, {"groups": 0}, {"groups": 3.0}, {"groups": 3, "act": "relu"}, {"groups": 3, "eps": -1.0}, {"groups": 3, "eps": float("nan")}):
        with pytest.raises(ValueError):
            group_norm(x, **kw)
    for args in ((x[0, 0], 3), (x.half(), 3), (x, 3)):
        with pytest.raises(RuntimeError):
            group_norm(*args)
    with pytest.raises(RuntimeError):
        clip_norm_([x], 1.0)
    with pytest.raises(ValueError):
        clip_norm_([x], -1.0)
    assert float(clip_norm_([], 1.0)) == 0.0 and float(clip_grad_norm_([torch.nn.Parameter(x)], 1.0)) == 0.0


def test_the_package_has_them():
    for n in ("linear_attention", "linear_attention_step", "group_norm", "clip_norm_", "clip_grad_norm_"):
        assert n in mamba2d_b200.__all__ and callable(getattr(mamba2d_b200, n))
