"""The gated recurrence, layer normalisation and the distillation loss without a device: refusals of the Python entry points and of the C ABI."""
import ctypes

import pytest
import torch

import mamba2d_b200
from mamba2d_b200 import _lib, distillation_loss, gated_recurrence, gated_recurrence_step, layer_norm

OK, NULL, DTYPE, SHAPE, WORKSPACE, ABI, LARGE, FLAGS, PITCH = 0, -1, -2, -3, -6, -8, -9, -10, -5


class RecurTensor(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("batch", ctypes.c_int64), ("token", ctypes.c_int64)]


class RecurDesc(ctypes.Structure):
    """Mirror of ``m2d_recur_desc``."""
    _fields_ = [("struct_bytes", ctypes.c_uint32), *[(n, ctypes.c_int32) for n in ("dtype", "B", "T", "C", "form")], ("flags", ctypes.c_uint32), ("x", RecurTensor), ("gate", RecurTensor),
                *[(n, ctypes.c_void_p) for n in ("lengths", "state", "state_out", "y", "marks")], ("d_y", RecurTensor),
                *[(n, ctypes.c_void_p) for n in ("d_state_out", "d_x", "d_gate", "d_state")]]


class LnDesc(ctypes.Structure):
    """Mirror of ``m2d_ln_desc``."""
    _fields_ = [("struct_bytes", ctypes.c_uint32), ("dtype", ctypes.c_int32), ("N", ctypes.c_int64), ("C", ctypes.c_int32), ("params_f32", ctypes.c_int32), ("eps", ctypes.c_float),
                ("x", ctypes.c_void_p), ("x_row", ctypes.c_int64), ("residual", ctypes.c_void_p), ("residual_row", ctypes.c_int64),
                *[(n, ctypes.c_void_p) for n in ("weight", "bias", "sum", "y", "stats", "d_y")], ("d_y_row", ctypes.c_int64), ("d_sum", ctypes.c_void_p), ("d_sum_row", ctypes.c_int64),
                *[(n, ctypes.c_void_p) for n in ("d_x", "d_weight", "d_bias", "workspace")], ("workspace_bytes", ctypes.c_uint64)]


class DistillDesc(ctypes.Structure):
    """Mirror of ``m2d_distill_desc``."""
    _fields_ = [("struct_bytes", ctypes.c_uint32), *[(n, ctypes.c_int32) for n in ("dtype", "teacher_dtype", "V", "K", "index_64", "labels_64")],
                ("temperature", ctypes.c_float), ("label_weight", ctypes.c_float), ("N", ctypes.c_int64), ("logits", ctypes.c_void_p), ("logits_row", ctypes.c_int64),
                ("teacher", ctypes.c_void_p), ("teacher_row", ctypes.c_int64), ("index", ctypes.c_void_p), ("index_row", ctypes.c_int64),
                *[(n, ctypes.c_void_p) for n in ("labels", "loss", "stats", "d_loss")], ("d_loss_row", ctypes.c_int64), ("d_logits", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


@pytest.fixture(scope="module")
def L():
    from mamba2d_b200 import build
    build.build()
    raw = ctypes.CDLL(_lib.LIB_PATH)
    raw.m2d_recur_marks.restype = raw.m2d_ln_bwd_workspace.restype = raw.m2d_distill_stats.restype = raw.m2d_distill_fwd_workspace.restype = ctypes.c_uint64
    return raw


def test_recurrence_descriptors(L):
    t = RecurTensor(256, 0, 0)

    def desc(**kw):
        d = RecurDesc(struct_bytes=ctypes.sizeof(RecurDesc), dtype=0, B=2, T=100, C=64, form=0, x=t, gate=t)
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)
    for kw, rc in (({}, NULL), ({"struct_bytes": 8}, ABI), ({"dtype": 2}, DTYPE), ({"form": 2}, FLAGS), ({"flags": 0x100}, FLAGS), ({"flags": 1}, FLAGS), ({"B": 0}, SHAPE), ({"T": 0}, SHAPE), ({"C": -1}, SHAPE),
                   ({"T": (1 << 31) - 1}, LARGE), ({"B": 1 << 27}, LARGE), ({"x": RecurTensor(None, 0, 0)}, NULL), ({"gate": RecurTensor(258, 0, 0)}, PITCH), ({"y": 258}, PITCH), ({"d_x": 257}, PITCH), ({"C": (1 << 29) + 1}, LARGE)):
        assert L.m2d_recur_fwd(desc(**kw), None) == rc and L.m2d_recur_bwd(desc(**kw), None) == rc, kw
    step = lambda **kw: L.m2d_recur_step(desc(**kw), ctypes.c_int64(64), None)  # noqa: E731
    assert step() == SHAPE and step(T=1) == NULL and step(T=1, y=256, state=256) == NULL and L.m2d_recur_fwd(None, None) == NULL
    assert L.m2d_recur_bwd(desc(d_y=t, d_x=256, d_gate=256), None) == NULL               # no marks
    assert L.m2d_recur_marks(desc()) == 2 * 2 * 64 and L.m2d_recur_marks(desc(T=0)) == 0


def test_refusals_of_the_recurrence():
    x, g, s = torch.randn(2, 5, 8), torch.randn(2, 5, 8), torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="CUDA device"):
        gated_recurrence(x, g)
    for args in ((x, g[:, :4]), (x[0], g[0]), (x, g.bfloat16()), (x.half(), g.half()), (x.double(), g.double()), (x, g[..., :1])):
        with pytest.raises(RuntimeError):
            gated_recurrence(*args)
    for state in (s[:1], s.double(), s.bfloat16(), s[..., :7], s[:, None]):
        with pytest.raises(RuntimeError):
            gated_recurrence(x, g, initial_state=state)
        with pytest.raises(RuntimeError):
            gated_recurrence_step(x[:, 0], g[:, 0], state)
    for form in ("keep", None, 0):
        with pytest.raises(ValueError):
            gated_recurrence(x, g, form=form)
        with pytest.raises(ValueError):
            gated_recurrence_step(x[:, 0], g[:, 0], s, form=form)
    with pytest.raises(RuntimeError):
        gated_recurrence_step(x[:, 0], g[:, 0], None)


def test_layer_norm_descriptors(L):
    def desc(**kw):
        d = LnDesc(struct_bytes=ctypes.sizeof(LnDesc), dtype=1, N=10, C=64, eps=1e-5)
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)
    for kw, rc in (({}, NULL), ({"struct_bytes": 8}, ABI), ({"dtype": 2}, DTYPE), ({"N": 0}, SHAPE), ({"C": 0}, SHAPE), ({"N": 1 << 31}, LARGE), ({"C": (1 << 30) + 1}, LARGE), ({"x": 257}, PITCH), ({"weight": 258, "params_f32": 1}, PITCH), ({"d_x": 255}, PITCH)):
        assert L.m2d_ln_fwd(desc(**kw), None) == rc and L.m2d_ln_bwd(desc(**kw), None) == rc, kw
    assert L.m2d_ln_fwd(None, None) == NULL and L.m2d_ln_fwd(desc(x=256, y=256, residual=256), None) == NULL        # nowhere to put the sum
    p = dict(x=256, x_row=64, d_y=256, d_y_row=64, d_x=256, stats=256, d_weight=256)
    need = L.m2d_ln_bwd_workspace(desc(**p))
    assert need >= 2 * 4 * 64 and L.m2d_ln_bwd_workspace(desc(**{**p, "d_weight": None})) == 0
    for kw in ({}, {"workspace": 256, "workspace_bytes": need - 1}, {"workspace": 128, "workspace_bytes": need}):
        assert L.m2d_ln_bwd(desc(**p, **kw), None) == WORKSPACE


def test_refusals_of_layer_norm():
    x, w = torch.randn(3, 12), torch.randn(12)
    with pytest.raises(RuntimeError, match="CUDA device"):
        layer_norm(x, w, w, residual=x)
    for args, kw in (((x.half(),), {}), ((x.double(),), {}), ((x, w[:5]), {}), ((x, w.bfloat16()), {}), ((x, w, w.double()), {}), ((x, w[None]), {}), ((x.sum(),), {}),
                     ((x,), {"residual": x[:2]}), ((x,), {"residual": x.bfloat16()}), ((x,), {"residual": x[0]})):
        with pytest.raises(RuntimeError):
            layer_norm(*args, **kw)
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            layer_norm(x, eps=eps)


def test_distillation_descriptors(L):
    def desc(**kw):
        d = DistillDesc(struct_bytes=ctypes.sizeof(DistillDesc), V=100, K=8, N=10, temperature=2.0, logits=256, teacher=256, index=256)
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)
    for kw, rc in (({}, NULL), ({"struct_bytes": 8}, ABI), ({"dtype": 2}, DTYPE), ({"teacher_dtype": -1}, DTYPE), ({"N": 0}, SHAPE), ({"V": 0}, SHAPE), ({"K": 0}, SHAPE), ({"K": 513}, LARGE),
                   ({"N": 1 << 26}, LARGE), ({"V": (1 << 31) - 1}, LARGE), ({"temperature": 0.0}, FLAGS), ({"temperature": float("nan")}, FLAGS), ({"temperature": float("inf")}, FLAGS),
                   ({"label_weight": 1.5}, FLAGS), ({"label_weight": 0.5}, NULL), ({"logits": None}, NULL), ({"index": None}, NULL), ({"logits": 258}, PITCH), ({"index": 260, "index_64": 1}, PITCH), ({"d_logits": 2}, PITCH)):
        assert L.m2d_distill_fwd(desc(**kw), None) == rc and L.m2d_distill_bwd(desc(**kw), None) == rc, kw
    assert L.m2d_distill_fwd(None, None) == NULL and L.m2d_distill_stats(desc()) > 0
    assert L.m2d_distill_fwd_workspace(desc()) == 0                                       # (short rows)
    need = L.m2d_distill_fwd_workspace(desc(V=50000))
    for kw in ({}, {"workspace": 256, "workspace_bytes": need - 1}, {"workspace": 128, "workspace_bytes": need}):
        assert L.m2d_distill_fwd(desc(V=50000, loss=256, **kw), None) == WORKSPACE


def test_refusals_of_the_distillation_loss():
    z, t, i, n = torch.randn(4, 20), torch.randn(4, 3), torch.zeros(4, 3, dtype=torch.long), torch.zeros(4, dtype=torch.long)
    with pytest.raises(RuntimeError, match="CUDA device"):
        distillation_loss(z, t, i)
    for args, kw in (((z.half(), t, i), {}), ((z, t.double(), i), {}), ((z, t, i.short()), {}), ((z, t[:3], i[:3]), {}), ((z, t, i[:, :2]), {}), ((z, t[:, :0], i[:, :0]), {}),
                     ((z, t[0], i[0]), {}), ((z, torch.zeros(4, 600), torch.zeros(4, 600, dtype=torch.long)), {}), ((z, t, i, n[:3]), {"label_weight": 0.5}),
                     ((z, t, i, n.float()), {"label_weight": 0.5}), ((z[:, :0], t, i), {})):
        with pytest.raises(RuntimeError):
            distillation_loss(*args, **kw)
    for args, kw in (((z, t, i), {"temperature": 0.0}), ((z, t, i), {"temperature": float("nan")}), ((z, t, i), {"temperature": float("inf")}), ((z, t, i), {"temperature": 1e-60}),
                     ((z, t, i, n), {"label_weight": 1.1}), ((z, t, i, n), {"label_weight": -0.1}), ((z, t, i, n), {}), ((z, t, i), {"label_weight": 0.5})):
        with pytest.raises(ValueError):
            distillation_loss(*args, **kw)


def test_the_package_has_them():
    for n in ("distillation_loss", "gated_recurrence", "gated_recurrence_step", "layer_norm"):
        assert n in mamba2d_b200.__all__ and callable(getattr(mamba2d_b200, n))
