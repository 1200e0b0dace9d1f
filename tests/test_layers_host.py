"""The gated recurrence without a device: refusals of the Python entry points and of the C ABI."""
import ctypes

import pytest
import torch

import mamba2d_b200
from mamba2d_b200 import _lib, gated_recurrence, gated_recurrence_step

OK, NULL, DTYPE, SHAPE, WORKSPACE, ABI, LARGE, FLAGS, PITCH = 0, -1, -2, -3, -6, -8, -9, -10, -5


class RecurTensor(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("batch", ctypes.c_int64), ("token", ctypes.c_int64)]


class RecurDesc(ctypes.Structure):
    """Mirror of ``m2d_recur_desc``."""
    _fields_ = [("struct_bytes", ctypes.c_uint32), *[(n, ctypes.c_int32) for n in ("dtype", "B", "T", "C", "form")], ("x", RecurTensor), ("gate", RecurTensor),
                *[(n, ctypes.c_void_p) for n in ("lengths", "state", "state_out", "y", "marks")], ("d_y", RecurTensor),
                *[(n, ctypes.c_void_p) for n in ("d_state_out", "d_x", "d_gate", "d_state")]]


@pytest.fixture(scope="module")
def L():
    from mamba2d_b200 import build
    build.build()
    raw = ctypes.CDLL(_lib.LIB_PATH)
    raw.m2d_recur_marks.restype = ctypes.c_uint64
    return raw


def test_recurrence_descriptors(L):
    t = RecurTensor(256, 0, 0)

    def desc(**kw):
        d = RecurDesc(struct_bytes=ctypes.sizeof(RecurDesc), dtype=0, B=2, T=100, C=64, form=0, x=t, gate=t)
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)
    for kw, rc in (({}, NULL), ({"struct_bytes": 8}, ABI), ({"dtype": 2}, DTYPE), ({"form": 2}, FLAGS), ({"B": 0}, SHAPE), ({"T": 0}, SHAPE), ({"C": -1}, SHAPE),
                   ({"T": (1 << 31) - 1}, LARGE), ({"B": 1 << 27}, LARGE), ({"x": RecurTensor(None, 0, 0)}, NULL), ({"gate": RecurTensor(258, 0, 0)}, PITCH)):
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


def test_the_package_has_the_recurrence():
    for n in ("gated_recurrence", "gated_recurrence_step"):
        assert n in mamba2d_b200.__all__ and callable(getattr(mamba2d_b200, n))
