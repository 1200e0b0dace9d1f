"""What the distillation loss and the C ABI of the recurrent layers refuse, without a device: sizes beyond 32 bits, misaligned fp32 arrays."""
import ctypes

import pytest
import torch

from mamba2d_b200 import distillation_loss
from test_layers_host import LARGE, L, PITCH, DistillDesc, LnDesc, RecurDesc, RecurTensor  # noqa: F401


def test_more_classes_than_32_bits_count():
    """A number of classes whose lower 32 bits look like a small one."""
    for V in (1 << 31, (1 << 32) + 100):
        z, t, index = torch.zeros(1).expand(1, V), torch.zeros(1, 4), torch.zeros(1, 4, dtype=torch.long)
        with pytest.raises(RuntimeError, match="out of range"):
            distillation_loss(z, t, index)


def test_alignment_of_the_recurrences_arrays(L):  # noqa: F811
    t = RecurTensor(256, 64, 64)
    names = ("lengths", "state", "state_out", "marks", "d_state_out", "d_state")

    def desc(**kw):
        d = RecurDesc(struct_bytes=ctypes.sizeof(RecurDesc), dtype=1, B=2, T=100, C=64, form=0, x=t, gate=t, d_y=t, **{**dict.fromkeys(("y", "d_x", "d_gate", *names), 256), **kw})
        return ctypes.byref(d)
    for n in names:
        for off in (257, 258):
            assert L.m2d_recur_fwd(desc(**{n: off}), None) == PITCH and L.m2d_recur_bwd(desc(**{n: off}), None) == PITCH, n
    for n in ("state", "state_out"):
        d = RecurDesc(struct_bytes=ctypes.sizeof(RecurDesc), dtype=1, B=2, T=1, C=64, form=0, x=t, gate=t, **{**dict.fromkeys(("y", "state", "state_out"), 256), n: 258})
        assert L.m2d_recur_step(ctypes.byref(d), ctypes.c_int64(64), None) == PITCH


def test_alignment_of_the_norms_statistics(L):  # noqa: F811
    """Pairs of floats."""
    for off in (258, 260):
        d = LnDesc(struct_bytes=ctypes.sizeof(LnDesc), dtype=1, N=10, C=64, eps=1e-5, x=256, x_row=64, y=256, d_y=256, d_y_row=64, d_x=256, stats=off)
        assert L.m2d_ln_fwd(ctypes.byref(d), None) == PITCH and L.m2d_ln_bwd(ctypes.byref(d), None) == PITCH


def test_alignment_of_the_distillations_arrays(L):  # noqa: F811
    for n in ("loss", "stats", "d_loss"):
        d = DistillDesc(struct_bytes=ctypes.sizeof(DistillDesc), V=100, K=8, N=10, temperature=2.0, **{**dict.fromkeys(("logits", "teacher", "index", "loss", "stats", "d_loss", "d_logits"), 256), n: 258})
        assert L.m2d_distill_fwd(ctypes.byref(d), None) == PITCH and L.m2d_distill_bwd(ctypes.byref(d), None) == PITCH, n
