"""The linear attention's C interface without a device."""
import ctypes

from test_sequence_host import FLAGS, L, attn  # noqa: F401  (L is a fixture)


def test_there_are_no_flags(L):  # noqa: F811
    for fn in (L.m2d_attn_fwd, L.m2d_attn_bwd):
        assert fn(ctypes.byref(attn(flags=1)), None) == FLAGS
