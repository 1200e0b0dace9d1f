"""The linear attention's C interface without a device."""
import ctypes

from test_sequence_host import FLAGS, NULL, L, attn  # noqa: F401  (L is a fixture)


def test_there_are_no_flags(L):  # noqa: F811
    for fn in (L.m2d_attn_fwd, L.m2d_attn_bwd):
        assert fn(ctypes.byref(attn(flags=1)), None) == FLAGS


def test_the_hook_is_refused_without_the_environment_variable(L, monkeypatch):  # noqa: F811
    for fn in (L.m2d_attn_fwd, L.m2d_attn_bwd):
        monkeypatch.delenv("M2D_TEST_HOOKS", raising=False)
        assert fn(ctypes.byref(attn(flags=0x100)), None) == FLAGS
        monkeypatch.setenv("M2D_TEST_HOOKS", "1")
        assert fn(ctypes.byref(attn(flags=0x100)), None) == NULL        # accepted: next check
        assert fn(ctypes.byref(attn(flags=0x101)), None) == FLAGS
