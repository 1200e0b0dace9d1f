"""The linear attention's C interface without a device."""
import ctypes

import pytest

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


@pytest.mark.parametrize("shape", [dict(B=1, T=196, H=5, G=5, K=64, V=64), dict(B=6, T=1395, H=3, G=3, K=64, V=64), dict(B=2, T=2561, H=2, G=1, K=128, V=128), dict(B=64, T=1000, H=16, G=16, K=64, V=64)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_a_workspace_query_needs_no_pointers(L, shape, dtype):  # noqa: F811
    """The same with and without lengths: a caller may ask before there are any tensors."""
    for query, more in ((L.m2d_attn_fwd_workspace, {}), (L.m2d_attn_bwd_workspace, {}), (L.m2d_attn_bwd_workspace, {"d_log_decay": 256})):
        without, with_lengths = (query(ctypes.byref(attn(dtype=dtype, **shape, **more, **kw))) for kw in ({}, {"lengths": 256}))
        assert without == with_lengths
