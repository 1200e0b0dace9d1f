"""Calls of the linear attention that its documentation allows and its own tests do not make.  Tolerances are those of its
own tests (see test_attention_gpu.py) where nothing else is said."""
import pytest
import torch

from mamba2d_b200 import linear_attention

pytestmark = pytest.mark.gpu


def test_as_many_tokens_as_there_may_be():
    """Just below 2^31 tokens, in segments whose last would end behind 2^31.  All tokens are the same one: o is the geometric
    series, 2 - 2^-t, which bf16 cannot tell from 2 after ten tokens."""
    T = 2 ** 31 - 2049
    one = torch.ones(1, 1, 1, 1, dtype=torch.bfloat16, device="cuda").expand(1, T, 1, 1)
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
