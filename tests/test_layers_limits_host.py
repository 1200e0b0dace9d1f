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
