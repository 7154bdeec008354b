"""A vocabulary that the kernel's 32-bit counts cannot hold is refused."""
from __future__ import annotations

import pytest
import torch

from drinkme_b200 import logits

pytestmark = pytest.mark.gpu


def test_a_vocabulary_past_32_bits_is_refused():
    x = torch.zeros(1, (1 << 32) + 5, dtype=torch.bfloat16, device="cuda:0")  # 8.6 GB
    with pytest.raises(ValueError, match="vocabulary"):
        logits.process(x, out=x)
