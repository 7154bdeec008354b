"""Logits operators (drinkme_b200.logits) over histories and biases longer than
the fields of a packed entry hold."""
from __future__ import annotations

import pytest
import torch

from drinkme_b200 import logits
from test_gpu_logits import check, inputs, on

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [500, 9001])
@pytest.mark.parametrize("n,k", [(70000, 0), (70000, 40), (100, 33000)])
def test_long_histories_and_biases(dtype, vocab, n, k):
    x, a = inputs(2, vocab, n, k, dtype, seed=vocab + n + k)
    if n > 65535:
        a["total_len"][0] = n
        a["history"][0, 1000:] = 7  # a count past 16 bits
    check(logits.process(x.to("cuda:0"), **on(a)), x, a)
    y = x.to("cuda:0")
    check(logits.process(y, **on(a), out=y), x, a)
