"""Sliding windows over a table whose pages before the window have been given
back: the same bits as with every page there, and nothing is reported."""
from __future__ import annotations

import pytest
import torch

from drinkme_b200 import _lib, kv4
from test_gpu_kv4 import DEV, make, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("gone", [-1, 1 << 30])
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [5, 2, 5, 1], [40, 9, 70, 64], [300, 1, 30, 7]])
@pytest.mark.parametrize("window", [1, 33, 100, 257])
def test_pages_before_the_window_need_not_be_there(page, gone, q_lens, window):
    lens = [313, 501, 777, 1031]
    cache, table = make(2, 128, page, lens, seed=page)
    q = queries(sum(q_lens), 8, 128)
    want = kv4.attention(cache, kv4.Batch.of(table, q_lens, lens), q, window=window)
    cut = table.clone()
    for b, (n, length) in enumerate(zip(q_lens, lens)):
        first = max(0, length - n - window + 1)  # the first position that a new token of b sees
        cut[b, : first // page] = gone
    batch = kv4.Batch.of(cut, q_lens, lens)
    got = kv4.attention(cache, batch, q, window=window)
    batch.check()
    assert torch.equal(got, want)


@pytest.mark.parametrize("q_len", [1, 40])
def test_a_missing_page_inside_the_window_is_still_reported(q_len):
    cache, table = make(2, 128, 16, [313], seed=3)
    cut = table.clone()
    cut[0, (313 - q_len - 100 + 1) // 16] = -1  # holds the first token's first position
    batch = kv4.Batch.of(cut, [q_len], [313])
    kv4.attention(cache, batch, queries(q_len, 8, 128), window=100)
    with pytest.raises(_lib.DrinkmeError, match="not covered"):
        batch.check()
    assert DEV == str(cache.device)
