"""The serving loop at the end of a sequence's allocation: the host refuses the
step that has no row, before it is launched; and what the kernels recorded."""
from __future__ import annotations

import pytest
import torch

from drinkme_b200 import _lib, batch_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SMALL = dict(layers=1, hidden=1024, inter=2048, heads=8, kv_heads=2, head_dim=128, vocab=1000)


def test_sequences_run_to_the_end_of_their_allocation_and_no_further():
    st = batch_step.BatchStack(SMALL, DEV, seqs=2, max_len=16, page=16, seed=5)
    st.prefill([[1, 2, 3], [5] * 13])
    st.capture()
    st.replay()
    st.step()
    st.replay()  # the second sequence has its 16 rows
    kept = st.history.clone()
    for call in (st.replay, st.step, st.capture):
        with pytest.raises(ValueError, match="max_len"):
            call()
    st.batch.check()
    assert st.kv_len.tolist() == [6, 16] and st.total_len.tolist() == [7, 17] and torch.equal(st.history, kept)
    st.prefill([[1], [2]])  # and starts over
    st.replay()
    st.batch.check()
    assert st.kv_len.tolist() == [2, 2]


def test_what_the_kernels_recorded_is_raised_when_asked_for():
    st = batch_step.BatchStack(SMALL, DEV, seqs=2, max_len=64, page=16, seed=5)
    st.prefill([[1, 2, 3], [5] * 15])
    st.replay()
    st.check()
    st.table[1, 1] = -1  # the page of the second sequence's next rows
    st.replay()
    with pytest.raises(_lib.DrinkmeError, match="not covered"):
        st.check()
    st.check()  # said once
