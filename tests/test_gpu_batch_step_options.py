"""The serving loop's request options (masks, penalties) when they are set or
replaced after the step was captured."""
from __future__ import annotations

import pytest
import torch

from drinkme_b200 import batch_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SMALL = dict(layers=1, hidden=1024, inter=2048, heads=8, kv_heads=2, head_dim=128, vocab=1000)


def only(tokens):
    """A mask of one row a sequence, each of which may say its one token."""
    m = torch.zeros(len(tokens), 32, dtype=torch.int32, device=DEV)
    for b, t in enumerate(tokens):
        m[b, t // 32] = (1 << (t % 32)) if t % 32 < 31 else -(1 << 31)
    return m


def captured():
    st = batch_step.BatchStack(SMALL, DEV, seqs=2, max_len=64, page=16, seed=5)
    st.prefill([[1, 2], [3]])
    st.capture()
    return st


def test_a_mask_given_after_the_capture_is_obeyed():
    st = captured()
    st.replay()
    st.allowed = only([103, 41])
    st.replay()
    assert st.token.tolist() == [103, 41]
    st.allowed = only([31, 999])  # another tensor
    st.replay()
    assert st.token.tolist() == [31, 999]
    st.allowed.copy_(only([7, 8]))  # the same one, other contents
    st.replay()
    assert st.token.tolist() == [7, 8]
    st.allowed[1] = -1  # a row of its own
    st.allowed[0] = only([64])[0]
    st.replay()
    assert st.token[0].item() == 64


def test_a_mask_filled_in_place_needs_no_assignment():
    st = captured()
    st.allowed.copy_(only([500, 501]))
    st.replay()
    assert st.token.tolist() == [500, 501]


def test_options_replaced_after_the_capture_are_those_of_an_eager_step():
    a, b = captured(), captured()
    for name, value in (("repetition", 1.7), ("presence", 3.0), ("frequency", 0.9)):
        for st in (a, b):
            setattr(st, name, torch.full((2,), value, device=DEV))
        for _ in range(2):
            a.step()
            b.replay()
            assert torch.equal(a.logits, b.logits) and torch.equal(a.token, b.token), name
    a.allowed = b.allowed = None
    a.step()
    b.replay()
    assert torch.equal(a.logits, b.logits)
