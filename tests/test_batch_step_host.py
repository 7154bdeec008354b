"""What batch_step.BatchStack refuses on the host, and its history at the end of
the allocation (CPU: no kernel runs)."""
from __future__ import annotations

import pytest
import torch

from drinkme_b200 import batch_step


def stack(seqs=2, max_len=6, vocab=10):
    """A stack's host side and its small state on the CPU, without weights."""
    st = batch_step.BatchStack.__new__(batch_step.BatchStack)
    st.graph = None
    st.s, st.dev, st.seqs, st.max_len = dict(vocab=vocab, heads=1, kv_heads=1, head_dim=64, inter=1), torch.device("cpu"), seqs, max_len
    st.token = torch.zeros(seqs, dtype=torch.int64)
    st.history = torch.zeros(seqs, max_len + 1, dtype=torch.int32)
    st.prompt_len, st.total_len = torch.zeros(seqs, dtype=torch.int32), torch.zeros(seqs, dtype=torch.int32)
    st.last = torch.full((seqs,), max_len, dtype=torch.int64)
    st.repetition, st.presence, st.frequency = torch.ones(seqs), torch.zeros(seqs), torch.zeros(seqs)
    st.allowed = None
    st.logits = torch.randn(seqs, vocab)
    st.rows = [0] * seqs
    return st


def test_the_history_ends_where_the_allocation_does(monkeypatch):
    """Lengths past the allocation (as a device state that nobody counted would
    have them) index no column outside the history."""
    monkeypatch.setattr(batch_step.logits, "process", lambda x, **kw: kw["out"])
    st = stack()
    for _ in range(9):
        st._choose()
    assert st.total_len.tolist() == [9, 9] and st.history[:, 0].tolist() == st.token.tolist()


def test_a_step_past_the_allocation_is_refused_before_any_launch():
    class Graph:
        replays = 0

        def replay(self):
            self.replays += 1

    st, g = stack(max_len=6), Graph()
    st.graph, st.rows = g, [2, 4]
    done = []
    st._enqueue = lambda: done.append(1)
    st.step()
    st.replay()
    assert st.rows == [4, 6] and done == [1] and g.replays == 1
    for call in (st.step, st.replay, st.capture):
        with pytest.raises(ValueError, match="max_len"):
            call()
    assert st.rows == [4, 6] and done == [1] and g.replays == 1


def test_the_command_line_counts_its_steps():
    with pytest.raises(SystemExit):
        batch_step.main(["--prompt", "500", "--max-len", "512", "--steps", "20"])


@pytest.mark.parametrize("bad", [10, -1, 1 << 40])
def test_prompt_tokens_outside_the_vocabulary_are_refused(bad):
    st = stack(vocab=10)
    for prompts in ([[1, 2], [3, bad]], [[bad], [1]]):
        with pytest.raises(ValueError, match="vocabulary"):
            st.prefill(prompts)
    assert st.rows == [0, 0] and not st.history.any()


def test_options_of_another_shape_or_type_are_refused_when_given():
    st = stack(seqs=2, vocab=70)
    for name, bad in (("allowed", torch.zeros(2, 2, dtype=torch.int32)), ("allowed", torch.zeros(2, 3)),
                      ("allowed", torch.zeros(1, 3, dtype=torch.int32)), ("repetition", torch.ones(3)),
                      ("presence", torch.ones(2, dtype=torch.float64)), ("frequency", torch.ones(4)[::2])):
        kept = getattr(st, name)
        with pytest.raises(ValueError, match=name):
            setattr(st, name, bad)
        assert getattr(st, name) is kept
    st.allowed = torch.zeros(2, 3, dtype=torch.int32)
    st.repetition = None
