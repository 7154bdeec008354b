"""The serving loop over the paged 4-bit cache (batch_step.BatchStack): prompts
and decode steps against a float32 recomputation over the held rows, graph
replays equal to eager steps, penalties and masks at work."""
from __future__ import annotations

import math

import pytest
import torch

import kv4_oracle as oracle
from drinkme_b200 import batch_step, radix_ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SMALL = dict(layers=2, hidden=1024, inter=2048, heads=8, kv_heads=2, head_dim=128, vocab=1000)


def float32_logits(st, b, token, p):
    """Logits of sequence b's token at position p, recomputed in float32 with
    the rows that the cache holds."""
    s = st.s
    nh, nkv, hd, I = s["heads"], s["kv_heads"], s["head_dim"], s["inter"]

    def rms(x, w):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + batch_step.EPS) * w.float()

    h = st.w.embed[token].float()[None]
    for lay, cache in zip(st.w.layers, st.caches):
        W = {k: radix_ops.decode_weight(lay[k]).float() for k in ("qkv", "o", "gate_up", "down")}
        qkv = rms(h, lay["ln1"]) @ W["qkv"].T
        q = rms(qkv[0, : nh * hd].view(nh, hd), lay["qn"])
        c, sn, half = st.cos[p], st.sin[p], hd // 2
        q = torch.cat([q[:, :half] * c - q[:, half:] * sn, q[:, half:] * c + q[:, :half] * sn], -1)
        K, V, _ = oracle.held(cache.codes.cpu(), cache.scales.cpu(), st.table.cpu(), b, p + 1)
        K, V = K.float().to(DEV), V.float().to(DEV)
        a = torch.softmax(torch.matmul(q.view(nkv, nh // nkv, hd), K.transpose(1, 2)) / math.sqrt(hd), -1)
        h = h + torch.matmul(a, V).reshape(1, nh * hd) @ W["o"].T
        gu = rms(h, lay["ln2"]) @ W["gate_up"].T
        h = h + (torch.nn.functional.silu(gu[:, :I]) * gu[:, I:]) @ W["down"].T
    return (rms(h, st.w.norm) @ st.w.head.float().T)[0]


def test_prompts_then_steps_track_float32_and_graphs_equal_eager():
    prompts = [[1, 2, 3, 4, 5], [7], list(range(100, 170))]
    a = batch_step.BatchStack(SMALL, DEV, seqs=3, max_len=200, page=16, seed=3)
    b = batch_step.BatchStack(SMALL, DEV, seqs=3, max_len=200, page=16, seed=3)
    for st in (a, b):
        st.prefill(prompts)
    for i, p in enumerate(prompts):
        ref = float32_logits(a, i, p[-1], len(p) - 1)
        assert (a.logits[i].float() - ref).norm() / ref.norm() < 3e-2  # bf16 activations between the ops vs float32
    b.capture()
    for n in range(5):
        fed = a.token.clone()
        a.step()
        b.replay()
        assert torch.equal(a.logits, b.logits) and torch.equal(a.token, b.token) and torch.equal(a.history, b.history)
        for i, p in enumerate(prompts):
            ref = float32_logits(a, i, int(fed[i]), len(p) + n)
            assert (a.logits[i].float() - ref).norm() / ref.norm() < 3e-2
    a.batch.check()
    assert a.kv_len.tolist() == [len(p) + 5 for p in prompts] and a.total_len.tolist() == [len(p) + 6 for p in prompts]


def test_masks_and_penalties_reach_the_choice():
    st = batch_step.BatchStack(SMALL, DEV, seqs=2, max_len=64, page=16, seed=5)
    st.allowed = torch.full((2, 32), -1, dtype=torch.int32, device=DEV)
    st.allowed[1] = 0
    st.allowed[1, 3] = 1 << 7  # the second sequence may say token 103 only
    st.frequency.fill_(1000.0)  # nobody says a token twice
    st.prefill([[1, 2], [3]])
    said = [st.token.clone()]
    for _ in range(6):
        st.replay()
        said.append(st.token.clone())
    said = torch.stack(said, 1).tolist()
    assert len(set(said[0])) == 7 and said[1] == [103] * 7


def test_refusals():
    with pytest.raises(ValueError):
        batch_step.BatchStack(SMALL, DEV, seqs=9)
    st = batch_step.BatchStack(SMALL, DEV, seqs=1, max_len=16, page=16)
    for bad in ([], [[]], [[1] * 16], [[1], [2]]):
        with pytest.raises(ValueError):
            st.prefill(bad)
