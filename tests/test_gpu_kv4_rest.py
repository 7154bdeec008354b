"""Rows of the attention's output that no sequence's tokens are: zeros, as append
and read give them."""
from __future__ import annotations

import pytest
import torch

from drinkme_b200 import _lib, kv4
from test_gpu_kv4 import DEV, make, queries

pytestmark = pytest.mark.gpu


def starts(*at):
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def poisoned(q, dtype=torch.bfloat16):
    return torch.full_like(q, float("nan"), dtype=dtype)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh", [2, 8, 20, 34])  # a single token's rows a kv head: 1, 4, 10, 17
@pytest.mark.parametrize("cut", [[1], [1, 1, 1], [5, 0, 2], [40], [30, 1], [1, 70, 3]])
def test_padding_before_between_and_after(hd, nh, cut):
    lens = [50 + 7 * i for i in range(len(cut))]
    cache, table = make(2, hd, 16, lens, seed=nh)
    T, before, after = sum(cut), 3, 9
    q = queries(before + T + after, nh, hd)
    q[:before] = float("nan")  # padding may hold anything
    q[before + T:] = float("nan")
    at = [before]
    for n in cut:
        at.append(at[-1] + n)
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = kv4.attention(cache, kv4.Batch(table, starts(*(a - before for a in at)), kv_len, tokens=T, max_q=max(cut)),
                         q[before:before + T].contiguous())
    for dtype in (torch.bfloat16, torch.float32):
        batch = kv4.Batch(table, starts(*at), kv_len, tokens=len(q), max_q=max(cut))
        out = kv4.attention(cache, batch, q, out=poisoned(q, dtype))
        batch.check()  # padding is no error
        assert torch.equal(out[before:before + T].to(torch.bfloat16), want)
        assert bool((out[:before] == 0).all()) and bool((out[before + T:] == 0).all())


@pytest.mark.parametrize("max_q", [2, 30])
def test_a_refused_sequence_is_zeros_and_reported(max_q):
    """More new tokens than max_q: the sequence is left out, the others are not."""
    cut, lens = [1, max_q + 3, 2], [60, 90, 70]
    cache, table = make(2, 128, 16, lens, seed=1)
    T = sum(cut)
    q = queries(T, 8, 128)
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    batch = kv4.Batch(table, starts(0, 1, T - 2, T), kv_len, tokens=T, max_q=max_q)
    out = kv4.attention(cache, batch, q, out=poisoned(q))
    with pytest.raises(_lib.DrinkmeError, match="not covered"):
        batch.check()
    # the split of the work may differ from the smaller batch's: two roundings of 2^-8
    alone = kv4.attention(cache, kv4.Batch(table, starts(0, 1, 1, 3), kv_len, tokens=3, max_q=2),
                          torch.cat((q[:1], q[-2:])))
    assert bool((out[1:-2] == 0).all())
    got = torch.cat((out[:1], out[-2:]))
    assert not bool(got.isnan().any()) and float((got.float() - alone.float()).norm() / alone.float().norm()) < 2.0 ** -7


def test_a_graph_for_more_tokens_leaves_zeros_behind():
    """Captured for 64 tokens, replayed with fewer: what an earlier replay left is gone."""
    cache, table = make(2, 128, 64, [400, 400], seed=2)
    q = queries(64, 8, 128)
    batch = kv4.Batch(table, starts(0, 60, 64), starts(300, 350), tokens=64, max_q=64)
    out = kv4.attention(cache, batch, q)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        kv4.attention(cache, batch, q, out=out)
    for at in ((0, 60, 64), (0, 1, 2), (0, 0, 0), (0, 40, 40), (0, 3, 60)):
        batch.q_start.copy_(torch.tensor(at, dtype=torch.int32))
        graph.replay()
        batch.check()
        assert bool((out[at[-1]:] == 0).all()) and bool((out[: at[-1]] != 0).any(-1).all()), at
