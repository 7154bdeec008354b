"""The attention's workspace: made while a graph is captured, and two batches
at once on two streams."""
from __future__ import annotations

import pytest
import torch

from drinkme_b200 import kv4
from test_gpu_kv4 import DEV, make, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_len,length", [(1, 5000), (64, 3000)])
def test_a_workspace_first_needed_in_a_capture(q_len, length):
    """Calls before the graph's first replay, after it, and replays all give the
    answer, although the capture's memory held something else before."""
    cache, table = make(2, 128, 64, [length], seed=1)
    q = queries(q_len, 8, 128)
    want = kv4.attention(cache, kv4.Batch.of(table, [q_len], [length]), q)
    side = torch.cuda.Stream()
    used = torch.cuda.CUDAGraph()
    with torch.cuda.graph(used, stream=side):
        full = torch.full((64 << 20,), 255, dtype=torch.uint8, device=DEV)
    used.replay()
    torch.cuda.synchronize()
    del full  # the pool's memory, all ones
    batch = kv4.Batch.of(table, [q_len], [length])
    graph = torch.cuda.CUDAGraph()
    captured, eager = torch.empty_like(want), torch.empty_like(want)
    with torch.cuda.graph(graph, stream=side, pool=used.pool()):
        kv4.attention(cache, batch, q, out=captured)
        kv4.attention(cache, batch, q, out=captured)
    for turn in range(3):
        eager.fill_(float("nan"))
        kv4.attention(cache, batch, q, out=eager)
        assert torch.equal(eager, want), turn
        captured.fill_(float("nan"))
        graph.replay()
        assert torch.equal(captured, want), turn
    batch.check()


def test_two_batches_at_once_on_two_streams():
    """Each batch has its own workspace: the same bits as one after the other."""
    cache, table = make(4, 128, 64, [4000, 900, 2500], seed=2)
    work = []
    for i, (q_lens, lens) in enumerate((([1, 1, 1], [4000, 900, 2500]), ([50, 1, 200], [3000, 800, 2100]))):
        batch = kv4.Batch.of(table, q_lens, lens)
        q = queries(sum(q_lens), 16, 128, seed=i)
        work.append((batch, q, kv4.attention(cache, batch, q)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(20):
        for i, (batch, q, _) in enumerate(work):
            with torch.cuda.stream(streams[i]):
                outs[i].append(kv4.attention(cache, batch, q))
    torch.cuda.synchronize()
    for i, (batch, _, want) in enumerate(work):
        batch.check()
        assert all(torch.equal(o, want) for o in outs[i])
