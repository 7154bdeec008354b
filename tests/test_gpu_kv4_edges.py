"""The paged 4-bit cache (drinkme_b200.kv4) where sizes and values end: byte
offsets past 32 bits, queries and keys that are not finite, more sequences
than a block has threads, prompts alone, and lengths that change under a graph."""
from __future__ import annotations

import pytest
import torch

from drinkme_b200 import kv4
from test_gpu_kv4 import DEV, check_attention, make, queries

pytestmark = pytest.mark.gpu


def test_byte_offsets_past_32_bits():
    """Pages on both sides of the 4 GB boundary of the codes give the bits that the
    same rows give in a small cache."""
    nh, nkv, hd, page, n = 16, 8, 128, 256, 700
    pages = (1 << 32) // (nkv * 2 * page * hd // 2) + 64
    big = kv4.Cache.empty(pages, page, nkv, hd, device=DEV)
    table = torch.tensor([[pages - 1, 5, pages - 40]], dtype=torch.int32, device=DEV)
    small, near = make(nkv, hd, page, [n], seed=2)
    cos, sin = kv4.rope_tables(hd, 1024, 1e4, device=DEV)
    x = torch.randn(n, (nh + 2 * nkv) * hd, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    got = []
    for cache, t in ((big, table), (small, near)):
        batch = kv4.Batch.of(t, [n], [n])
        q = kv4.append(cache, batch, *kv4.split_qkv(x, nh, nkv, hd), cos, sin)
        one = kv4.Batch.of(t, [1], [n])
        got.append((q, *kv4.read(cache, batch), kv4.attention(cache, batch, q),
                    kv4.attention(cache, one, q[-1:].contiguous())))
        batch.check()
        one.check()
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("q_len", [1, 5, 40])
def test_queries_that_are_not_finite(q_len):
    """A NaN or an infinity in a head's query makes that head's row NaN, and no other."""
    lens = [90, 300]
    cache, table = make(2, 128, 64, lens, seed=3)
    batch = kv4.Batch.of(table, [q_len, q_len], lens)
    q = queries(2 * q_len, 8, 128)
    ref = kv4.attention(cache, batch, q)
    for at, value in ((5, float("nan")), (127, float("inf")), (0, -float("inf"))):
        bad = q.clone()
        bad[q_len, 6, at] = value
        out = kv4.attention(cache, batch, bad)
        assert bool(out[q_len, 6].isnan().all()), (at, value)
        out[q_len, 6] = ref[q_len, 6]
        assert torch.equal(out, ref)


@pytest.mark.parametrize("q_len", [1, 6, 150])
def test_a_key_of_nan_reaches_those_who_see_it_only(q_len):
    n = 200
    cache, table = make(2, 128, 64, [n, n], seed=4)
    batch = kv4.Batch.of(table, [q_len, q_len], [n, n])
    q = queries(2 * q_len, 8, 128)
    ref = kv4.attention(cache, batch, q)
    for position in (74, n - 1, n - 2):
        at = (int(table[1, position // 64]), 1, position % 64)
        kept = cache.scales[at].clone()
        cache.scales[at][:2] = float("nan")
        out = kv4.attention(cache, batch, q)
        sees = (torch.arange(n - q_len, n) >= position).to(DEV)
        assert bool(out[q_len:][sees][:, 4:].isnan().all())
        out[q_len:, 4:] = torch.where(sees[:, None, None], ref[q_len:, 4:], out[q_len:, 4:])
        assert torch.equal(out, ref)
        cache.scales[at] = kept


@pytest.mark.parametrize("hd,q_len", [(128, 1), (64, 7)])
def test_more_sequences_than_threads(hd, q_len):
    """700 sequences, some without rows; with 4 heads a kv head 7 tokens are 28 rows."""
    g = torch.Generator().manual_seed(q_len)
    lens = torch.randint(0, 40, (700,), generator=g).tolist()
    cache, table = make(2, hd, 16, lens, seed=5)
    check_attention(cache, table, [q_len] * 700, lens, 8)


@pytest.mark.parametrize("nh,nkv,hd,n,length", [(8, 2, 128, 700, 700), (4, 1, 64, 300, 5000), (8, 8, 128, 200, 1000),
                                                (2, 2, 64, 129, 129), (16, 1, 128, 17, 3000)])
def test_a_prompt_alone(nh, nkv, hd, n, length):
    cache, table = make(nkv, hd, 64, [length], seed=n)
    check_attention(cache, table, [n], [length], nh)
    check_attention(cache, table, [n], [length], nh, window=150, out_dtype=torch.float32)


def test_lengths_that_change_under_a_graph():
    """The lengths are read on the device: a graph captured for 300 tokens of one
    sequence (and of two) serves fewer, down to one."""
    nh, nkv, hd = 8, 2, 128
    cache, table = make(nkv, hd, 64, [900, 900], seed=6)
    q = queries(300, nh, hd)
    for seqs, cuts in ((1, ([300], [200], [7], [1])), (2, ([290, 10], [1, 299], [30, 30], [0, 4]))):
        first = kv4.Batch.of(table[:seqs], cuts[0], [900] * seqs)
        batch = kv4.Batch(table[:seqs], first.q_start, first.kv_len, tokens=300, max_q=300)
        out = kv4.attention(cache, batch, q)
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            kv4.attention(cache, batch, q, out=out)
        for cut in cuts:
            lens = [600 + c for c in cut]
            T = sum(cut)
            batch.q_start.copy_(torch.tensor([0, *torch.tensor(cut).cumsum(0).tolist()], dtype=torch.int32))
            batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
            graph.replay()
            batch.check()
            want = kv4.attention(cache, kv4.Batch.of(table[:seqs], cut, lens), q[:T])
            err = (out[:T].float() - want.float()).abs().max()
            # few rows may be taken by the other kernel: two roundings of 2^-8 of values up to 16
            assert float(err) <= 2 * 16 * 2.0 ** -8, (cut, float(err))
