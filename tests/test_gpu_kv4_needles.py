"""Attention that must not lose a position: needles.

Every key is a row of zeros but for the needles', which are alike and whose score is
85 above the others'; needle i's value row is 15 in element i and 0 elsewhere. A query
row that sees N needles gives 15 / N in their elements and 0 in the others: a
position that is lost, or taken twice, changes its element by all of that. There
is a needle in every run of 16 positions, and at the sides of pages, blocks and pieces.

The bound is that of the other tests, 2^-8 of sum p (|v| + 8 s) = 15 / N + 8, and the
output's rounding: at most 0.033 of a signal of 15 / 100 = 0.15."""
from __future__ import annotations

import math

import pytest
import torch

import kv4_oracle as oracle
from drinkme_b200 import kv4
from test_gpu_kv4 import DEV, make, queries

pytestmark = pytest.mark.gpu
MOST = 100


def haystack(nkv, hd, page, length):
    """A cache of one sequence whose rows are all zeros, and its table."""
    cache, table = make(nkv, hd, page, [length], seed=length, junk=False)
    cache.codes.zero_()
    cache.scales.copy_(torch.tensor([1.0, 0.0, 1.0, 0.0], dtype=torch.bfloat16, device=DEV).expand_as(cache.scales))
    return cache, table


def put(cache, table, h, positions, on: bool):
    page = cache.page_size
    for i, p in enumerate(positions):
        at = (int(table[0, p // page]), h)
        cache.codes[at][0, p % page] = 0xFF if on else 0
        cache.codes[at][1, p % page, i // 2] = (0x0F if i % 2 == 0 else 0xF0) if on else 0


def rounds(nkv, hd, length, seed):
    """Lists of needles by kv head, until every run of 16 positions and both
    sides of every multiple of 256 have had one."""
    g = torch.Generator().manual_seed(seed)
    want = [min(length - 1, 16 * u + int(torch.randint(16, (1,), generator=g))) for u in range(-(-length // 16))]
    want += [p for k in range(0, length, 256) for p in (k - 1, k) if 0 <= p < length] + [length - 1]
    want = sorted(set(want))
    most = min(MOST, hd - 1)
    lists = [want[i::max(1, -(-len(want) // most))] for i in range(max(1, -(-len(want) // most)))]
    return [lists[i:i + nkv] for i in range(0, len(lists), nkv)]


@pytest.mark.parametrize("nh,nkv,hd,page,q_len,length,window", [
    (8, 2, 128, 64, 1, 1000, 0), (32, 8, 128, 64, 1, 5000, 0), (64, 8, 128, 16, 1, 20001, 0), (8, 4, 64, 32, 1, 9000, 0),
    (32, 8, 128, 64, 5, 4000, 0), (12, 4, 128, 256, 8, 2049, 0), (24, 8, 64, 16, 8, 3001, 0),
    (32, 8, 128, 64, 40, 4500, 0), (8, 4, 64, 16, 300, 6001, 0), (16, 8, 128, 128, 700, 3000, 0),
    (32, 8, 128, 64, 1, 5000, 1777), (12, 4, 128, 16, 8, 3000, 1001), (16, 8, 128, 64, 300, 3000, 901)])
def test_no_position_is_lost(nh, nkv, hd, page, q_len, length, window):
    cache, table = haystack(nkv, hd, page, length)
    batch = kv4.Batch.of(table, [q_len], [length])
    grp = nh // nkv
    # 85 = q . K / sqrt(hd): q's elements alike, K's 15
    q = torch.full((q_len, nh, hd), 85.0 / (15 * math.sqrt(hd)), device=DEV).to(torch.bfloat16)
    p = torch.arange(length - q_len, length)[:, None]
    for needles in rounds(nkv, hd, length, seed=nh + q_len):
        for h, at in enumerate(needles):
            put(cache, table, h, at, True)
        out = kv4.attention(cache, batch, q, window=window, out_dtype=torch.float32).double().cpu()
        batch.check()
        for h, at in enumerate(needles):
            j = torch.tensor(at)[None, :]
            seen = (j <= p) & (j > p - window if window else j >= 0)
            n = seen.sum(-1, keepdim=True)
            want = torch.zeros(q_len, hd, dtype=torch.float64)
            want[:, : len(at)] = torch.where(seen, 15.0 / n.clamp(min=1), 0.0)
            bound = (15.0 / n.clamp(min=1) + 8) * 2.0 ** -8 + 1e-6
            err = (out[:, h * grp:(h + 1) * grp] - want[:, None]).abs()
            rows = (n[:, 0] > 0)
            assert bool((err <= bound[:, None])[rows].all()), (h, float(err[rows].max()))
        for h, at in enumerate(needles):
            put(cache, table, h, at, False)


@pytest.mark.parametrize("nh,nkv,hd,q_lens,lens", [
    (32, 8, 128, [1], [5000]), (8, 1, 128, [1], [20001]), (32, 8, 128, [1] * 6, [900, 3000, 64, 2000, 1, 700]),
    (32, 8, 128, [5, 5], [4000, 300]), (8, 2, 64, [300], [5000]), (8, 2, 128, [200, 1, 33], [900, 700, 2000])])
def test_relative_error(nh, nkv, hd, q_lens, lens):
    """Weights rounded to bf16 (relative rms about 0.0016, of terms with random signs) and
    the output's own rounding (as much) make about 0.0023 of the output's norm;
    bound 0.004, and 0.0025 where the output is fp32."""
    cache, table = make(nkv, hd, 64, lens, seed=nh)
    q = queries(sum(q_lens), nh, hd)
    ref, _ = oracle.attention(cache.codes, cache.scales, table, q_lens, lens, q, 1 / math.sqrt(hd))
    for dtype, bound in ((torch.bfloat16, 0.004), (torch.float32, 0.0025)):
        batch = kv4.Batch.of(table, q_lens, lens)
        out = kv4.attention(cache, batch, q, out_dtype=dtype).double().cpu()
        batch.check()
        assert float((out - ref).norm() / ref.norm()) < bound


def test_a_graph_whose_lengths_change_is_right_each_time():
    """Captured for 300 tokens, replayed for others: against float64, element by element."""
    nh, nkv, hd = 8, 2, 128
    cache, table = make(nkv, hd, 64, [900, 900], seed=6, junk=False)
    q = queries(300, nh, hd)
    for seqs, cuts in ((1, ([300], [200], [7], [1])), (2, ([290, 10], [1, 299], [30, 30], [0, 4], [2, 1]))):
        batch = kv4.Batch(table[:seqs], *(torch.tensor(x, dtype=torch.int32, device=DEV) for x in
                                          ([0, *torch.tensor(cuts[0]).cumsum(0).tolist()], [900] * seqs)), tokens=300, max_q=300)
        out = kv4.attention(cache, batch, q)
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            kv4.attention(cache, batch, q, out=out)
        for cut in cuts:
            lens = [600 - 37 * i + c for i, c in enumerate(cut)]
            T = sum(cut)
            batch.q_start.copy_(torch.tensor([0, *torch.tensor(cut).cumsum(0).tolist()], dtype=torch.int32))
            batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
            graph.replay()
            batch.check()
            ref, slack = oracle.attention(cache.codes, cache.scales, table[:seqs], cut, lens, q[:T], 1 / math.sqrt(hd))
            err = (out[:T].double().cpu() - ref).abs()
            assert bool((err <= slack * 2.0 ** -8 + ref.abs() * 2.0 ** -8 + 1e-6).all()), cut
            assert float((out[:T].double().cpu() - ref).norm() / ref.norm()) < 0.004, cut
