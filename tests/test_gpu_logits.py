"""Penalties, biases and grammar masks (drinkme_b200.logits) against a plain
float64 restatement, and the ends of the types."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from drinkme_b200 import logits

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def restated(x, history=None, prompt_len=None, total_len=None, repetition=None, presence=None, frequency=None,
             bias_ids=None, bias_values=None, allowed=None):
    """float64 numpy, token by token; `scale` [rows, vocab]: the sum of the magnitudes that went into a value."""
    y = x.double().cpu().numpy().copy()
    mag = np.abs(y)
    rows, vocab = y.shape
    for r in range(rows):
        if history is not None:
            ids = history[r].tolist()
            n = len(ids) if total_len is None else max(0, min(len(ids), int(total_len[r])))
            p = 0 if prompt_len is None else int(prompt_len[r])
            made = {}
            for i, v in enumerate(ids[:n]):
                if 0 <= v < vocab:
                    made[v] = made.get(v, 0) + (i >= p)
            for v, times in made.items():
                if repetition is not None:
                    f = float(repetition[r])
                    y[r, v] = y[r, v] / f if y[r, v] > 0 else y[r, v] * f
                    mag[r, v] = max(mag[r, v], abs(y[r, v]))
                f = float(frequency[r]) * times if frequency is not None else 0.0
                g = float(presence[r]) if presence is not None and times else 0.0
                y[r, v] -= f + g
                mag[r, v] += abs(f) + abs(g)
        if bias_ids is not None:
            last = {v: k for k, v in enumerate(bias_ids[r].tolist()) if 0 <= v < vocab}
            for v, k in last.items():
                y[r, v] += float(bias_values[r, k])
                mag[r, v] += abs(float(bias_values[r, k]))
        if allowed is not None:
            w = allowed[r].cpu().numpy().view(np.uint32)
            bits = (w[:, None] >> np.arange(32, dtype=np.uint32)) & 1
            y[r, bits.reshape(-1)[:vocab] == 0] = -np.inf
    return y, mag


def inputs(rows, vocab, n, k, dtype, seed, mask=True):
    g = torch.Generator().manual_seed(seed)
    a = dict(history=torch.randint(-2, vocab + 3, (rows, n), generator=g, dtype=torch.int32) if n else None,
             repetition=0.8 + 0.8 * torch.rand(rows, generator=g), presence=torch.rand(rows, generator=g) - 0.3,
             frequency=0.3 * torch.rand(rows, generator=g) - 0.1)
    if n:
        a["history"][:, : n // 3] = a["history"][:, n // 3: 2 * (n // 3)]  # repeats
        a["total_len"] = torch.randint(0, n + 1, (rows,), generator=g, dtype=torch.int32)
        a["prompt_len"] = (a["total_len"].float() * torch.rand(rows, generator=g)).to(torch.int32)
    else:
        a = {}
    if k:
        a["bias_ids"] = torch.randint(-1, vocab + 1, (rows, k), generator=g, dtype=torch.int32)
        a["bias_values"] = 4 * torch.randn(rows, k, generator=g)
    if mask:
        a["allowed"] = torch.randint(-(1 << 31), 1 << 31, (rows, -(-vocab // 32)), generator=g).to(torch.int32)
        a["allowed"][rows - 1] = 0
    x = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
    return x, {k: v for k, v in a.items() if v is not None}


def on(a):
    return {k: v.to(DEV) for k, v in a.items()}


def check(got, x, a):
    want, mag = restated(x, **a)
    got = got.double().cpu().numpy()
    inf = np.isinf(want)
    assert np.array_equal(np.isinf(got), inf) and np.all(got[inf] == want[inf])
    # four fp32 roundings on the way, one to the output's type
    bound = mag * 4 * 2.0 ** -24 + np.where(inf, 0, np.abs(want)) * (2.0 ** -8 if x.dtype == torch.bfloat16 else 0)
    assert np.all(np.abs(got[~inf] - want[~inf]) <= bound[~inf])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,n,k,mask", [(1, 1, 3, 1, True), (1, 1000, 50, 7, True), (3, 1001, 200, 0, False),
                                                 (2, 4096, 0, 3, True), (5, 4097, 9, 300, True), (2, 8191, 1, 0, True),
                                                 (1, 151936, 3000, 16, True), (70, 513, 33, 5, True),
                                                 (2, 33000, 5000, 64, False)])
def test_against_float64(dtype, rows, vocab, n, k, mask):
    x, a = inputs(rows, vocab, n, k, dtype, seed=rows + vocab, mask=mask)
    xd = x.to(DEV)
    got = logits.process(xd, **on(a))
    check(got, x, a)
    assert torch.equal(xd.cpu(), x)
    assert logits.process(xd, **on(a), out=xd) is xd and torch.equal(xd, got)  # in place, and the same bits again


@pytest.mark.parametrize("vocab", [1000, 1003])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_and_misaligned_rows(vocab, dtype):
    x, a = inputs(3, vocab, 40, 5, dtype, seed=1)
    ref = logits.process(x.to(DEV), **on(a))
    wide = torch.zeros(3, vocab + 11, dtype=dtype, device=DEV)
    for off in (0, 1, 8):
        view = wide[:, off:off + vocab]
        view.copy_(x)
        out = torch.full((3, vocab + 16), 5.0, dtype=dtype, device=DEV)
        logits.process(view, **on(a), out=out[:, 8:8 + vocab])
        assert torch.equal(out[:, 8:8 + vocab], ref)
        assert bool((out[:, :8] == 5).all()) and bool((out[:, 8 + vocab:] == 5).all())  # nothing beside the row


def test_infinities_nan_and_lowest_values():
    x = torch.zeros(2, 64)
    low = torch.finfo(torch.float32).min
    x[0, :6] = torch.tensor([float("inf"), float("-inf"), float("nan"), low, -low, 0.0])
    hist = torch.arange(6, dtype=torch.int32)[None].repeat(2, 1)
    a = dict(history=hist, repetition=torch.tensor([2.0, 1.0]), frequency=torch.tensor([0.5, 0.0]))
    got = logits.process(x.to(DEV), **on(a)).cpu()
    assert got[0, 0] == float("inf") and got[0, 1] == float("-inf") and got[0, 2].isnan()
    assert got[0, 3] == float("-inf") and got[0, 4] == -low / 2 and got[0, 5] == -0.5
    mask = torch.tensor([[~0b111 & 0x7fffffff, 0], [0, 0]], dtype=torch.int32)
    got = logits.process(x.to(DEV), allowed=mask.to(DEV)).cpu()
    assert bool((got[0, :3] == float("-inf")).all()) and got[0, 3] == low and got[0, 5] == 0
    assert bool((got[0, 31:] == float("-inf")).all()) and bool((got[1] == float("-inf")).all())


def test_nothing_asked_copies():
    x = torch.randn(3, 777, device=DEV)
    assert torch.equal(logits.process(x), x)


def test_counts_of_a_long_history_of_one_token():
    n = 70001
    hist = torch.full((1, n), 5, dtype=torch.int32, device=DEV)
    x = torch.zeros(1, 100, device=DEV)
    got = logits.process(x, history=hist, prompt_len=torch.tensor([1], dtype=torch.int32, device=DEV),
                         frequency=torch.tensor([0.25], device=DEV))
    assert float(got[0, 5]) == -0.25 * (n - 1) and bool((got[0, :5] == 0).all())


def test_captured_in_a_graph():
    x, a = inputs(2, 5000, 60, 4, torch.bfloat16, seed=3)
    xd, a = x.to(DEV), on(a)
    ref = logits.process(xd, **a)
    out = torch.empty_like(xd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        logits.process(xd, **a, out=out)
    graph.replay()
    assert torch.equal(out, ref)
