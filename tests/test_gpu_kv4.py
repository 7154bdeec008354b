"""The paged 4-bit cache (drinkme_b200.kv4) on the GPU: appended codes and
scales equal the definition bit for bit, read rows and attention against
float64, at the lengths, layouts and masks where they can go wrong."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import kv4_oracle as oracle
from drinkme_b200 import _lib, kv4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(nkv, hd, page, kv_lens, seed=0, fill=True, cols=0, junk=True):
    """A cache whose rows past the lengths, spare pages and unused table entries
    hold what must not be read as values."""
    g = torch.Generator().manual_seed(seed)
    need = [max(0, -(-n // page)) for n in kv_lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(kv_lens), max(max(need), 1, cols)), 1 << 30, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    codes = torch.randint(0, 256, (pages, nkv, 2, page, hd // 2), generator=g, dtype=torch.uint8)
    s = 0.1 + 0.4 * torch.rand(pages, nkv, page, 2, generator=g)
    m = -7.5 * s + 0.3 * torch.randn(pages, nkv, page, 2, generator=g)
    scales = torch.stack((s[..., 0], m[..., 0], s[..., 1], m[..., 1]), -1).to(torch.bfloat16)
    if junk:
        keep = torch.zeros(pages, page, dtype=torch.bool)
        for b, n in enumerate(kv_lens):
            for j in range(need[b]):
                keep[table[b, j].long(), : min(page, n - j * page)] = True
        scales[~keep[:, None, :].expand(pages, nkv, page)] = float("nan")
    if not fill:
        scales[:] = float("nan")
    return kv4.Cache(codes.to(DEV), scales.to(DEV)), table.to(DEV)


def queries(T, nh, hd, seed=1, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(T, nh, hd, generator=g)).to(torch.bfloat16).to(DEV)


def check_attention(cache, table, q_lens, kv_lens, nh, window=0, scale=None, out_dtype=torch.bfloat16, seed=1,
                    qscale=1.5):
    hd = cache.head_dim
    batch = kv4.Batch.of(table, q_lens, kv_lens)
    q = queries(sum(q_lens), nh, hd, seed, qscale)
    out = kv4.attention(cache, batch, q, window=window, scale=scale, out_dtype=out_dtype)
    batch.check()
    ref, slack = oracle.attention(cache.codes, cache.scales, table, q_lens, kv_lens, q,
                                  1 / math.sqrt(hd) if scale is None else scale, window)
    # weights (or the values themselves, for prompts) are rounded to bf16 (2^-8
    # relative), fp32 sums, then the output's own rounding
    bound = slack * 2.0 ** -8 + ref.abs() * (2.0 ** -8 if out_dtype == torch.bfloat16 else 0) + 1e-6
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    again = kv4.attention(cache, batch, q, window=window, scale=scale, out_dtype=out_dtype)
    assert torch.equal(out, again)
    return out


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv", [(8, 2), (32, 8), (4, 4), (10, 1), (40, 1)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_decode_lengths(hd, nh, nkv, page):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700, 1025]
    cache, table = make(nkv, hd, page, lens, seed=hd + nh)
    check_attention(cache, table, [1] * len(lens), lens, nh)


@pytest.mark.parametrize("hd,nh,nkv,length", [(128, 32, 8, 5000), (128, 8, 1, 20001), (64, 16, 16, 3000),
                                              (128, 64, 8, 4096)])
def test_one_long_sequence(hd, nh, nkv, length):
    cache, table = make(nkv, hd, 64, [length], seed=3)
    check_attention(cache, table, [1], [length], nh)
    check_attention(cache, table, [1], [length], nh, out_dtype=torch.float32)


@pytest.mark.parametrize("q_len", [2, 3, 5, 8])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (32, 8, 64), (64, 8, 128), (6, 6, 128)])
def test_verify_batches(q_len, nh, nkv, hd):
    lens = [q_len, q_len + 1, 16, 17, 100, 128 + q_len, 600]
    cache, table = make(nkv, hd, 32, lens, seed=q_len)
    check_attention(cache, table, [q_len] * len(lens), lens, nh)


@pytest.mark.parametrize("nh,nkv,hd,page", [(8, 2, 128, 64), (4, 4, 64, 16), (12, 1, 128, 128), (32, 8, 128, 64),
                                            (14, 2, 64, 256)])
def test_prompts(nh, nkv, hd, page):
    q_lens, lens = [33, 130, 1, 257, 64, 9], [33, 200, 77, 257, 1000, 300]
    cache, table = make(nkv, hd, page, lens, seed=nh)
    check_attention(cache, table, q_lens, lens, nh)


@pytest.mark.parametrize("q_lens,lens", [([1, 1, 1], [50, 300, 1]), ([5, 5], [5, 400]), ([70, 200], [70, 500])])
@pytest.mark.parametrize("window", [1, 16, 17, 100, 5000])
def test_windows(q_lens, lens, window):
    cache, table = make(2, 128, 16, lens, seed=window)
    check_attention(cache, table, q_lens, lens, 8, window=window)


def test_empty_and_short_sequences():
    """Sequences without new tokens, without rows, and with more new tokens
    than rows: the tokens before position 0 see nothing and get zeros."""
    q_lens, lens = [1, 0, 3, 2, 0, 40, 1], [0, 0, 2, 0, 90, 7, 1]
    cache, table = make(2, 128, 16, lens, seed=9)
    out = check_attention(cache, table, q_lens, lens, 8)
    assert bool((out[0] == 0).all()) and bool((out[1] == 0).all()) and bool((out[4:6] == 0).all())
    assert bool((out[6:39] == 0).all()) and bool((out[39:46] != 0).any())


def test_all_tokens_without_rows():
    cache, table = make(2, 64, 16, [0, 0], seed=9)
    out = check_attention(cache, table, [1, 1], [0, 0], 4)
    assert bool((out == 0).all())


def test_large_scores_and_flat_scores():
    """Scores far outside exp's range at both ends, and no spread at all."""
    cache, table = make(2, 128, 64, [700, 3], seed=4)
    check_attention(cache, table, [1, 1], [700, 3], 8, scale=8.0, qscale=6.0)
    check_attention(cache, table, [1, 1], [700, 3], 8, scale=0.0)
    check_attention(cache, table, [60, 3], [700, 3], 8, scale=8.0, qscale=6.0)


def test_a_row_of_nan_reaches_those_who_see_it_only():
    cache, table = make(2, 128, 64, [200, 200], seed=4)
    page = int(table[0, 1])
    cache.scales[page, 1, 10, 2:] = float("nan")  # a value row of kv head 1, position 74
    batch = kv4.Batch.of(table, [1, 150], [200, 200])
    q = queries(151, 8, 128)
    out = kv4.attention(cache, batch, q)
    assert bool(out[0, 4:].isnan().all()) and not bool(out[0, :4].isnan().any()) and not bool(out[1:].isnan().any())
    batch = kv4.Batch.of(table, [150, 1], [200, 200])
    out = kv4.attention(cache, batch, q)
    seen = torch.arange(50, 200) >= 74
    assert bool(out[:150, 4:].isnan().all(-1).all(-1).cpu().eq(seen).all()) and not bool(out[:, :4].isnan().any())


def test_strided_queries_side_stream_and_graph():
    lens = [90, 300]
    cache, table = make(2, 128, 64, [400, 400], seed=6)
    wide = queries(2, 16, 128)
    q = wide[:, 3:11]
    batch = kv4.Batch.of(table, [1, 1], lens)
    ref = kv4.attention(cache, batch, q.contiguous())
    assert torch.equal(kv4.attention(cache, batch, q), ref)
    odd = torch.empty(2 * 8 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, 8, 128)  # off 16 bytes
    odd.copy_(q)
    assert torch.equal(kv4.attention(cache, batch, odd), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kv4.attention(cache, batch, q)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)
    # one graph serves every length
    out = torch.empty_like(ref)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kv4.attention(cache, batch, q, out=out)
    for new in (lens, [1, 400], [333, 17], [0, 64]):
        batch.kv_len.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, kv4.attention(cache, kv4.Batch.of(table, [1, 1], new), q)), new


def test_a_position_outside_the_table_is_skipped_and_reported():
    cache, table = make(2, 128, 16, [40, 40], seed=6)
    short = table[:, :2].contiguous()  # covers 32 positions
    batch = kv4.Batch.of(short, [1, 1], [40, 20])
    q = queries(2, 8, 128)
    out = kv4.attention(cache, batch, q)
    with pytest.raises(_lib.DrinkmeError, match="not covered"):
        batch.check()
    batch.check()  # cleared
    ref, slack = oracle.attention(cache.codes, cache.scales, table[1:], [1], [20], q[1:], 1 / math.sqrt(128))
    assert bool(((out[1:].double().cpu() - ref).abs() <= slack * 2.0 ** -8 + ref.abs() * 2.0 ** -8 + 1e-6).all())
    k = torch.randn(2, 2, 128, device=DEV)
    before = cache.codes.clone()
    kv4.append(cache, batch, None, k, k)
    with pytest.raises(_lib.DrinkmeError):
        batch.check()
    changed = (cache.codes != before).flatten(2).any(-1).any(-1).nonzero().flatten().tolist()
    assert changed == [int(table[1, 1])]


# ------------------------------------------------------------------ append --

def tables(rot, positions):
    return kv4.rope_tables(rot, positions, 1e4, device=DEV) if rot else (None, None)


@pytest.mark.parametrize("hd,rot", [(128, 128), (128, 64), (128, 48), (64, 64), (64, 16), (64, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_is_the_definition_bit_for_bit(hd, rot, interleaved, norm, dtype):
    nh, nkv, page = 6, 3, 16
    q_lens, kv_lens = [1, 5, 0, 40, 1], [1, 21, 9, 57, 160]
    T = sum(q_lens)
    cache, table = make(nkv, hd, page, kv_lens, seed=rot, fill=False)
    before = cache.codes.clone(), cache.scales.clone()
    g = torch.Generator().manual_seed(hd)
    qkv = torch.randn(T, (nh + 2 * nkv) * hd, generator=g)
    qkv[3] *= 1e-3
    qkv[7] *= 300.0
    qkv[9, 40:] += 50.0
    qkv = qkv.to(dtype)
    qn = (1 + 0.2 * torch.randn(hd, generator=g)).to(torch.bfloat16) if norm else None
    kn = (1 + 0.2 * torch.randn(hd, generator=g)).to(torch.bfloat16) if norm else None
    cos, sin = tables(rot, 200)
    batch = kv4.Batch.of(table, q_lens, kv_lens)
    q, k, v = kv4.split_qkv(qkv.to(DEV), nh, nkv, hd)
    on = (lambda w: None if w is None else w.to(DEV))
    got = kv4.append(cache, batch, q, k, v, cos, sin, q_norm=on(qn), k_norm=on(kn), interleaved=interleaved)
    batch.check()
    pos = np.concatenate([np.arange(n - a, n) for a, n in zip(q_lens, kv_lens)]).astype(int)
    seq = np.repeat(np.arange(len(q_lens)), q_lens)
    x = qkv.float().numpy().reshape(T, -1, hd)
    c, s = (cos.cpu().numpy()[pos], sin.cpu().numpy()[pos]) if rot else (None, None)
    w = (lambda t: None if t is None else t.float().numpy())
    want_q = oracle.rotate(x[:, :nh], w(qn), c, s, 1e-6, interleaved)
    assert np.array_equal(got.float().cpu().numpy(), oracle.bf16(want_q))
    rows = np.stack((oracle.rotate(x[:, nh:nh + nkv], w(kn), c, s, 1e-6, interleaved), x[:, nh + nkv:]), 2)
    sc, m, code = oracle.quantise(rows)
    codes, scales = before[0].cpu(), before[1].cpu()
    at = table.cpu()[torch.from_numpy(seq), torch.from_numpy(pos // page)].long()
    slot = torch.from_numpy(pos % page)
    codes[at, :, :, slot] = torch.from_numpy(oracle.pack(code))
    four = np.stack((sc[:, :, 0], m[:, :, 0], sc[:, :, 1], m[:, :, 1]), -1)
    scales[at, :, slot] = torch.from_numpy(four.astype(np.float32)).to(torch.bfloat16)
    assert torch.equal(cache.codes.cpu(), codes)  # every other byte as it was
    assert torch.equal(cache.scales.cpu().view(torch.int16), scales.view(torch.int16)) or \
        torch.equal(cache.scales.cpu().nan_to_num(7e30), scales.nan_to_num(7e30))
    # read: the values that the codes stand for, in one rounding each
    val = m[..., None] + sc[..., None] * code.astype(np.float32)
    kf, vf = kv4.read(cache, batch, dtype=torch.float32)
    assert np.array_equal(kf.cpu().numpy(), val[:, :, 0]) and np.array_equal(vf.cpu().numpy(), val[:, :, 1])
    kb, vb = kv4.read(cache, batch)
    assert np.array_equal(kb.float().cpu().numpy(), oracle.bf16(val[:, :, 0]))
    # and the held values are within half a step of the rotated ones in float64 (s and m
    # are rounded to 8 bits: 15 steps of 2^-9, and 2^-9 of m)
    y = rows.astype(np.float64)
    step = sc[..., None].astype(np.float64)
    assert np.all(np.abs(val - y) <= step * (0.5 + 15 * 2.0 ** -8) + np.abs(m[..., None]) * 2.0 ** -8 + 1e-30)


def test_append_rotation_against_float64():
    nh, nkv, hd, n = 2, 1, 128, 300
    cache, table = make(nkv, hd, 64, [n], fill=False)
    batch = kv4.Batch.of(table, [n], [n])
    g = torch.Generator().manual_seed(1)
    x = torch.randn(n, (nh + 2 * nkv) * hd, generator=g)
    cos, sin = kv4.rope_tables(hd, n, 1e6, device=DEV)
    q, k, v = kv4.split_qkv(x.to(DEV), nh, nkv, hd)
    got = kv4.append(cache, batch, q, k, v, cos, sin).double().cpu()
    f = 1e6 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    z = torch.polar(torch.ones(n, hd // 2, dtype=torch.float64), torch.arange(n)[:, None] * f)
    y = x.double().view(n, -1, hd)[:, :nh]
    y = torch.complex(y[..., : hd // 2], y[..., hd // 2:]) * z[:, None]
    want = torch.cat((y.real, y.imag), -1)
    # bf16 rounding, and fp32 tables and products
    assert bool(((got - want).abs() <= want.abs() * 2.0 ** -8 + 2e-6).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_rows_at_the_ends_of_the_type(dtype):
    """Equal values, tiny and huge rows, infinities, NaN: as the definition says."""
    hd, nkv = 64, 1
    big = torch.finfo(dtype).max
    rows = torch.zeros(10, hd)
    rows[0] = 0.0
    rows[1] = -3.25
    rows[2, 5] = 1e-41 if dtype == torch.float32 else 1e-40
    rows[3, 7] = float("inf")
    rows[4, 0] = float("-inf")
    rows[5, 63] = float("nan")
    rows[6] = torch.linspace(-1, 1, hd) * big
    rows[7] = torch.linspace(0.25, 0.75, hd) * big
    rows[8] = torch.linspace(-1, 1, hd) * 3e-38
    rows[9] = 1e4 + torch.linspace(0, 1, hd)
    rows = rows.to(dtype)
    cache, table = make(nkv, hd, 16, [10], fill=False)
    batch = kv4.Batch.of(table, [10], [10])
    x = rows[:, None].to(DEV)
    kv4.append(cache, batch, None, x, x)
    sc, m, code = oracle.quantise(rows[:, None].float().numpy())
    page = int(table[0, 0])
    assert np.array_equal(cache.codes[page, 0, 0, :10].cpu().numpy(), oracle.pack(code)[:, 0])
    got = cache.scales[page, 0, :10].float().cpu().numpy()
    assert np.array_equal(got[:, 0], sc[:, 0], equal_nan=True) and np.array_equal(got[:, 1], m[:, 0], equal_nan=True)
    assert np.array_equal(got[:, 2:], got[:, :2], equal_nan=True)
    k, _ = kv4.read(cache, batch, dtype=torch.float32)
    assert k[3:7].isnan().all() and not k[[0, 1, 2, 8, 9]].isnan().any()
    assert torch.equal(k[0].cpu(), torch.zeros(1, hd)) and torch.equal(k[1].cpu(), torch.full((1, hd), -3.25))


def test_append_strides_and_alignment():
    """Separate, padded and misaligned inputs give the bits of the packed ones."""
    nh, nkv, hd, T = 4, 2, 128, 7
    g = torch.Generator().manual_seed(2)
    x = torch.randn(T, (nh + 2 * nkv) * hd, generator=g).to(torch.bfloat16).to(DEV)
    cos, sin = tables(hd, 100)
    results = []
    for how in range(4):
        cache, table = make(nkv, hd, 16, [T + 3], seed=1, fill=False)
        batch = kv4.Batch.of(table, [T], [T + 3])
        if how == 0:
            parts = kv4.split_qkv(x, nh, nkv, hd)
        elif how == 1:
            wide = torch.zeros(T, x.shape[1] + 24, dtype=x.dtype, device=DEV)
            wide[:, 3:3 + x.shape[1]] = x
            parts = kv4.split_qkv(wide[:, 3:3 + x.shape[1]].contiguous(), nh, nkv, hd)
            y = wide[:, 3:3 + x.shape[1]].unflatten(1, (-1, hd))
            parts = (y[:, :nh], y[:, nh:nh + nkv], y[:, nh + nkv:])
        elif how == 2:
            parts = tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in kv4.split_qkv(x, nh, nkv, hd))
        else:
            parts = tuple(t.contiguous() for t in kv4.split_qkv(x, nh, nkv, hd))
        q = kv4.append(cache, batch, *parts, cos, sin)
        results.append((q, cache.codes.clone(), cache.scales.nan_to_num(1e30)))
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))


def test_tokens_before_position_zero_are_not_appended():
    cache, table = make(1, 64, 16, [3], seed=1, fill=False)
    before = cache.codes.clone()
    batch = kv4.Batch.of(table, [5], [3])
    x = torch.randn(5, 1, 64, device=DEV)
    q = kv4.append(cache, batch, x, x, x, *tables(64, 16))
    batch.check()
    assert bool((q[:2] == 0).all()) and bool((q[2:] != 0).any())
    k, v = kv4.read(cache, batch)
    assert bool((k[:2] == 0).all()) and bool((v[2:] != 0).any())
    assert torch.equal(cache.codes[:, :, :, 3:], before[:, :, :, 3:])


def test_append_then_attention_is_attention_of_the_rotated_rows():
    """The step as it is used: what append writes, attention reads."""
    nh, nkv, hd = 8, 2, 128
    q_lens, kv_lens = [60, 1, 4], [60, 33, 300]
    cache, table = make(nkv, hd, 32, kv_lens, seed=8, junk=False)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(sum(q_lens), (nh + 2 * nkv) * hd, generator=g).to(torch.bfloat16).to(DEV)
    batch = kv4.Batch.of(table, q_lens, kv_lens)
    q = kv4.append(cache, batch, *kv4.split_qkv(x, nh, nkv, hd), *tables(hd, 400))
    out = kv4.attention(cache, batch, q)
    ref, slack = oracle.attention(cache.codes, cache.scales, table, q_lens, kv_lens, q, 1 / math.sqrt(hd))
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= slack * 2.0 ** -8 + ref.abs() * 2.0 ** -8 + 1e-6).all())
