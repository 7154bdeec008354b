"""What the paged 4-bit cache and the logits operators refuse, before a device is
touched: the C ABI's argument checks and the Python layer's; and the rotary
tables (CPU)."""
from __future__ import annotations

import ctypes as ct
import math

import pytest
import torch

from drinkme_b200 import _lib, kv4, logits

FAKE = 0x10000  # never dereferenced: the checks refuse first


def cache(**kw):
    f = dict(codes=FAKE, scales=FAKE, pages=4, page_size=16, kv_heads=2, head_dim=128)
    f.update(kw)
    return _lib.KV4Cache(**f)


def batch(**kw):
    f = dict(page_table=FAKE, q_start=FAKE, kv_len=FAKE, table_stride=3, table_cols=3, seqs=2, tokens=2, max_q=1,
             error=FAKE, work=FAKE, work_bytes=1 << 30)
    f.update(kw)
    return _lib.KV4Batch(**f)


def append_args(**kw):
    f = dict(q=FAKE, k=FAKE, v=FAKE, q_stride=1024, k_stride=1024, v_stride=1024, in_dtype=_lib.DM_BF16, heads=8,
             eps=1e-6, rot=128, cos_table=FAKE, sin_table=FAKE, positions=100, q_out=FAKE)
    f.update(kw)
    return _lib.KV4AppendArgs(**f)


@pytest.mark.parametrize("bad", [dict(codes=None), dict(pages=0), dict(page_size=48), dict(page_size=512),
                                 dict(head_dim=96), dict(codes=FAKE + 8), dict(kv_heads=0)])
def test_bad_caches(bad):
    for fn, args in (("dm_kv4_append", (append_args(),)), ("dm_kv4_read", (FAKE, FAKE, 0)),
                     ("dm_kv4_attention", (FAKE, 1024, 8, 0.1, 0, FAKE, 0))):
        with pytest.raises(ValueError):
            _lib.call(fn, cache(**bad), batch(), *args, None)


@pytest.mark.parametrize("bad", [dict(page_table=None), dict(seqs=0), dict(table_cols=0), dict(table_stride=2),
                                 dict(error=None), dict(error=FAKE + 2), dict(max_q=0),
                                 dict(tokens=-1)])
def test_bad_batches(bad):
    for fn, args in (("dm_kv4_append", (append_args(),)), ("dm_kv4_read", (FAKE, FAKE, 0)),
                     ("dm_kv4_attention", (FAKE, 1024, 8, 0.1, 0, FAKE, 0))):
        with pytest.raises(ValueError):
            _lib.call(fn, cache(), batch(**bad), *args, None)


@pytest.mark.parametrize("bad", [dict(k=None), dict(heads=0), dict(q_out=None), dict(q_out=FAKE + 2), dict(rot=8),
                                 dict(rot=144), dict(cos_table=None), dict(sin_table=FAKE + 4), dict(positions=0),
                                 dict(in_dtype=7), dict(k_stride=-1)])
def test_bad_append_arguments(bad):
    with pytest.raises(ValueError):
        _lib.call("dm_kv4_append", cache(), batch(), append_args(**bad), None)


@pytest.mark.parametrize("args", [(None, 1024, 8, 0.1, 0, FAKE, 0), (FAKE, 1024, 7, 0.1, 0, FAKE, 0),
                                  (FAKE, 1023, 8, 0.1, 0, FAKE, 0), (FAKE + 2, 1024, 8, 0.1, 0, FAKE, 0),
                                  (FAKE, 1024, 8, 0.1, -1, FAKE, 0), (FAKE, 1024, 8, 0.1, 0, FAKE + 8, 0),
                                  (FAKE, 1024, 8, 0.1, 0, FAKE, 5), (FAKE, 1024, 0, 0.1, 0, FAKE, 0)])
def test_bad_attention_arguments(args):
    with pytest.raises(ValueError):
        _lib.call("dm_kv4_attention", cache(), batch(), *args, None)


def test_short_workspace_and_workspace_sizes():
    L = _lib.lib()
    n = L.dm_kv4_workspace_bytes(cache(), 2, 1, 8)
    assert n > 0 and L.dm_kv4_workspace_bytes(cache(), 2, 1, 7) < 0 and L.dm_kv4_workspace_bytes(cache(), 0, 1, 8) < 0
    for bad in (dict(work_bytes=n - 1), dict(work=None), dict(work=FAKE + 4)):
        with pytest.raises(ValueError):
            _lib.call("dm_kv4_attention", cache(), batch(**bad), FAKE, 1024, 8, 0.1, 0, FAKE, 0, None)
    assert L.dm_kv4_workspace_bytes(cache(), 2, 100, 8) > n  # prompts: the parts of whole row tiles


def test_read_needs_an_output():
    for args in ((None, None, 0), (FAKE + 8, None, 0), (FAKE, None, 9)):
        with pytest.raises(ValueError):
            _lib.call("dm_kv4_read", cache(), batch(), *args, None)


@pytest.mark.parametrize("bad", [dict(logits=None), dict(out=None), dict(dtype=4), dict(rows=-1), dict(rows=70000),
                                 dict(vocab=0), dict(stride=50), dict(out_stride=50), dict(logits=FAKE + 1),
                                 dict(bias_ids=FAKE), dict(bias_values=FAKE), dict(history_stride=-1),
                                 dict(allowed=FAKE, allowed_stride=3)])
def test_bad_logits_arguments(bad):
    f = dict(logits=FAKE, out=FAKE, stride=100, out_stride=100, dtype=_lib.DM_F32, rows=2, vocab=100)
    f.update(bad)
    with pytest.raises(ValueError):
        _lib.call("dm_logits_process", _lib.LogitsArgs(**f), None)


def test_null_structs():
    for fn, args in (("dm_kv4_append", (None, None, None)), ("dm_kv4_read", (None, None, FAKE, FAKE, 0)),
                     ("dm_kv4_attention", (None, None, FAKE, 8, 8, 0.1, 0, FAKE, 0)), ("dm_logits_process", (None,))):
        with pytest.raises(ValueError):
            _lib.call(fn, *args, None)
    with pytest.raises(ValueError):
        _lib.call("dm_kv4_check", None, ct.byref(ct.c_int32()), None)


def test_python_refuses_host_tensors_and_bad_shapes():
    with pytest.raises(ValueError, match="CUDA"):
        kv4.Cache(torch.zeros(1, 1, 2, 16, 64, dtype=torch.uint8), torch.zeros(1, 1, 16, 4, dtype=torch.bfloat16))
    t = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kv4.Batch(t, torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), tokens=2, max_q=1)
    with pytest.raises(ValueError, match="columns"):
        kv4.split_qkv(torch.zeros(2, 100), 2, 1, 64)
    with pytest.raises(ValueError, match="CUDA"):
        logits.process(torch.zeros(2, 10))


# ---------------------------------------------------------- rotary tables --

def test_rope_tables_plain_and_linear():
    cos, sin = kv4.rope_tables(64, 50, 1e4, device="cpu")
    f = [1e4 ** (-2 * i / 64) for i in range(32)]
    for p in (0, 1, 7, 49):
        for i in (0, 5, 31):
            assert abs(float(cos[p, i]) - math.cos(p * f[i])) < 1e-7 and abs(float(sin[p, i]) - math.sin(p * f[i])) < 1e-7
    half, _ = kv4.rope_tables(64, 99, 1e4, scaling={"type": "linear", "factor": 2.0}, device="cpu")
    assert torch.allclose(half[2 * torch.arange(49)], cos[:49], atol=1e-6)


@pytest.mark.parametrize("scaling", [{"type": "yarn", "factor": 4.0, "original": 4096},
                                     {"type": "bands", "factor": 8.0, "original": 4096, "low": 1, "high": 4}])
def test_scaled_tables_keep_fast_frequencies_and_divide_slow_ones(scaling):
    rot, theta = 128, 1e6
    cos, sin = kv4.rope_tables(rot, 3, theta, scaling=scaling, device="cpu")
    ang = torch.atan2(sin[1].double(), cos[1].double())
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    turns = scaling["original"] * f / (2 * math.pi)
    fast, slow = turns > 40, turns < 0.9
    assert int(fast.sum()) > 4 and int(slow.sum()) > 4
    assert torch.allclose(ang[fast], f[fast], rtol=1e-5)
    assert torch.allclose(ang[slow], f[slow] / scaling["factor"], rtol=1e-4, atol=1e-9)
    assert bool((ang <= f * (1 + 1e-5)).all()) and bool((ang >= f / scaling["factor"] * (1 - 1e-4) - 1e-9).all())
    gain = 0.1 * math.log(4.0) + 1.0 if scaling["type"] == "yarn" else 1.0
    assert torch.allclose((cos ** 2 + sin ** 2).sqrt(), torch.full_like(cos, gain), rtol=1e-5)


def test_rope_tables_refuse():
    with pytest.raises(ValueError):
        kv4.rope_tables(8, 10)
    with pytest.raises(ValueError):
        kv4.rope_tables(64, 10, scaling={"type": "other", "factor": 2.0})
    with pytest.raises(ValueError):
        kv4.rope_tables(64, 10, scaling={"type": "linear", "factor": 0.5})
