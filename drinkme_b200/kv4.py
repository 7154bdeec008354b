"""A paged key/value cache in 4 bits and the operators over it: append (rotary
positions, per-head RMSNorm, quantisation and the page write in one launch),
causal grouped-query attention for single tokens, verify batches and prompt
chunks, and reading rows back. The kernels are csrc/kv4*.cu behind the C ABI
(include/drinkme_b200.h, dm_kv4_*), which gives the formulas.

    cache = kv4.Cache.empty(pages, 64, kv_heads, head_dim, "cuda")   # one per layer
    batch = kv4.Batch(page_table, q_start, kv_len, tokens=T, max_q=1)  # one per step shape, all layers
    q, k, v = kv4.split_qkv(qkv, heads, kv_heads, head_dim)
    qr = kv4.append(cache, batch, q, k, v, cos, sin, q_norm=qn, k_norm=kn)
    out = kv4.attention(cache, batch, qr)

A row of 128 values takes 68 bytes instead of bf16's 256. The page table, the
lengths and the tokens' places are device tensors that the kernels read, so a
captured graph serves every step; `kv_len` counts a sequence's rows with the
step's new ones. Calls run on torch's current stream and do not synchronise; a
Batch's workspace belongs to one stream at a time. A position that the page
table or the rotary tables do not cover is skipped and reported by
`Batch.check`.

The reference has no counterpart in its kernels: it keeps transformers' caches
(src/drinkme/serving/kvcache.py).
"""
from __future__ import annotations

import ctypes as ct
import math

import torch

from . import _lib

_DT = {torch.bfloat16: _lib.DM_BF16, torch.float32: _lib.DM_F32}
_ERRORS = {1: "a position is not covered by the page table, the pages or the rotary tables",
           2: "a kernel's bounded wait gave up"}


def _call(index: int, fn: str, *args) -> None:
    """`fn` on torch's current stream of device `index` (the raw handle:
    torch.cuda.current_stream builds an object, 3 us of a decode step's call)."""
    if torch.cuda.current_device() == index:
        _lib.call(fn, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            _lib.call(fn, *args, torch._C._cuda_getCurrentRawStream(index))


def _device_tensor(t: torch.Tensor, what: str, dtype: torch.dtype, dim: int) -> None:
    if t.device.type != "cuda":
        raise ValueError(f"kv4: {what} must be on a CUDA device, not {t.device}")
    if t.dtype != dtype:
        raise TypeError(f"kv4: {what} must be {dtype}, not {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"kv4: {what} must have {dim} dimensions, not {t.dim()}")


class Cache:
    """One layer's pages: codes uint8 [pages, kv_heads, 2, page_size,
    head_dim / 2] and scales bf16 [pages, kv_heads, page_size, 4]."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        _device_tensor(codes, "codes", torch.uint8, 5)
        _device_tensor(scales, "scales", torch.bfloat16, 4)
        pages, nkv, two, ps, half = codes.shape
        if two != 2 or tuple(scales.shape) != (pages, nkv, ps, 4) or scales.device != codes.device:
            raise ValueError("kv4: codes [pages, kv_heads, 2, page_size, head_dim / 2] and scales "
                             f"[pages, kv_heads, page_size, 4], not {tuple(codes.shape)} and {tuple(scales.shape)}")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("kv4: the cache's tensors must be contiguous")
        if half not in (32, 64) or ps not in (16, 32, 64, 128, 256):
            raise ValueError(f"kv4: head_dim 64 or 128 and page_size 16 .. 256 by powers of two, not {2 * half} and {ps}")
        self.codes, self.scales, self.device, self.index = codes, scales, codes.device, codes.get_device()
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, nkv, ps, 2 * half
        self.c = _lib.KV4Cache(codes.data_ptr(), scales.data_ptr(), pages, ps, nkv, 2 * half)

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, device="cuda") -> "Cache":
        dev = torch.device(device)
        return cls(torch.zeros(pages, kv_heads, 2, page_size, head_dim // 2, dtype=torch.uint8, device=dev),
                   torch.zeros(pages, kv_heads, page_size, 4, dtype=torch.bfloat16, device=dev))


class Batch:
    """One step's sequences: page_table int32 [sequences, pages of the longest],
    q_start int32 [sequences + 1] (the new tokens of sequence b are rows
    [q_start[b], q_start[b + 1])), kv_len int32 [sequences], with the new
    tokens. `tokens` new tokens in all, at most `max_q` of one sequence. The
    tensors may change between steps; the counts may not."""

    def __init__(self, page_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor, *, tokens: int,
                 max_q: int):
        _device_tensor(page_table, "page_table", torch.int32, 2)
        _device_tensor(q_start, "q_start", torch.int32, 1)
        _device_tensor(kv_len, "kv_len", torch.int32, 1)
        B = page_table.shape[0]
        if q_start.shape[0] != B + 1 or kv_len.shape[0] != B or B < 1 or page_table.shape[1] < 1:
            raise ValueError(f"kv4: {B} rows of the page table, {q_start.shape[0]} starts, {kv_len.shape[0]} lengths")
        if page_table.device != q_start.device or page_table.device != kv_len.device:
            raise ValueError("kv4: the batch's tensors are on different devices")
        if (page_table.shape[1] > 1 and page_table.stride(1) != 1) or not q_start.is_contiguous() \
                or not kv_len.is_contiguous():
            raise ValueError("kv4: q_start, kv_len and the page table's rows must be contiguous")
        if tokens < 0 or max_q < 1 or max_q > max(tokens, 1):
            raise ValueError(f"kv4: tokens {tokens} and max_q {max_q}")
        self.page_table, self.q_start, self.kv_len, self.device = page_table, q_start, kv_len, page_table.device
        self.index = page_table.get_device()
        self.seqs, self.tokens, self.max_q = B, int(tokens), int(max_q)
        stride = max(page_table.stride(0), page_table.shape[1]) if B == 1 else page_table.stride(0)
        if stride < page_table.shape[1]:
            raise ValueError("kv4: the page table's rows overlap")
        self.error = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.c = _lib.KV4Batch(page_table.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(), stride,
                               page_table.shape[1], B, self.tokens, self.max_q, self.error.data_ptr(), None, 0)
        self._work: dict = {}      # by cache shape and heads
        self._captured: dict = {}  # the same, made within captures

    @classmethod
    def of(cls, page_table: torch.Tensor, q_lens, kv_lens) -> "Batch":
        """A batch of host lists: new tokens, and rows with them, by sequence."""
        dev = page_table.device
        starts = [0]
        for n in q_lens:
            starts.append(starts[-1] + int(n))
        return cls(page_table, torch.tensor(starts, dtype=torch.int32, device=dev),
                   torch.tensor([int(n) for n in kv_lens], dtype=torch.int32, device=dev), tokens=starts[-1],
                   max_q=max(1, max(int(n) for n in q_lens)))

    def reserve(self, cache: Cache, heads: int) -> None:
        """The attention's workspace for `heads` query heads over caches of this
        shape. Layers share it. The first attention call makes it; where that is
        within a graph's capture, the memory is the graph's and zeroed again by every
        captured call, so reserve it before."""
        key = (cache.kv_heads, cache.head_dim, heads)
        work = self._work.get(key)
        if work is None:
            n = _lib.lib().dm_kv4_workspace_bytes(cache.c, self.seqs, self.max_q, heads)
            if n < 0:
                raise ValueError(f"kv4: {heads} heads are no multiple of {cache.kv_heads} kv heads")
            with torch.cuda.device(self.index):
                capturing = torch.cuda.is_current_stream_capturing()
            if capturing:
                work = self._captured.get(key)
                if work is None:
                    work = self._captured[key] = torch.empty(n, dtype=torch.uint8, device=self.device)
                work.zero_()
            else:
                work = self._work[key] = torch.zeros(n, dtype=torch.uint8, device=self.device)
        self.c.work, self.c.work_bytes = work.data_ptr(), work.numel()

    def check(self) -> None:
        """Raises what the kernels recorded since the last check; synchronises."""
        word = ct.c_int32(0)
        _call(self.index, "dm_kv4_check", self.error.data_ptr(), ct.byref(word))
        if word.value:
            raise _lib.DrinkmeError(_lib.DM_EDEVICE, f"kv4: {_ERRORS.get(word.value, word.value)}")


def split_qkv(qkv: torch.Tensor, heads: int, kv_heads: int, head_dim: int):
    """Views of a fused projection's rows [T, (heads + 2 kv_heads) * head_dim]
    as q, k, v [T, heads, head_dim]."""
    if qkv.shape[-1] != (heads + 2 * kv_heads) * head_dim:
        raise ValueError(f"kv4: {qkv.shape[-1]} columns for {heads} + 2 x {kv_heads} heads of {head_dim}")
    return qkv.view(-1, heads + 2 * kv_heads, head_dim).split((heads, kv_heads, kv_heads), 1)


def _rows(t: torch.Tensor, what: str, cache: Cache, T: int):
    """`t` [T, heads, head_dim] with a token's heads together, its number of
    heads and the elements from token to token."""
    if t.get_device() != cache.index:
        raise ValueError(f"kv4: {what} on {t.device}, the cache on {cache.device}")
    if t.dim() != 3:
        raise ValueError(f"kv4: {what} must be [tokens, heads, head_dim], not {tuple(t.shape)}")
    n, h, d = t.shape
    if n != T or d != cache.head_dim:
        raise ValueError(f"kv4: {what} is {tuple(t.shape)}, the batch has {T} tokens, the cache head_dim {cache.head_dim}")
    step, s1, s2 = t.stride()
    if s2 != 1 or (s1 != d and h != 1):
        t, step = t.contiguous(), h * d
    return t, h, step


def _output(t, shape, dtype, cache: Cache, what: str) -> torch.Tensor:
    if t is None:
        return torch.empty(shape, dtype=dtype, device=cache.device)
    if t.dtype is not dtype or t.shape != shape or t.get_device() != cache.index or not t.is_contiguous():
        raise ValueError(f"kv4: {what} must be a contiguous {dtype} tensor {tuple(shape)} on {cache.device}")
    return t


def _norm(w, what: str, cache: Cache):
    if w is None:
        return None
    if w.dtype is not torch.bfloat16 or w.numel() != cache.head_dim or w.get_device() != cache.index \
            or not w.is_contiguous():
        raise ValueError(f"kv4: {what} must be {cache.head_dim} bf16 values on {cache.device}")
    return w.data_ptr()


def _same_device(cache: Cache, batch: Batch) -> None:
    if batch.index != cache.index:
        raise ValueError(f"kv4: batch on {batch.device}, cache on {cache.device}")


def append(cache: Cache, batch: Batch, q, k: torch.Tensor, v: torch.Tensor, cos=None, sin=None, *, q_norm=None,
           k_norm=None, eps: float = 1e-6, interleaved: bool = False, q_out=None):
    """Rotates (and norms) the step's q and k, writes the 4-bit rows of k and v
    into the cache and returns q as bf16 [T, heads, head_dim] (None without
    q). q, k, v [T, heads, head_dim], bf16 or fp32, views of one fused
    buffer or not. cos, sin fp32 [positions, rot / 2] (`rope_tables`; None: no
    rotation): the first rot elements turn, pairs (i, i + rot / 2), or
    (2i, 2i + 1) when `interleaved`."""
    _same_device(cache, batch)
    T, dtype = batch.tokens, k.dtype
    if dtype not in _DT or v.dtype is not dtype or (q is not None and q.dtype is not dtype):
        raise TypeError("kv4: q, k and v must be all bf16 or all fp32")
    k, kh, k_step = _rows(k, "k", cache, T)
    v, vh, v_step = _rows(v, "v", cache, T)
    if kh != cache.kv_heads or vh != kh:
        raise ValueError(f"kv4: {kh} and {vh} kv heads, the cache {cache.kv_heads}")
    heads = q_step = rot = positions = 0
    q_ptr = q_out_ptr = cos_ptr = sin_ptr = None
    if q is not None:
        q, heads, q_step = _rows(q, "q", cache, T)
        q_out = _output(q_out, q.shape, torch.bfloat16, cache, "q_out")
        q_ptr, q_out_ptr = q.data_ptr(), q_out.data_ptr()
    else:
        q_out = None
    if cos is not None or sin is not None:
        if cos is None or sin is None or cos.shape != sin.shape or cos.dim() != 2 \
                or cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or not cos.is_contiguous() \
                or not sin.is_contiguous() or cos.get_device() != cache.index or sin.get_device() != cache.index:
            raise ValueError("kv4: cos and sin must be contiguous fp32 [positions, rot / 2] on the cache's device")
        positions, rot = cos.shape
        rot *= 2
        cos_ptr, sin_ptr = cos.data_ptr(), sin.data_ptr()
    if T:
        a = _lib.KV4AppendArgs(q_ptr, k.data_ptr(), v.data_ptr(), q_step, k_step, v_step, _DT[dtype], heads,
                               _norm(q_norm, "q_norm", cache), _norm(k_norm, "k_norm", cache), eps, rot,
                               1 if interleaved else 0, cos_ptr, sin_ptr, positions, q_out_ptr)
        _call(cache.index, "dm_kv4_append", cache.c, batch.c, a)
    return q_out


def read(cache: Cache, batch: Batch, *, dtype: torch.dtype = torch.bfloat16, k_out=None, v_out=None):
    """The rows of the batch's new tokens as the cache holds them: (k, v)
    [T, kv_heads, head_dim] in `dtype` (bf16 or fp32), or that of k_out."""
    _same_device(cache, batch)
    shape = (batch.tokens, cache.kv_heads, cache.head_dim)
    if k_out is not None:
        dtype = k_out.dtype
    if dtype not in _DT:
        raise TypeError(f"kv4: rows are read as bf16 or fp32, not {dtype}")
    k_out, v_out = _output(k_out, shape, dtype, cache, "k_out"), _output(v_out, shape, dtype, cache, "v_out")
    if batch.tokens:
        _call(cache.index, "dm_kv4_read", cache.c, batch.c, k_out.data_ptr(), v_out.data_ptr(), _DT[dtype])
    return k_out, v_out


def attention(cache: Cache, batch: Batch, q: torch.Tensor, *, scale: float | None = None, window: int = 0, out=None,
              out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Causal grouped-query attention of the new tokens over the cache: q bf16
    [T, heads, head_dim] -> [T, heads, head_dim] in `out_dtype` (or that of
    out). `scale` is 1 / sqrt(head_dim) unless given; `window`: a token sees
    at most that many of the last positions, its own among them (0: all); pages
    before every new token's window need not be in the table any more. Rows of no
    sequence become zeros. Weights are rounded to bf16 on the way, also for an fp32
    output."""
    _same_device(cache, batch)
    if q.dtype is not torch.bfloat16:
        raise TypeError(f"kv4: q must be bf16, not {q.dtype}")
    q, heads, step = _rows(q, "q", cache, batch.tokens)
    if q.data_ptr() % 16 or step % 8:
        q, step = q.clone(memory_format=torch.contiguous_format), heads * cache.head_dim
    if out is not None:
        out_dtype = out.dtype
    if out_dtype not in _DT:
        raise TypeError(f"kv4: the output is bf16 or fp32, not {out_dtype}")
    out = _output(out, q.shape, out_dtype, cache, "out")
    batch.reserve(cache, heads)
    if scale is None:
        scale = 1.0 / math.sqrt(cache.head_dim)
    if batch.tokens:
        _call(cache.index, "dm_kv4_attention", cache.c, batch.c, q.data_ptr(), step, heads, scale, window,
              out.data_ptr(), _DT[out_dtype])
    return out


def rope_tables(rot: int, positions: int, theta: float = 1e6, *, scaling: dict | None = None, device="cuda"):
    """cos, sin fp32 [positions, rot / 2] of the angles p * f_i, f_i =
    theta^(-2i / rot), computed in float64. `scaling` stretches them for
    contexts longer than the trained one (`original` positions) by `factor`:

      {"type": "linear", "factor"}: every f_i divided by factor.
      {"type": "yarn", "factor", "original", "beta_fast": 32, "beta_slow": 1}:
        f_i kept where it turns over `beta_fast` times within the trained context, divided
        where under `beta_slow` times, a linear ramp over i between; cos and
        sin times 0.1 ln(factor) + 1 (Peng et al. 2023).
      {"type": "bands", "factor", "original", "low": 1, "high": 4}: kept where it turns
        over `high` times, divided where under `low`, between them blended by
        the number of turns."""
    if rot % 16 or rot < 16:
        raise ValueError(f"kv4: rot must be a multiple of 16, not {rot}")
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    gain = 1.0
    if scaling is not None:
        kind, factor = scaling["type"], float(scaling["factor"])
        if factor < 1.0:
            raise ValueError(f"kv4: a rotary scaling factor below 1: {factor}")
        if kind == "linear":
            f = f / factor
        elif kind == "yarn":
            n = float(scaling["original"])

            def index_of(turns):  # the i whose frequency turns that often in n positions
                return rot * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(theta))

            low = max(0, math.floor(index_of(float(scaling.get("beta_fast", 32)))))
            high = min(rot - 1, math.ceil(index_of(float(scaling.get("beta_slow", 1)))))
            ramp = ((torch.arange(rot // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
            f = f * (1 - ramp) + f / factor * ramp
            gain = 0.1 * math.log(factor) + 1.0
        elif kind == "bands":
            low, high = float(scaling.get("low", 1)), float(scaling.get("high", 4))
            turns = float(scaling["original"]) * f / (2 * math.pi)
            keep = ((turns - low) / (high - low)).clamp(0, 1)
            f = f * keep + f / factor * (1 - keep)
        else:
            raise ValueError(f"kv4: unknown rotary scaling {kind!r}")
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * f[None, :]
    return (ang.cos() * gain).float().to(device), (ang.sin() * gain).float().to(device)
