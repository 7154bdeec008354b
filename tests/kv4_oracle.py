"""Plain restatements of the paged 4-bit cache's operators (drinkme_b200.kv4):
the codes in float32 with every operation rounded by itself (numpy), values and
attention in float64."""
from __future__ import annotations

import numpy as np
import torch


def halving_sum(x: np.ndarray) -> np.ndarray:
    while x.shape[-1] > 1:
        h = x.shape[-1] // 2
        x = x[..., :h] + x[..., h:]
    return x[..., 0]


def rotate(x: np.ndarray, w, cos, sin, eps: float, interleaved: bool) -> np.ndarray:
    """x float32 [T, heads, d], cos / sin [T, rot / 2] or None."""
    f = np.float32
    x = x.astype(f)
    if w is not None:
        ss = halving_sum(x * x) * f(1.0 / x.shape[-1]) + f(eps)
        r = f(1.0) / np.sqrt(ss)
        x = (x * r[..., None]) * w.astype(f)
    if cos is None:
        return x
    n = cos.shape[-1]
    c, s = cos[:, None].astype(f), sin[:, None].astype(f)
    y = x.copy()
    i = np.arange(n)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def bf16(x: np.ndarray) -> np.ndarray:
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16).float().numpy()


def quantise(y: np.ndarray):
    """(s, m, codes uint8) of float32 rows; rows that are held as NaN have s = m = NaN."""
    f = np.float32
    with np.errstate(all="ignore"):
        lo, hi = y.min(-1), y.max(-1)
        m, s = bf16(lo), bf16((hi - lo) * f(1.0 / 15.0))
        nan = ~np.isfinite(y).all(-1) | ~np.isfinite(s) | ~np.isfinite(m)
        tiny = s < np.finfo(f).tiny
        s = np.where(tiny, f(0), s)
        inv = np.where(tiny, f(0), f(1) / np.where(tiny, f(1), s))
        c = np.clip(np.rint((y - m[..., None]) * inv[..., None]), 0, 15)
        c = np.where((nan | tiny)[..., None], 0, c).astype(np.uint8)
    return np.where(nan, f(np.nan), s), np.where(nan, f(np.nan), m), c


def pack(c: np.ndarray) -> np.ndarray:
    return c[..., 0::2] | (c[..., 1::2] << 4)


def held(codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, b: int, n: int):
    """float64 keys and values [nkv, n, d] of sequence b's first n rows, and
    the value rows' scales [nkv, n] (CPU)."""
    ps = codes.shape[3]
    pages = table[b, : -(-n // ps)].long()
    c, two = codes[pages], scales[pages].double()  # [P, nkv, 2, ps, d / 2], [P, nkv, ps, 4]
    v = torch.stack((c & 15, c >> 4), -1).flatten(-2).double()
    s, m = two[..., 0::2].permute(0, 1, 3, 2), two[..., 1::2].permute(0, 1, 3, 2)
    v = v * s[..., None] + m[..., None]
    v = v.permute(2, 1, 0, 3, 4).flatten(2, 3)[:, :, :n]
    return v[0], v[1], s[:, :, 1].permute(1, 0, 2).flatten(1)[:, :n]


def attention(codes, scales, table, q_lens, kv_lens, q, scale, window: int = 0):
    """float64 (out, slack) [T, nh, d] on the CPU: slack is sum_j p_j (|v_j| + 8 s_j),
    what a relative error of the weights is multiplied by."""
    codes, scales, table, q = codes.cpu(), scales.cpu(), table.cpu(), q.cpu().double()
    T, nh, d = q.shape
    nkv = codes.shape[1]
    grp = nh // nkv
    out, slack, t = torch.zeros(T, nh, d, dtype=torch.float64), torch.zeros(T, nh, d, dtype=torch.float64), 0
    for b, (a, n) in enumerate(zip(q_lens, kv_lens)):
        if a and n:
            K, V, vs = held(codes, scales, table, b, n)
            p = torch.arange(n - a, n)[:, None]
            j = torch.arange(n)[None, :]
            seen = (j <= p) & ((j > p - window) if window else (j >= 0))
            for h in range(nh):
                g = h // grp
                s = (q[t:t + a, h] @ K[g].T) * scale
                s = s.masked_fill(~seen, -float("inf"))
                w = torch.where(seen.any(-1, keepdim=True), torch.softmax(s, -1), torch.zeros_like(s))
                w = torch.where(seen, w, torch.zeros_like(w))
                live = seen.any(0)  # rows that nobody sees may hold anything
                out[t:t + a, h] = w[:, live] @ V[g][live]
                slack[t:t + a, h] = w[:, live] @ (V[g][live].abs() + 8 * vs[g][live][:, None])
        t += a
    return out, slack
