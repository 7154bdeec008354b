"""Logits before a token is chosen: penalties for repeated tokens, biases and a
grammar's mask, one launch over a batch (csrc/logits.cu behind the C ABI's
dm_logits_process, which gives the formula). The reference does this in Python
over one row (src/drinkme/serving/sampling.py).

    y = logits.process(x, history=ids, prompt_len=n0, total_len=n, repetition=r, allowed=mask)
"""
from __future__ import annotations

import torch

from . import _lib
from .kv4 import _call

_DT = {torch.bfloat16: _lib.DM_BF16, torch.float32: _lib.DM_F32}


def _table(t, what: str, dtype, index: int, rows: int, cols: int):
    """Pointer and row length of an optional [rows, cols or more] tensor."""
    if t is None:
        return None, 0
    if t.dtype is not dtype:
        raise TypeError(f"logits: {what} must be {dtype}, not {t.dtype}")
    shape = t.shape
    if t.get_device() != index or len(shape) != 2 or shape[0] != rows or shape[1] < cols or not t.is_contiguous():
        raise ValueError(f"logits: {what} must be contiguous [{rows}, {cols or 'n'}] on the logits' device, "
                         f"not {tuple(shape)} on {t.device}")
    return t.data_ptr(), shape[1]


def _values(t, what: str, dtype, index: int, rows: int):
    """Pointer of an optional tensor of one value a row."""
    if t is None:
        return None
    if t.dtype is not dtype:
        raise TypeError(f"logits: {what} must be {dtype}, not {t.dtype}")
    if t.get_device() != index or t.numel() != rows or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"logits: {what} must be one contiguous value a row on the logits' device")
    return t.data_ptr()


def process(x: torch.Tensor, *, history=None, prompt_len=None, total_len=None, repetition=None, presence=None,
            frequency=None, bias_ids=None, bias_values=None, allowed=None, out=None) -> torch.Tensor:
    """x [rows, vocab], bf16 or fp32 -> the same type (`out` may be x itself).

    history     int32 [rows, n]: a row's token ids, the prompt's first, then those
                generated; ids outside the vocabulary count nothing
    prompt_len, total_len  int32 [rows]: how many ids are the prompt's (none by
                default) and how many count (all by default)
    repetition  fp32 [rows]: the logit of a token seen anywhere in the history
                is divided by it when positive, else multiplied
    frequency, presence  fp32 [rows]: frequency times the number of times the
                token was generated, and presence when it was, are taken off
    bias_ids, bias_values  int32, fp32 [rows, k]: added (an id outside the vocabulary,
                -1 say, marks an empty place; of places that name one id the last counts)
    allowed     int32 [rows, ceil(vocab / 32)]: token v's bit v % 32 of word v / 32;
                tokens without it become -inf

    fp32 arithmetic, one rounding at the end; a row whose mask allows nothing is
    all -inf."""
    index, dtype = x.get_device(), x.dtype
    if index < 0:
        raise ValueError(f"logits: the logits must be on a CUDA device, not {x.device}")
    if dtype not in _DT:
        raise TypeError(f"logits: the logits must be bf16 or fp32, not {dtype}")
    if x.dim() != 2 or x.shape[1] < 1 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError(f"logits: the logits must be [rows, vocab] with contiguous rows, not {tuple(x.shape)}")
    rows, vocab = x.shape
    if rows > 65535 or vocab >= 1 << 31:
        raise ValueError(f"logits: {rows} rows, at most 65535, of a vocabulary of {vocab}, below 2^31")
    if out is None:
        out = torch.empty((rows, vocab), dtype=dtype, device=x.device)
    elif out is not x and (out.dtype is not dtype or out.shape != x.shape or out.get_device() != index
                           or (vocab > 1 and out.stride(1) != 1)):
        raise ValueError("logits: `out` must be like the logits, with contiguous rows")
    if rows == 0:
        return out
    if history is None and (repetition is not None or presence is not None or frequency is not None):
        raise ValueError("logits: penalties need the history")
    if (bias_ids is None) != (bias_values is None) or (bias_ids is not None and bias_ids.shape != bias_values.shape):
        raise ValueError("logits: bias_ids and bias_values come together, with one shape")
    i32, f32 = torch.int32, torch.float32
    hist, hist_cols = _table(history, "history", i32, index, rows, 0)
    bias, bias_cols = _table(bias_ids, "bias_ids", i32, index, rows, 0)
    mask, mask_cols = _table(allowed, "allowed", i32, index, rows, -(-vocab // 32))
    a = _lib.LogitsArgs(x.data_ptr(), out.data_ptr(), x.stride(0), out.stride(0), _DT[dtype], rows, vocab, hist,
                        hist_cols, _values(prompt_len, "prompt_len", i32, index, rows),
                        _values(total_len, "total_len", i32, index, rows),
                        _values(repetition, "repetition", f32, index, rows),
                        _values(presence, "presence", f32, index, rows),
                        _values(frequency, "frequency", f32, index, rows), bias,
                        _table(bias_values, "bias_values", f32, index, rows, 0)[0], bias_cols, mask, mask_cols)
    _call(index, "dm_logits_process", a)
    return out
