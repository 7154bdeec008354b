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


def _table(t, what: str, dtype, x: torch.Tensor, cols: int | None):
    """Pointer and row stride of an optional [rows, n] tensor."""
    if t is None:
        return None, 0
    if t.dtype != dtype:
        raise TypeError(f"logits: {what} must be {dtype}, not {t.dtype}")
    if t.device != x.device or t.dim() != 2 or t.shape[0] != x.shape[0] or (cols is not None and t.shape[1] < cols):
        raise ValueError(f"logits: {what} is {tuple(t.shape)} on {t.device} for logits {tuple(x.shape)} on {x.device}")
    if not t.is_contiguous():
        raise ValueError(f"logits: {what} must be contiguous")
    return t.data_ptr(), t.shape[1]


def _row_values(t, what: str, dtype, x: torch.Tensor):
    if t is None:
        return None
    if t.dtype != dtype:
        raise TypeError(f"logits: {what} must be {dtype}, not {t.dtype}")
    if t.device != x.device or t.dim() != 1 or t.shape[0] != x.shape[0] or not t.is_contiguous():
        raise ValueError(f"logits: {what} must be one contiguous value a row on {x.device}")
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
    if x.device.type != "cuda":
        raise ValueError(f"logits: the logits must be on a CUDA device, not {x.device}")
    if x.dtype not in _DT:
        raise TypeError(f"logits: the logits must be bf16 or fp32, not {x.dtype}")
    if x.dim() != 2 or x.shape[1] < 1 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError(f"logits: the logits must be [rows, vocab] with contiguous rows, not {tuple(x.shape)}")
    rows, vocab = x.shape
    if rows > 65535:
        raise ValueError(f"logits: {rows} rows, at most 65535")
    if out is None:
        out = torch.empty((rows, vocab), dtype=x.dtype, device=x.device)
    elif out.dtype != x.dtype or out.shape != x.shape or out.device != x.device or (vocab > 1 and out.stride(1) != 1):
        raise ValueError("logits: `out` must be like the logits, with contiguous rows")
    if rows == 0:
        return out
    if history is None and (repetition is not None or presence is not None or frequency is not None):
        raise ValueError("logits: penalties need the history")
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("logits: bias_ids and bias_values come together")
    a = _lib.LogitsArgs()
    a.logits, a.out, a.dtype, a.rows, a.vocab = x.data_ptr(), out.data_ptr(), _DT[x.dtype], rows, vocab
    a.stride, a.out_stride = x.stride(0), out.stride(0)
    a.history, a.history_stride = _table(history, "history", torch.int32, x, None)
    a.prompt_len = _row_values(prompt_len, "prompt_len", torch.int32, x)
    a.total_len = _row_values(total_len, "total_len", torch.int32, x)
    a.repetition = _row_values(repetition, "repetition", torch.float32, x)
    a.presence = _row_values(presence, "presence", torch.float32, x)
    a.frequency = _row_values(frequency, "frequency", torch.float32, x)
    if bias_ids is not None:
        if bias_ids.shape != bias_values.shape:
            raise ValueError("logits: bias_ids and bias_values must have one shape")
        a.bias_ids, a.bias_stride = _table(bias_ids, "bias_ids", torch.int32, x, None)
        a.bias_values = _table(bias_values, "bias_values", torch.float32, x, None)[0]
    a.allowed, a.allowed_stride = _table(allowed, "allowed", torch.int32, x, -(-vocab // 32))
    _call(x.device, "dm_logits_process", a)
    return out
