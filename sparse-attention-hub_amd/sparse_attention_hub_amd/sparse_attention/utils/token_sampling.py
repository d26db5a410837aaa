"""The next token of each row of logits: temperature, top-k, top-p and min-p from given random numbers.

The reference's adapter answers greedily (`adapters/huggingface.py:417-484`); with a temperature of 0 this is that. The random numbers are an
input, so that the same numbers give the same tokens on every run; the caller's generator makes them.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from ... import _native as N

Setting = Union[None, float, int, torch.Tensor]


def _setting(value: Setting, what: str, off: float, dtype: torch.dtype, rows: int, device: torch.device):
    """(pointer to one value per row or None, the one value for all)"""
    if value is None:
        return None, off
    if not isinstance(value, torch.Tensor):
        if value != value:
            raise ValueError(f"{what} is NaN")
        if dtype == torch.int32 and not (value == value // 1 and -2 ** 31 <= value < 2 ** 31):
            raise ValueError(f"{what} must be a whole number that fits 32 bits, got {value}")
        return None, int(value) if dtype == torch.int32 else float(value)
    if value.device != device or value.dtype != dtype or value.shape != (rows,) or not value.is_contiguous():
        raise ValueError(f"{what} must be a number or a contiguous {dtype} tensor of {rows} values on {device}, got {value.dtype} "
                         f"{tuple(value.shape)} on {value.device}")
    return value.data_ptr(), off


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, temperature: Setting = None, top_k: Setting = None,
                  top_p: Setting = None, min_p: Setting = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token per row of `logits` `(rows, vocab)` from one number of `uniforms` `(rows,)` (float32 or float64, in [0, 1)) per row.

    Each setting is a number or a tensor of one value per row (float32; `top_k` int32). Applied in this order, ties going to the
    lower index: weights `exp((x - max) / temperature)` (default 1; at most 0: the largest logit); `top_k` largest (at most 0: all); of those
    the smallest first part whose weight reaches `top_p` of theirs (1 or more: all); of those the ones of at least `min_p` times the largest
    weight. The token is the first by index at which the running sum of the kept weights passes `uniforms` times their sum.
    NaN logits count as -inf. Returns int64 tokens (-1 for a row without a logit above -inf) and the float32 logarithms of their shares of the
    kept weight. Up to 2^20 logits a row; float32, bfloat16 or float16.
    """
    N.require_device(logits, "logits")
    device = logits.device
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be (rows, vocab), got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if logits.stride(1) != 1 and vocab > 1 or rows > 1 and logits.stride(0) < vocab:
        raise ValueError("logits' rows must be contiguous and apart")
    if uniforms.device != device or uniforms.dtype not in (torch.float32, torch.float64) or uniforms.shape != (rows,) \
            or not uniforms.is_contiguous():
        raise ValueError(f"uniforms must be {rows} contiguous float32 or float64 values on {device}, got {uniforms.dtype} "
                         f"{tuple(uniforms.shape)} on {uniforms.device}")
    t_ptr, t = _setting(temperature, "temperature", 1.0, torch.float32, rows, device)
    k_ptr, k = _setting(top_k, "top_k", 0, torch.int32, rows, device)
    p_ptr, p = _setting(top_p, "top_p", 1.0, torch.float32, rows, device)
    m_ptr, m = _setting(min_p, "min_p", 0.0, torch.float32, rows, device)
    tokens = torch.empty(rows, dtype=torch.int64, device=device)
    logprobs = torch.empty(rows, dtype=torch.float32, device=device)
    args = N.SampleArgs(
        logits.data_ptr(), max(logits.stride(0), vocab), N.dtype_code(logits.dtype), rows, vocab,
        uniforms.data_ptr(), int(uniforms.dtype == torch.float64), t_ptr, k_ptr, p_ptr, m_ptr, t, k, p, m,
        tokens.data_ptr(), logprobs.data_ptr(), N.stream_ptr(device))
    size = N.sample_work_bytes(args)
    if size:
        work = torch.empty(size, dtype=torch.uint8, device=device)
        args.work, args.work_bytes = work.data_ptr(), size
    N.call_on(device, "sah_sample_tokens", args)
    return tokens, logprobs
