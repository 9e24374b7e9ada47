"""Choice of tokens from logits: temperature, top-k, top-p, min-p and a given random number per row.

What follows the ``argmax`` of the throughput driver (``tps_estimate``) in a program that does not decode greedily; the random
numbers are inputs, so a choice can be repeated, checked and captured."""
from __future__ import annotations

import math
from typing import Tuple, Union

import torch

from . import _lib
from .state import _DTYPES, call_on

Setting = Union[float, int, torch.Tensor]


def _setting(value: Setting, name: str, rows: int, device: torch.device, dtype: torch.dtype, low: float):
    """(address or None, plain value) of one setting."""
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype or value.device != device or value.shape != (rows,) or not value.is_contiguous():
            raise ValueError(f"{name}: expected contiguous {dtype} [{rows}] on {device}, got {value.dtype} {tuple(value.shape)} on {value.device}")
        return value.data_ptr(), 0
    if not math.isfinite(value) or value < low:
        raise ValueError(f"{name} must be finite and at least {low}, got {value}")
    return None, (min(value, 2 ** 31 - 1) if dtype is torch.int32 else value)


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, *, temperature: Setting = 1.0, top_k: Setting = 0, top_p: Setting = 1.0,
                  min_p: Setting = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(tokens int64 [B], their log-probabilities fp32 [B]) of ``logits`` [B, V] and random numbers ``u`` fp32 [B] in [0, 1),
    in one launch (``lrqk_sample_tokens``).

    In this order: ``logits / temperature`` (0: greedy, the first maximum); the ``top_k`` largest (0: all; equal ones from
    the lowest index); of those, in descending order, while the mass before a token is below ``top_p`` of theirs (1: all);
    of those, at least ``min_p`` of the largest's probability (0: all); the first, in index order, whose cumulative
    probability exceeds ``u``.  The log-probability is that of the distribution the token was drawn from.

    Each setting is a number or a tensor [B] on the device (float32; ``top_k`` int32), read when the kernel runs.  NaN
    logits count as -inf; a row without any logit above -inf gives token -1 and NaN.  Nothing here has a gradient."""
    if logits.dim() != 2 or logits.dtype not in _DTYPES or not logits.is_cuda or logits.shape[1] == 0:
        raise ValueError(f"logits: expected a float32 or bfloat16 CUDA tensor [rows, vocab], got {logits.dtype} {tuple(logits.shape)} on {logits.device}")
    rows, vocab = logits.shape
    if u.dtype != torch.float32 or u.device != logits.device or u.shape != (rows,) or not u.is_contiguous():
        raise ValueError(f"u: expected contiguous float32 [{rows}] on {logits.device}, got {u.dtype} {tuple(u.shape)} on {u.device}")
    device = logits.device
    t, t_all = _setting(temperature, "temperature", rows, device, torch.float32, 0.0)
    k, k_all = _setting(top_k, "top_k", rows, device, torch.int32, 0)
    p, p_all = _setting(top_p, "top_p", rows, device, torch.float32, 0.0)
    m, m_all = _setting(min_p, "min_p", rows, device, torch.float32, 0.0)
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    tokens = torch.empty((rows,), dtype=torch.int64, device=device)
    logprobs = torch.empty_like(u)
    if rows:
        a = _lib.SampleArgs(_DTYPES[logits.dtype], rows, vocab, k_all, t_all, p_all, m_all, logits.data_ptr(), logits.stride(0) if rows > 1 else 0,
                            u.data_ptr(), t, p, m, k, tokens.data_ptr(), logprobs.data_ptr())
        _lib.check(call_on(device, _lib.lib().lrqk_sample_tokens, a), "lrqk_sample_tokens")
    return tokens, logprobs
