"""Rotary positions of queries and keys: frequencies (plain and scaled for long contexts) and their application.

``apply_rotary`` stands beside ``LayerState.rope_qkv``: that one turns a single decode token by the cos/sin rows a model's
rotary module made, in the model's rounding; this one takes positions and frequencies, works for whole prompts, single
tokens and drafted trees, keeps the angle right at positions of millions, and has the adjoint (gradient).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from .state import _DTYPES, call_on, has_tangent


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None, seq_len: Optional[int] = None,
                       device=None) -> Tuple[torch.Tensor, float]:
    """(inv_freq float64 [rotary_dim / 2] in radians per position, factor on cosine and sine).

    ``scaling`` names a stretch of the context in the words of a model's configuration (``rope_type`` or ``type``):

    * ``default``: ``base ** (-2 i / rotary_dim)``
    * ``linear``: divided by ``factor`` (position interpolation)
    * ``dynamic``: the base grown for ``seq_len`` tokens beyond ``original_max_position_embeddings`` (NTK-aware)
    * ``yarn``: slow pairs divided by ``factor``, pairs that turn more than ``beta_fast`` times over the original context
      left alone, a linear ramp between (down to ``beta_slow``); cosine and sine scaled by ``attention_factor``, by default
      ``0.1 ln(factor) + 1`` (or the ratio of that with ``mscale`` and ``mscale_all_dim``)
    * ``llama3``: bands by wavelength between ``low_freq_factor`` and ``high_freq_factor``
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"base must be positive and finite, got {base}")
    s = dict(scaling or {})
    kind = s.get("rope_type", s.get("type", "default")) or "default"
    exponent = torch.arange(rotary_dim // 2, dtype=torch.float64) * (2.0 / rotary_dim)
    inv = float(base) ** -exponent
    out = 1.0
    if kind != "default":
        if "factor" not in s or not s["factor"] >= 1.0:
            raise ValueError(f"rotary scaling {kind!r} needs a factor of at least 1")
        f = float(s["factor"])
        original = s.get("original_max_position_embeddings")
        if kind in ("dynamic", "yarn", "llama3") and not (original and original > 0):
            raise ValueError(f"rotary scaling {kind!r} needs original_max_position_embeddings")
    if kind == "default":
        pass
    elif kind == "linear":
        inv = inv / f
    elif kind == "dynamic":
        if rotary_dim < 4:
            raise ValueError("rotary scaling 'dynamic' needs a rotary_dim of at least 4")
        n = max(int(seq_len or original), int(original))
        inv = (float(base) * (f * n / original - (f - 1.0)) ** (rotary_dim / (rotary_dim - 2.0))) ** -exponent
    elif kind == "yarn":
        fast, slow = float(s.get("beta_fast") or 32.0), float(s.get("beta_slow") or 1.0)
        # index of the pair that turns r times over the original context
        pair = lambda r: rotary_dim * math.log(original / (r * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = pair(fast), pair(slow)
        if s.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rotary_dim - 1)
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        inv = inv / f * ramp + inv * (1.0 - ramp)
        m = lambda w: 1.0 if f <= 1.0 else 0.1 * w * math.log(f) + 1.0  # noqa: E731
        if s.get("attention_factor") is not None:
            out = float(s["attention_factor"])
        elif s.get("mscale") and s.get("mscale_all_dim"):
            out = m(float(s["mscale"])) / m(float(s["mscale_all_dim"]))
        else:
            out = m(1.0)
    elif kind == "llama3":
        lo, hi = float(s.get("low_freq_factor", 1.0)), float(s.get("high_freq_factor", 4.0))
        if not hi > lo:
            raise ValueError("rotary scaling 'llama3' needs high_freq_factor > low_freq_factor")
        smooth = ((original * inv / (2 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)
        inv = inv / f * (1.0 - smooth) + inv * smooth
    else:
        raise ValueError(f"unknown rotary scaling {kind!r}")
    return (inv if device is None else inv.to(device)), out


def _rotate(q, k, positions, inv_freq, factor, interleaved, adjoint):
    b, hq, n, d = q.shape
    qs = q.stride()
    if qs[3] != 1 and d > 1:
        q = q.contiguous()
        qs = q.stride()
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if k is None:
        hk, k_out, k_at, k_to, ks = 0, None, None, None, (0, 0, 0)
    else:
        ks = k.stride()
        if ks[3] != 1 and d > 1:
            k = k.contiguous()
            ks = k.stride()
        hk, k_out = k.shape[1], torch.empty_like(k, memory_format=torch.contiguous_format)
        k_at, k_to = k.data_ptr(), k_out.data_ptr()
    if b and n:
        a = _lib.RotaryArgs(_DTYPES[q.dtype], b, n, hq, hk, d, 2 * inv_freq.shape[0], interleaved, adjoint, positions.dtype is torch.int64,
                            q.data_ptr(), k_at, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], q_out.data_ptr(), k_to, positions.data_ptr(),
                            positions.stride(0) if positions.shape[0] > 1 else 0, inv_freq.data_ptr(), factor)
        _lib.check(call_on(q.device, _lib.lib().lrqk_rotary, a), "lrqk_rotary")
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """The rotation is linear: its gradient is the adjoint rotation of the gradients, its tangent that of the tangents."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, factor, interleaved, adjoint):
        ctx.save_for_backward(positions, inv_freq)
        ctx.save_for_forward(positions, inv_freq)
        ctx.how, ctx.two = (factor, interleaved, adjoint), k is not None
        q_out, k_out = _rotate(q, k, positions, inv_freq, factor, interleaved, adjoint)
        return (q_out,) if k is None else (q_out, k_out)

    @staticmethod
    def backward(ctx, gq, gk=None):
        positions, inv_freq = ctx.saved_tensors
        factor, interleaved, adjoint = ctx.how
        got = apply_rotary(gq, gk, positions, inv_freq, factor=factor, interleaved=interleaved, adjoint=not adjoint)
        gq, gk = got if gk is not None else (got, None)
        return gq, gk, None, None, None, None, None

    @staticmethod
    def jvp(ctx, dq, dk, *_):
        positions, inv_freq = ctx.saved_tensors
        factor, interleaved, adjoint = ctx.how
        turn = lambda x: None if x is None else apply_rotary(x, None, positions, inv_freq, factor=factor, interleaved=interleaved, adjoint=adjoint)  # noqa: E731
        return (turn(dq), turn(dk)) if ctx.two else (turn(dq),)


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor, *,
                 factor: float = 1.0, interleaved: bool = False, adjoint: bool = False):
    """Rotate ``q`` [B, Hq, L, d] and ``k`` [B, Hk, L, d] (or ``None``) by their positions in one launch (``lrqk_rotary``).

    * ``positions``: int64 or int32, [L], [1, L] or [B, L]; any sign, in any order
    * ``inv_freq``, ``factor``: of :func:`rotary_frequencies` (float64 [part / 2], ``part <= d``; the rest of a head is copied)
    * ``interleaved``: pairs are neighbours (x[2i], x[2i+1]) instead of (x[i], x[i + part/2])
    * ``adjoint``: turn backwards with the same factor, which is the gradient of the forward rotation

    Strided inputs (a transposed projection) are read as they are; the results are contiguous.  Differentiable in ``q`` and
    ``k``, backwards and in forward mode (dual tensors).  Returns ``(q', k')``, or ``q'`` when ``k`` is ``None``."""
    if q.dim() != 4 or q.dtype not in _DTYPES or not q.is_cuda:
        raise ValueError(f"q: expected a float32 or bfloat16 CUDA tensor [batch, heads, length, head_dim], got {q.dtype} {tuple(q.shape)} on {q.device}")
    b, _, n, d = q.shape
    device = q.device
    if k is not None and (k.dim() != 4 or k.dtype is not q.dtype or k.device != device or k.shape[0] != b or k.shape[2] != n or k.shape[3] != d):
        raise ValueError(f"k: expected {q.dtype} [{b}, heads, {n}, {d}] on {device}, got {k.dtype} {tuple(k.shape)} on {k.device}")
    if positions.dtype not in (torch.int64, torch.int32) or positions.device != device:
        raise ValueError(f"positions: expected int64 or int32 on {device}, got {positions.dtype} on {positions.device}")
    if positions.dim() == 1:
        positions = positions.unsqueeze(0)
    if positions.dim() != 2 or positions.shape[1] != n or positions.shape[0] not in (1, b):
        raise ValueError(f"positions: expected [{n}], [1, {n}] or [{b}, {n}], got {tuple(positions.shape)}")
    if n > 1 and positions.stride(1) != 1:
        positions = positions.contiguous()
    if inv_freq.dtype is not torch.float64 or inv_freq.device != device or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError(f"inv_freq: expected a contiguous float64 vector on {device}, got {inv_freq.dtype} {tuple(inv_freq.shape)} "
                         f"on {inv_freq.device}")
    if not 0 < 2 * inv_freq.shape[0] <= d:
        raise ValueError(f"inv_freq: {inv_freq.shape[0]} pairs do not fit a head of {d}")
    factor = float(factor)
    if not math.isfinite(factor):
        raise ValueError(f"factor must be finite, got {factor}")
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)) or has_tangent(q, k):
        got = _Rotary.apply(q, k, positions, inv_freq, factor, bool(interleaved), bool(adjoint))
        return got[0] if k is None else got
    got = _rotate(q, k, positions, inv_freq, factor, bool(interleaved), bool(adjoint))
    return got[0] if k is None else got
