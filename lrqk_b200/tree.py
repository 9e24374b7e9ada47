"""Attention of a tree of drafted tokens over a cache: the verification step of speculative decoding.

``tree_attention`` stands beside ``LayerState.flash_decode`` (one query per head over the resident rows): here every query
head brings a row per drafted node, which attends to the cache and to the nodes it descends from.  The cache is an ordinary
one (a key/value row per token and KV head, as ``FullOffloadCache.update`` hands out) or the resident rows of a decoding
layer (``DynamicLRQKCache.attend_tree``).
"""
from __future__ import annotations

import math
from typing import Dict, Optional, Sequence, Union

import torch

from . import _lib
from .state import _DTYPES, call_on, has_tangent

MAX_NODES = 256


def tree_mask(parents: Union[Sequence[int], torch.Tensor], device=None) -> torch.Tensor:
    """bool [T, T] (or [B, T, T] for [B, T] parents): node i sees itself and its ancestors.  ``parents[i]`` is the
    index of an earlier node, or -1 where the node follows the context directly."""
    par = torch.as_tensor(parents, dtype=torch.int64).cpu()
    if par.dim() == 2:
        return torch.stack([tree_mask(p, device) for p in par]) if par.shape[0] else torch.zeros((0, par.shape[1], par.shape[1]), dtype=torch.bool, device=device)
    if par.dim() != 1:
        raise ValueError(f"parents: expected [T] or [B, T], got {tuple(par.shape)}")
    t = par.shape[0]
    mask = torch.zeros((t, t), dtype=torch.bool)
    for i, p in enumerate(par.tolist()):
        if not -1 <= p < i:
            raise ValueError(f"parents[{i}] = {p}: a node's parent is an earlier node or -1")
        if p >= 0:
            mask[i] = mask[p]
        mask[i, i] = True
    return mask if device is None else mask.to(device)


_status: Dict[int, torch.Tensor] = {}


def _status_word(device: torch.device) -> Optional[int]:
    """Address of the device's status word.  Made and cleared once, with a synchronisation so that every stream finds it
    cleared; a first call under capture goes without one (its clearing would only run at the replays) and has one of its own,
    cleared at every replay: its rows turn NaN all the same, but nobody is told."""
    word = _status.get(device.index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            return None
        word = torch.zeros(4, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()
        word = _status.setdefault(device.index, word)            # (two threads' first calls: one word)
    return word.data_ptr()


def check_tree_status(device=None) -> None:
    """Synchronising look at the status word of a device's ``tree_attention`` calls, on whichever stream: raises
    ``LrqkError`` if a bounded wait of one ran out (its rows, and those of later calls until this look, are NaN), and
    clears it.  A graph whose capture held the device's very first call has a word of its own that this look does not see."""
    index = torch.cuda.current_device() if device is None or torch.device(device).index is None else torch.device(device).index
    word = _status.get(index)
    if word is None:
        return
    torch.cuda.synchronize(index)                                # calls of other streams than the current one
    code = int(word[0])
    if code != 0:
        word.zero_()
        torch.cuda.synchronize(index)                            # the next call on any stream finds it cleared
        raise _lib.LrqkError(code, "lrqk_tree_attention", _lib.lib().lrqk_strerror(code).decode())


def _refuse_rows(**tensors):
    for name, x in tensors.items():
        s, e = x.stride(), x.element_size()
        if x.numel() and (x.data_ptr() % 16 or any(n > 1 and v * e % 16 for n, v in zip(x.shape[:3], s))):
            raise ValueError(f"{name}: rows must start on 16 bytes; strides {tuple(s)} at address {x.data_ptr():#x}")


def tree_attention(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, tree_k: torch.Tensor, tree_v: torch.Tensor,
                   mask: Optional[torch.Tensor] = None, *, cache_lens: Optional[torch.Tensor] = None,
                   scale: Optional[float] = None, return_lse: bool = False):
    """Attention of ``q`` [B, Hq, T, d] over the first ``cache_lens[b]`` rows of ``cache_k`` / ``cache_v`` [B, Hc, S, d]
    and over the drafted nodes ``tree_k`` / ``tree_v`` [B, Ht, T, d] that each node sees (``lrqk_tree_attention``).

    * ``mask``: bool (or uint8) [T, T] or [B, T, T], ``mask[i, j]``: node i sees node j (:func:`tree_mask`); ``None``: a
      chain, node i sees nodes 0..i
    * ``cache_lens``: int32 [B] on the device, read when the kernel runs (a captured call follows it), cut to [0, S];
      ``None``: all S rows.  Rows behind a length may hold anything (an infinite value before it gives infinity or NaN)
    * ``Ht`` divides ``Hc`` divides ``Hq``; query head h reads cache head ``h // (Hq / Hc)`` and drafted head
      ``h // (Hq / Ht)``
    * ``scale``: default ``d ** -0.5``; T up to 256, d 64 or 128, float32 or bfloat16

    Strided inputs (and expanded batches and heads) are read as they are as long as rows are dense and start on 16 bytes.  Inference only (no gradient).
    Returns [B, Hq, T, d], with ``return_lse`` also the fp32 [B, Hq, T] natural log-sum-exp; a row that sees nothing gives
    zeros and -inf."""
    if q.dim() != 4 or q.dtype not in _DTYPES or not q.is_cuda:
        raise ValueError(f"q: expected a float32 or bfloat16 CUDA tensor [batch, heads, nodes, head_dim], got {q.dtype} {tuple(q.shape)} on {q.device}")
    b, hq, t, d = q.shape
    device, dtype = q.device, q.dtype
    if cache_k.dim() != 4 or tree_k.dim() != 4:
        raise ValueError(f"cache_k, tree_k: expected [{b}, heads, rows, {d}], got {tuple(cache_k.shape)}, {tuple(tree_k.shape)}")
    cb, hc, cap, cd = cache_k.shape
    tb, ht, tt, td = tree_k.shape
    if not (cb == tb == b and cd == td == d and tt == t and cache_v.shape == cache_k.shape and tree_v.shape == tree_k.shape
            and cache_k.dtype is dtype and cache_v.dtype is dtype and tree_k.dtype is dtype and tree_v.dtype is dtype
            and cache_k.device == device and cache_v.device == device and tree_k.device == device and tree_v.device == device):
        raise ValueError(f"cache_k, cache_v: expected {dtype} [{b}, cache heads, rows, {d}], tree_k, tree_v: [{b}, tree heads, {t}, {d}], all on {device}; got "
                         + ", ".join(f"{n} {x.dtype} {tuple(x.shape)} on {x.device}"
                                     for n, x in (("cache_k", cache_k), ("cache_v", cache_v), ("tree_k", tree_k), ("tree_v", tree_v))))
    if hc == 0 or ht == 0 or hq == 0 or hq % hc or hc % ht:
        raise ValueError(f"heads: tree heads divide cache heads divide query heads; got q {hq}, cache {hc}, tree {ht}")
    if t > MAX_NODES:
        raise ValueError(f"at most {MAX_NODES} nodes, got {t}")
    if d not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {d}")
    if torch.is_grad_enabled() and (q.requires_grad or cache_k.requires_grad or cache_v.requires_grad or tree_k.requires_grad or tree_v.requires_grad):
        raise ValueError("tree_attention has no gradient: call it under torch.no_grad()")
    if has_tangent(q, cache_k, cache_v, tree_k, tree_v):
        raise ValueError("tree_attention has no forward-mode derivative: call it on the primals")
    scale = d ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    qs, ks, vs, tks, tvs = q.stride(), cache_k.stride(), cache_v.stride(), tree_k.stride(), tree_v.stride()
    if not qs[3] == ks[3] == vs[3] == tks[3] == tvs[3] == 1:
        raise ValueError("q, cache_k, cache_v, tree_k, tree_v: rows must be dense (last stride 1)")
    if (cap > 1 and not (ks[2] and vs[2])) or (t > 1 and not (qs[2] and tks[2] and tvs[2])):
        raise ValueError("q, cache_k, cache_v, tree_k, tree_v: one row expanded to many is not supported")
    mask_at = lens_at = lse_at = None
    mask_stride = 0
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8) or mask.device != device or mask.shape[-2:] != (t, t) or \
                not (mask.dim() == 2 or (mask.dim() == 3 and mask.shape[0] in (1, b))):
            raise ValueError(f"mask: expected bool [{t}, {t}] or [{b}, {t}, {t}] on {device}, got {mask.dtype} {tuple(mask.shape)} on {mask.device}")
        mask = mask.contiguous()
        mask_at, mask_stride = mask.data_ptr(), t * t if mask.dim() == 3 and mask.shape[0] > 1 else 0
    if cache_lens is not None:
        if cache_lens.dtype is not torch.int32 or cache_lens.device != device or cache_lens.shape != (b,) or not cache_lens.is_contiguous():
            raise ValueError(f"cache_lens: expected contiguous int32 [{b}] on {device}, got {cache_lens.dtype} {tuple(cache_lens.shape)} on {cache_lens.device}")
        lens_at = cache_lens.data_ptr()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = None
    if return_lse:
        lse = torch.empty((b, hq, t), dtype=torch.float32, device=device)
        lse_at = lse.data_ptr()
    if b and t:
        lib = _lib.lib()
        a = _lib.TreeArgs(_DTYPES[dtype], b, t, hq, hc, ht, d, scale, cap, q.data_ptr(), cache_k.data_ptr(), cache_v.data_ptr(),
                          tree_k.data_ptr(), tree_v.data_ptr(), qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                          tks[0], tks[1], tks[2], tvs[0], tvs[1], tvs[2], lens_at, mask_at, mask_stride, out.data_ptr(), lse_at,
                          _status_word(device))
        ws = torch.empty(lib.lrqk_tree_attention_workspace_bytes(a), dtype=torch.uint8, device=device)
        code = call_on(device, lib.lrqk_tree_attention, a, ws.data_ptr())
        if code == _lib.EUNSUPPORTED:
            _refuse_rows(q=q, cache_k=cache_k, cache_v=cache_v, tree_k=tree_k, tree_v=tree_v)
        _lib.check(code, "lrqk_tree_attention")
    return (out, lse) if return_lse else out
