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
from .state import _DTYPES, _stream, on_device

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
    cleared; a first call under capture goes without one (its clearing would only run at the replays)."""
    word = _status.get(device.index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            return None
        word = torch.zeros(4, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()
        _status[device.index] = word
    return word.data_ptr()


def check_tree_status(device=None) -> None:
    """Synchronising look at the status word of a device's ``tree_attention`` calls: raises ``LrqkError`` if a bounded
    wait of one ran out (its rows, and those of later calls until this look, are NaN), and clears it."""
    index = torch.cuda.current_device() if device is None or torch.device(device).index is None else torch.device(device).index
    word = _status.get(index)
    if word is not None and int(word[0]) != 0:
        code = int(word[0])
        word.zero_()
        raise _lib.LrqkError(code, "lrqk_tree_attention", _lib.lib().lrqk_strerror(code).decode())


def _rows(x: torch.Tensor, name: str, q: torch.Tensor, rows: Optional[int]) -> torch.Tensor:
    if x.dim() != 4 or x.dtype != q.dtype or x.device != q.device or x.shape[0] != q.shape[0] or x.shape[3] != q.shape[3] or \
            (rows is not None and x.shape[2] != rows):
        raise ValueError(f"{name}: expected {q.dtype} [{q.shape[0]}, heads, {'rows' if rows is None else rows}, {q.shape[3]}] on {q.device}, "
                         f"got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x


def _strides(x: torch.Tensor, name: str):
    """(batch, head, row) strides; rows start on 16 bytes.  A dimension of one row has no stride that matters."""
    s, e = x.stride(), x.element_size()
    st = [0 if n == 1 else v for n, v in zip(x.shape[:3], s[:3])]
    if (x.shape[3] > 1 and s[3] != 1) or x.data_ptr() % 16 or any(v * e % 16 for v in st):
        raise ValueError(f"{name}: rows must be dense and start on 16 bytes; strides {tuple(s)} at address {x.data_ptr():#x}")
    return st


def tree_attention(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, tree_k: torch.Tensor, tree_v: torch.Tensor,
                   mask: Optional[torch.Tensor] = None, *, cache_lens: Optional[torch.Tensor] = None,
                   scale: Optional[float] = None, return_lse: bool = False):
    """Attention of ``q`` [B, Hq, T, d] over the first ``cache_lens[b]`` rows of ``cache_k`` / ``cache_v`` [B, Hc, S, d]
    and over the drafted nodes ``tree_k`` / ``tree_v`` [B, Ht, T, d] that each node sees (``lrqk_tree_attention``).

    * ``mask``: bool (or uint8) [T, T] or [B, T, T], ``mask[i, j]``: node i sees node j (:func:`tree_mask`); ``None``: a
      chain, node i sees nodes 0..i
    * ``cache_lens``: int32 [B] on the device, read when the kernel runs (a captured call follows it), cut to [0, S];
      ``None``: all S rows.  Rows behind a length may hold anything.
    * ``Ht`` divides ``Hc`` divides ``Hq``; query head h reads cache head ``h // (Hq / Hc)`` and drafted head
      ``h // (Hq / Ht)``
    * ``scale``: default ``d ** -0.5``; T up to 256, d 64 or 128, float32 or bfloat16

    Strided inputs are read as they are as long as rows are dense and start on 16 bytes.  Inference only (no gradient).
    Returns [B, Hq, T, d], with ``return_lse`` also the fp32 [B, Hq, T] natural log-sum-exp; a row that sees nothing gives
    zeros and -inf."""
    if q.dim() != 4 or q.dtype not in _DTYPES or not q.is_cuda:
        raise ValueError(f"q: expected a float32 or bfloat16 CUDA tensor [batch, heads, nodes, head_dim], got {q.dtype} {tuple(q.shape)} on {q.device}")
    b, hq, t, d = q.shape
    _rows(cache_k, "cache_k", q, None)
    _rows(cache_v, "cache_v", q, cache_k.shape[2])
    _rows(tree_k, "tree_k", q, t)
    _rows(tree_v, "tree_v", q, t)
    hc, ht, cap = cache_k.shape[1], tree_k.shape[1], cache_k.shape[2]
    if cache_v.shape[1] != hc or tree_v.shape[1] != ht or hc == 0 or ht == 0 or hq % hc or hc % ht or hq == 0:
        raise ValueError(f"heads: keys and values alike, tree heads dividing cache heads dividing query heads; got q {hq}, "
                         f"cache {hc} / {cache_v.shape[1]}, tree {ht} / {tree_v.shape[1]}")
    if t > MAX_NODES:
        raise ValueError(f"at most {MAX_NODES} nodes, got {t}")
    if d not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {d}")
    if torch.is_grad_enabled() and (q.requires_grad or cache_k.requires_grad or cache_v.requires_grad or tree_k.requires_grad or tree_v.requires_grad):
        raise ValueError("tree_attention has no gradient: call it under torch.no_grad()")
    scale = d ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    out = torch.empty((b, hq, t, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((b, hq, t), dtype=torch.float32, device=q.device) if return_lse else None
    if out.numel() == 0:
        return (out, lse) if return_lse else out
    a = _lib.TreeArgs()
    a.dtype, a.batch, a.nodes, a.q_heads, a.cache_heads, a.tree_heads, a.head_dim = _DTYPES[q.dtype], b, t, hq, hc, ht, d
    a.scale, a.capacity = scale, cap
    a.q, a.q_stride[:] = q.data_ptr(), _strides(q, "q")
    if cap:
        a.cache_k, a.cache_k_stride[:] = cache_k.data_ptr(), _strides(cache_k, "cache_k")
        a.cache_v, a.cache_v_stride[:] = cache_v.data_ptr(), _strides(cache_v, "cache_v")
    a.tree_k, a.tree_k_stride[:] = tree_k.data_ptr(), _strides(tree_k, "tree_k")
    a.tree_v, a.tree_v_stride[:] = tree_v.data_ptr(), _strides(tree_v, "tree_v")
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8) or mask.device != q.device or mask.shape[-2:] != (t, t) or \
                not (mask.dim() == 2 or (mask.dim() == 3 and mask.shape[0] in (1, b))):
            raise ValueError(f"mask: expected bool [{t}, {t}] or [{b}, {t}, {t}] on {q.device}, got {mask.dtype} {tuple(mask.shape)} on {mask.device}")
        mask = mask.contiguous()
        a.mask, a.mask_stride = mask.data_ptr(), t * t if mask.dim() == 3 and mask.shape[0] > 1 else 0
    if cache_lens is not None:
        if cache_lens.dtype != torch.int32 or cache_lens.device != q.device or cache_lens.shape != (b,) or not cache_lens.is_contiguous():
            raise ValueError(f"cache_lens: expected contiguous int32 [{b}] on {q.device}, got {cache_lens.dtype} {tuple(cache_lens.shape)} on {cache_lens.device}")
        a.cache_lens = cache_lens.data_ptr()
    a.out, a.lse = out.data_ptr(), None if lse is None else lse.data_ptr()
    lib = _lib.lib()
    with on_device(q.device):
        a.status = _status_word(q.device)
        ws = torch.empty((lib.lrqk_tree_attention_workspace_bytes(a),), dtype=torch.uint8, device=q.device)
        _lib.check(lib.lrqk_tree_attention(a, ws.data_ptr(), _stream()), "lrqk_tree_attention")
    return (out, lse) if return_lse else out
