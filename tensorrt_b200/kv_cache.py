"""The paged key-value cache of a decoder that generates text, and the attention around it.

    paged_append      K and V rows of new tokens into their pages (FP8 E4M3 pages: quantized under a calibrated abs-max)
    paged_attention   one new token of every sequence over its pages
    paged_evict       the keys of the largest attention weights stay, their rows move to fresh pages
    window_attention  causal attention with a sliding window and sinks over contiguous K and V (prompts and their chunks)

Pages are tensors [pages, kv heads, rows, D] (any strides with D contiguous) of float16, bfloat16, float8_e4m3fn or uint8 (FP8
codes); token t of sequence b is row t % rows of page block_table[b, t // rows].  `lens` [B] counts the tokens of each sequence that
are in the cache, the newest included, in every call.  Everything is enqueued on the current stream of the tensors' device, nothing
synchronises, and the calls can be captured in a CUDA graph.
"""
from __future__ import annotations

import torch

from . import _native
from .ops import load_ops

load_ops()
_ops = torch.ops.tensorrt
_append, _attention = _ops.b200_paged_append.default, _ops.b200_paged_attention.default
_evict, _window = _ops.b200_paged_evict.default, _ops.b200_window_attention.default


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                 cu_new: torch.Tensor | None = None, *, k_amax: torch.Tensor | None = None, v_amax: torch.Tensor | None = None) -> None:
    """Writes k, v [tokens, kv heads, D] into the pages.  The tokens of sequence b are rows cu_new[b] .. cu_new[b + 1] and the last of
    its lens[b] (cu_new None: one token of every sequence).  FP8 pages: codes of x / (amax / 448), `k_amax` and `v_amax` one value or
    one per kv head."""
    if not _native.paged_append(k, v, k_pages, v_pages, block_table, lens, cu_new, k_amax, v_amax):
        _append(k, v, k_pages, v_pages, block_table, lens, cu_new, k_amax, v_amax)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, *,
                    k_amax: torch.Tensor | None = None, v_amax: torch.Tensor | None = None, weights: torch.Tensor | None = None,
                    scale: float | None = None, window: int = 0, sinks: int = 0) -> torch.Tensor:
    """softmax(q K^T * scale) V of one new token of every sequence: q [B, query heads, D] -> the same shape and type.  With
    window > 0 the token sees the last `window` keys and the first `sinks`.  `weights` (float32 [B, kv heads, keys]) gets each seen
    key's attention weight added, summed over the query heads of its kv head.  scale None: 1 / sqrt(D)."""
    args = (q, k_pages, v_pages, block_table, lens, weights, k_amax, v_amax, 0.0 if scale is None else scale, window, sinks)
    out = _native.paged_attention(*args)
    return _attention(*args) if out is None else out


def paged_evict(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, weights: torch.Tensor,
                out_table: torch.Tensor, *, keep: int, recent: int = 0, sinks: int = 0):
    """Cuts every sequence to `keep` tokens per kv head: the first `sinks`, the last `recent` and, of the others, those with the
    largest weights (equal ones: the lower token).  Their rows move, in order, to the pages of `out_table` [B, pages], which must not
    be among the pages read.  -> (kept tokens int32 [B, kv heads, keep], -1 beyond a shorter sequence; new lens; new weights)."""
    args = (k_pages, v_pages, block_table, lens, weights, out_table, keep, recent, sinks)
    out = _native.paged_evict(*args)
    return _evict(*args) if out is None else out


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None, window: int = 0, sinks: int = 0,
                     q_lens: torch.Tensor | None = None, k_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Causal (lower-right aligned) attention: q [B, query heads, Sq, D], k and v [B, kv heads, Sk, D] -> q's shape and type.  With
    window > 0 a query sees the last `window` keys up to its own and the first `sinks`.  `q_lens`, `k_lens` int32 [B]: the queries and
    keys that each sequence has; rows beyond them, and rows that see no key, are zero.  scale None: 1 / sqrt(D)."""
    args = (q, k, v, q_lens, k_lens, 0.0 if scale is None else scale, window, sinks)
    out = _native.window_attention(*args)
    return _window(*args) if out is None else out
