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
    its lens[b] (cu_new None: one token of every sequence); rows behind cu_new[B] are written nowhere.  FP8 pages: codes of
    x / (amax / 448), `k_amax` and `v_amax` one value or one per kv head."""
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
    largest weights (equal ones: the lower token).  Tokens in pages that the table does not name are not among those that stay.  The rows
    move, in order, to the pages of `out_table` [B, pages], which must not be among the pages read.  -> (kept tokens int32 [B, kv heads,
    keep], -1 beyond a shorter sequence; new lens; new weights)."""
    args = (k_pages, v_pages, block_table, lens, weights, out_table, keep, recent, sinks)
    out = _native.paged_evict(*args)
    return _evict(*args) if out is None else out


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None, window: int = 0, sinks: int = 0,
                     q_lens: torch.Tensor | None = None, k_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Causal (lower-right aligned) attention: q [B, query heads, Sq, D], k and v [B, kv heads, Sk, D] -> q's shape and type.  With
    window > 0 a query sees the last `window` keys up to its own and the first `sinks`.  `q_lens`, `k_lens` int32 [B]: the queries and
    keys that each sequence has; rows beyond them, and rows that see no key, are zero.  What lies in keys beyond them does not matter, but
    infinities and NaN there make the call many times slower: clear padding that was never written.  scale None: 1 / sqrt(D)."""
    args = (q, k, v, q_lens, k_lens, 0.0 if scale is None else scale, window, sinks)
    out = _native.window_attention(*args)
    return _window(*args) if out is None else out


def _on_device(values, device, dtype=torch.int32) -> torch.Tensor:
    """Values of the host as a tensor on `device`, without a wait for its stream (a copy from pageable memory is one)."""
    t = torch.as_tensor(values, dtype=dtype)
    return t.pin_memory().to(device, non_blocking=True) if device.type == "cuda" else t


_WHOLE = "prompts are attended to as a whole: a sequence that brings tokens must hold no older ones"


class PagedKvCache:
    """The pages of a batch of sequences for every layer of a decoder, and the calls above on them.

    Page p of a sequence is the same page number in every layer; the pools, [pages, kv heads, page_size, head_dim] each, are allocated
    once.  Pages are handed out on the host: `grow` before the layers of a step, with the number of new tokens of each sequence
    (`grow_all`: one of each that goes on), then `append` and `attend` (or `attend_prompt`) once a layer.  Inside a captured CUDA graph
    only these two belong; `grow` outside it, and a graph that is replayed on a fixed table needs the pages of its whole run reserved
    in front (`reserve`).

    dtype bfloat16 or float16 as the tokens are, or float8_e4m3fn with `k_amax`, `v_amax`: per layer one value or one per kv head.
    `weights` True keeps the sums of attention weights by which `evict` chooses."""

    def __init__(self, layers: int, batch: int, n_kv: int, head_dim: int, pages: int, max_tokens: int, page_size: int = 16, dtype=torch.bfloat16,
                 k_amax=None, v_amax=None, weights: bool = False, device="cuda"):
        if page_size < 1 or pages < 1 or max_tokens < 1:
            raise ValueError("pages, their rows and the tokens of a sequence must be at least one")
        if dtype not in (torch.bfloat16, torch.float16, torch.float8_e4m3fn):
            raise ValueError(f"received pages of {dtype} type. Supported types: float16 | bfloat16 | float8_e4m3fn")
        if (dtype == torch.float8_e4m3fn) != (k_amax is not None) or (k_amax is None) != (v_amax is None):
            raise ValueError("FP8 pages need k_amax and v_amax of every layer, other pages take none")
        self.layers, self.batch, self.page_size, self.max_tokens = layers, batch, page_size, max_tokens
        self.n_kv, self.head_dim = n_kv, head_dim
        self.k_amax, self.v_amax = k_amax or [None] * layers, v_amax or [None] * layers
        shape = (pages, n_kv, page_size, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
        width = -(-max_tokens // page_size)
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.weights = [torch.zeros(batch, n_kv, max_tokens, device=device) for _ in range(layers)] if weights else [None] * layers
        self._free = list(range(pages - 1, -1, -1))
        self._pages: list = [[] for _ in range(batch)]     # of each sequence, in order
        self._tokens = [0] * batch
        self._released: set = set()
        self._padded = None
        self._new, self._cu, self._rows = [0] * batch, None, batch      # of the last `grow`: counts, their sums on the device, rows of an append

    def tokens(self) -> list:
        """Tokens of each sequence."""
        return list(self._tokens)

    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, tokens: list) -> None:
        """Pages for sequences of up to `tokens[b]` tokens."""
        if len(tokens) != self.batch or any(n > self.max_tokens for n in tokens):
            raise ValueError(f"expected {self.batch} counts of up to {self.max_tokens} tokens, got {tokens}")
        need = [max(0, -(-n // self.page_size) - len(p)) for n, p in zip(tokens, self._pages)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"{sum(need)} pages are needed and {len(self._free)} are free")
        rows, cols, vals = [], [], []
        for b, n in enumerate(need):
            for _ in range(n):
                rows.append(b), cols.append(len(self._pages[b])), vals.append(self._free.pop())
                self._pages[b].append(vals[-1])
        if vals:
            at = _on_device([rows, cols, vals], self.table.device)
            self.table[at[0], at[1]] = at[2]

    def _check_counts(self, new: list) -> None:
        if len(new) != self.batch or any(n < 0 for n in new):
            raise ValueError(f"expected {self.batch} counts of new tokens, got {new}")

    def grow(self, new: list) -> None:
        """Makes room for new[b] tokens of sequence b; the next `append` of every layer brings them."""
        self._check_counts(new)
        self.reserve([t + n for t, n in zip(self._tokens, new)])
        self._tokens = [t + n for t, n in zip(self._tokens, new)]
        self._released -= {b for b, n in enumerate(new) if n}
        self._new, self._rows = list(new), sum(new)
        if all(n == 1 for n in new):
            self._cu = None
            self.lens += 1
        else:
            counts = torch.tensor([0] + self._new, dtype=torch.int32)
            both = _on_device(torch.stack([counts.cumsum(0), counts]), self.lens.device)
            self._cu = both[0]
            self.lens += both[1, 1:]
        self._padded = self._padding()

    def _padding(self):
        """Of prompts of different lengths: (longest, lengths, place of each token among rows of that length); else None.  Made once for
        all layers, from what the host knows."""
        new = [n for n in self._new if n]
        if not new or min(new) == max(new) or self._new != [t if n else 0 for n, t in zip(self._new, self._tokens)]:
            return None
        counts = torch.tensor(new)
        first = counts.cumsum(0) - counts
        place = torch.arange(sum(new)) + torch.repeat_interleave(torch.arange(len(new)) * max(new) - first, counts)
        return max(new), _on_device(counts, self.lens.device), _on_device(place, self.lens.device, torch.int64)

    def grow_all(self) -> None:
        """Makes room for one new token of every sequence that has not been released.  `append` and `attend` take a row of each all the
        same: a released one's goes nowhere, and its result is zero."""
        new = [0 if b in self._released else 1 for b in range(self.batch)]
        self.grow(new)
        self._cu, self._rows = None, self.batch      # a sequence of no tokens has no place for a new one

    def check_prompt(self, new: list) -> None:
        """Raises where `attend_prompt` would after `grow(new)`."""
        self._check_counts(new)
        if any(n and t for n, t in zip(new, self._tokens)):
            raise ValueError(_WHOLE)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """K and V rows [tokens, kv heads, head_dim] of the tokens that `grow` made room for, sequence after sequence."""
        if k.shape[0] != self._rows or v.shape[0] != self._rows:
            raise ValueError(f"expected the rows of {self._rows} new tokens, got {k.shape[0]} and {v.shape[0]}")
        paged_append(k, v, self.k[layer], self.v[layer], self.table, self.lens, self._cu, k_amax=self.k_amax[layer], v_amax=self.v_amax[layer])

    def attend(self, layer: int, q: torch.Tensor, *, scale: float | None = None, window: int = 0, sinks: int = 0) -> torch.Tensor:
        """Attention of the newest token of every sequence: q [batch, query heads, head_dim]."""
        return paged_attention(q, self.k[layer], self.v[layer], self.table, self.lens, k_amax=self.k_amax[layer], v_amax=self.v_amax[layer],
                               weights=self.weights[layer], scale=scale, window=window, sinks=sinks)

    def attend_prompt(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None, window: int = 0,
                      sinks: int = 0) -> torch.Tensor:
        """Attention of the tokens of whole prompts over themselves: q, k, v [tokens, heads, head_dim], sequence after sequence ->
        [tokens, query heads, head_dim].  A sequence that brings tokens holds no older ones; one that brings none (a sequence that is
        generating beside it) takes no part."""
        if any(n and n != t for n, t in zip(self._new, self._tokens)):
            raise ValueError(_WHOLE)
        if q.shape[0] != sum(self._new):
            raise ValueError(f"expected the rows of {sum(self._new)} new tokens, got {q.shape[0]}")
        new = [n for n in self._new if n]
        if not new:
            return torch.empty_like(q)
        if self._padded is None:
            rows = lambda t: t.unflatten(0, (len(new), new[0])).transpose(1, 2)  # noqa: E731
            return window_attention(rows(q), rows(k), rows(v), scale=scale, window=window, sinks=sinks).transpose(1, 2).flatten(0, 1)
        most, lens, place = self._padded

        def rows(t):
            out = t.new_zeros(len(new) * most, *t.shape[1:])
            return out.index_copy_(0, place, t).unflatten(0, (len(new), most)).transpose(1, 2)

        out = window_attention(rows(q), rows(k), rows(v), scale=scale, window=window, sinks=sinks, q_lens=lens, k_lens=lens)
        return out.transpose(1, 2).flatten(0, 1).index_select(0, place)

    def evict(self, keep: int, recent: int = 0, sinks: int = 0) -> list:
        """Cuts every sequence to `keep` tokens per kv head, by the sums of attention weights of each layer, and frees the pages they
        were in, reserved ones among them.  Only `attend` adds to the sums: right behind a prompt all are equal, and beside the first
        `sinks` and the last `recent` the lowest tokens stay.  -> the kept tokens of every layer, int32 [batch, kv heads, keep]."""
        if self.weights[0] is None:
            raise ValueError("eviction goes by attention weights: the cache was made with weights=False")
        if min(keep, recent, sinks) < 0 or recent + sinks > keep or keep > self.max_tokens:
            raise ValueError(f"need recent + sinks <= keep <= {self.max_tokens} tokens, none negative, got {recent}, {sinks}, {keep}")
        width, need = -(-keep // self.page_size), [-(-min(keep, t) // self.page_size) for t in self._tokens]
        if sum(need) > len(self._free):
            raise RuntimeError(f"{sum(need)} pages are needed and {len(self._free)} are free")
        fresh = [[self._free.pop() for _ in range(n)] for n in need]
        try:
            out = _on_device([p + [-1] * (max(width, 1) - len(p)) for p in fresh], self.table.device)
            cut = [paged_evict(self.k[layer], self.v[layer], self.table, self.lens, self.weights[layer], out, keep=keep, recent=recent, sinks=sinks)
                   for layer in range(self.layers)]
        except BaseException:                    # nothing but rows of the fresh pages has been written yet
            self._free.extend(p for pages in reversed(fresh) for p in reversed(pages))
            raise
        kept = [which for which, _, _ in cut]
        for w, (_, lens, left) in zip(self.weights, cut):
            w.copy_(left)                        # in place, as the table and the lengths: a captured step reads them where they are
        self.lens.copy_(lens)
        self.table.fill_(-1)
        self.table[:, :width] = out[:, :width]
        for old in self._pages:
            self._free.extend(old)
        self._pages, self._tokens = fresh, [min(keep, t) for t in self._tokens]
        self._new = [0] * self.batch
        return kept

    def release(self, b: int) -> None:
        """Sequence b is done: its pages are free, and it is empty until `grow` brings it tokens again."""
        self._free.extend(self._pages[b])
        self._pages[b], self._tokens[b], self._new[b] = [], 0, 0
        self._released.add(b % self.batch)
        self.lens[b].zero_()
        self.table[b].fill_(-1)
        for w in self.weights:
            if w is not None:
                w[b].zero_()


class CachedDecoder:
    """A `DecoderStack` on one rank that generates: prompts and single tokens through its layers, with the attention of a
    `PagedKvCache` in the place of the stack's own (no position encoding, as in the stack).

        decoder = CachedDecoder(stack, cache, window=4096, sinks=4)
        decoder.prompt(h, [n0, n1, ..])      # h [n0 + n1 + .., hidden]: the prompts, one behind the other -> the same shape
        decoder.prompt(h, [0, n1, ..])       # sequences that go on bring none: a released one takes a new prompt
        decoder.step(h)                      # h [batch, hidden]: one token of every sequence that is not released -> the same shape
    """

    def __init__(self, stack, cache: PagedKvCache, window: int = 0, sinks: int = 0):
        cfg = stack.cfg
        if stack.world != 1:
            raise ValueError("the cached decoder runs on one rank")
        if (cache.layers, cache.n_kv, cache.head_dim) != (len(stack.layers), cfg.n_kv, cfg.head_dim):
            raise ValueError(f"cache of {cache.layers} layers, {cache.n_kv} kv heads of {cache.head_dim} for a stack of {len(stack.layers)}, "
                             f"{cfg.n_kv} of {cfg.head_dim}")
        if cache.k[0].dtype == torch.float16:
            raise ValueError("the stack's tokens are bfloat16: pages of that type or of float8_e4m3fn, not float16")
        self.stack, self.cache, self.window, self.sinks = stack, cache, window, sinks

    def _walk(self, h: torch.Tensor, attend) -> torch.Tensor:
        cfg, delta = self.stack.cfg, None
        for i, layer in enumerate(self.stack.layers):
            def core(qkv, i=i):
                heads = qkv.unflatten(1, (cfg.n_q + 2 * cfg.n_kv, cfg.head_dim))
                q, k, v = heads.split((cfg.n_q, cfg.n_kv, cfg.n_kv), dim=1)
                self.cache.append(i, k, v)
                return attend(i, q, k, v).flatten(1)

            h, delta = layer.forward(h, delta, core)
        return self.stack.backend.add(h, delta)

    # What is refused is refused before `grow`: later the cache counts tokens that no layer holds.
    def _check(self, h: torch.Tensor, rows: int) -> None:
        hidden = self.stack.cfg.hidden
        if h.dim() != 2 or tuple(h.shape) != (rows, hidden) or h.dtype != torch.bfloat16:
            raise ValueError(f"expected [{rows}, {hidden}] of bfloat16, got {tuple(h.shape)} of {h.dtype}")

    def prompt(self, h: torch.Tensor, lens: list) -> torch.Tensor:
        self._check(h, sum(lens))
        self.cache.check_prompt(lens)
        self.cache.grow(lens)
        return self._walk(h, lambda i, q, k, v: self.cache.attend_prompt(i, q, k, v, window=self.window, sinks=self.sinks))

    def step(self, h: torch.Tensor) -> torch.Tensor:
        self._check(h, self.cache.batch)
        self.cache.grow_all()
        return self._walk(h, lambda i, q, k, v: self.cache.attend(i, q, window=self.window, sinks=self.sinks))
