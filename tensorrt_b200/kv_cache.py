"""The paged key-value cache of a decoder that generates text, and the attention around it.

    paged_append      K and V rows of new tokens into their pages (FP8 E4M3 pages: quantized under a calibrated abs-max)
    paged_attention   one new token of every sequence over its pages
    paged_evict       the keys of the largest attention weights stay, their rows move to fresh pages
    window_attention  causal attention with a sliding window and sinks over contiguous K and V (prompts and their chunks)
    paged_copy        pages to other pages, in the pools of all layers at once
    shared_prefix_attention  paged_attention of a batch in which groups of sequences share the pages of a prefix (`SharedPrefix`)

Pages are tensors [pages, kv heads, rows, D] (any strides with D contiguous) of float16, bfloat16, float8_e4m3fn or uint8 (FP8
codes); token t of sequence b is row t % rows of page block_table[b, t // rows].  `lens` [B] counts the tokens of each sequence that
are in the cache, the newest included, in every call.  Everything is enqueued on the current stream of the tensors' device, nothing
synchronises (but the first call with a `SharedPrefix`, which waits for the copy of its plan), and the calls can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, _native
from .ops import load_ops
from .scores import TokenScores, token_log_probs

load_ops()
_ops = torch.ops.tensorrt
_append, _attention = _ops.b200_paged_append.default, _ops.b200_paged_attention.default
_evict, _window = _ops.b200_paged_evict.default, _ops.b200_window_attention.default
_copy, _shared = _ops.b200_paged_copy.default, _ops.b200_shared_prefix_attention.default


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


def paged_copy(k_pages, v_pages, src: list, dst: list, rows: list | None = None) -> None:
    """Copies page src[i] to page dst[i] in every pool: `k_pages` and `v_pages` a tensor each, or lists of as many (a layer's pools, or all
    layers').  rows[i]: the first rows of the page that are copied (None: all).  The numbers are the host's and travel with the launch.  No
    page may be written twice, nor be both read and written."""
    k, v = ([p] if isinstance(p, torch.Tensor) else list(p) for p in (k_pages, v_pages))
    args = (k, v, list(src), list(dst), None if rows is None else list(rows))
    if not _native.paged_copy(*args):
        _copy(*args)


class SharedPrefix:
    """Which sequences of a batch share a prefix: the sequences members[g] have their first tokens[g] tokens in the same pages, which are found
    through the line of the block table of the first of them.  It goes by sequences and stays valid as they grow.

    Groups of one sequence and prefixes of no token are left out: nothing is shared.  The first call of every pair of head counts makes a plan of the work
    on the host, outside a stream capture, and has it on the device before it returns, so that calls on any stream find it there.  `update` says anew who shares what,
    in place, so that a captured call goes by it; it takes up to `groups` groups of up to `largest` sequences (None: those given here).  A captured call reads the plan
    of this object: keep it as long as the graph."""

    def __init__(self, members: list, tokens: list, batch: int, device="cuda", groups: int | None = None, largest: int | None = None):
        if batch < 0 or batch > 65535:
            raise ValueError(f"need a batch of up to 65535 sequences, got {batch}")
        kept = self._kept(members, tokens)
        self.batch = batch
        self.groups = len(kept) if groups is None else groups
        self.largest = max([len(m) for m, _ in kept], default=0) if largest is None else largest
        if not 0 <= self.groups <= batch or not 0 <= self.largest <= batch:
            raise ValueError(f"{self.groups} groups of up to {self.largest} sequences are not in a batch of {batch}")
        if self.largest < 2:                                                # nobody to share with
            self.groups = 0
        self.device, self._plans = torch.device(device), {}
        self.update(members, tokens)

    @staticmethod
    def _kept(members: list, tokens: list) -> list:
        if len(members) != len(tokens):
            raise ValueError(f"expected as many prefixes ({len(tokens)}) as groups ({len(members)})")
        if any(t < 0 or t > 0x7FFFFFFF for t in tokens):
            raise ValueError(f"a prefix has from 0 to {0x7FFFFFFF} tokens, got {tokens}")
        return [(list(m), t) for m, t in zip(members, tokens) if len(m) > 1 and t > 0]

    def update(self, members: list, tokens: list) -> None:
        """Who shares what from now on, as given to the constructor; outside a capture, whose replays go by the plan as it is then.  Plans that calls
        have made are written on the current stream, as a block table would be: calls and replays on other streams are ordered with that by the caller."""
        if self._plans and self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the plan of a shared prefix is made on the host: update it outside the capture")
        kept = self._kept(members, tokens)
        if len(kept) > self.groups or any(len(m) > self.largest for m, _ in kept):
            raise ValueError(f"made for {self.groups} groups of up to {self.largest} sequences, got groups of {[len(m) for m, _ in kept]}")
        flat = [b for m, _ in kept for b in m]
        seen = set(flat)
        if len(seen) != len(flat) or any(b < 0 or b >= self.batch for b in seen):
            raise ValueError(f"a sequence of a batch of {self.batch} is in one group at most, got {members}")
        ends = [0]
        for m, _ in kept:
            ends.append(ends[-1] + len(m))
        ends += ends[-1:] * (self.groups - len(kept))                       # empty groups
        shared = [t for _, t in kept] + [0] * (self.groups - len(kept))
        self.tokens = max(shared, default=0)                                # of the longest prefix
        self._lists = [(ctypes.c_int32 * max(len(v), 1))(*v) for v in (flat, ends, shared)]
        for heads, plan in self._plans.items() if self.groups else ():     # of no groups: empty, whatever they are
            host = self._made(*heads)
            plan.copy_(host.pin_memory() if plan.is_cuda else host, non_blocking=True)
            if plan.is_cuda:
                plan.record_stream(torch.cuda.current_stream(plan.device))

    def _made(self, n_q: int, n_kv: int) -> torch.Tensor:
        lib, sizes = _lib.load(), (self.batch, n_q, n_kv, self.groups, self.largest)
        plan = torch.empty(lib.b200q_shared_prefix_plan_values(*sizes), dtype=torch.int32)
        _lib.check(lib.b200q_shared_prefix_plan(*self._lists, *sizes, plan.data_ptr()), "b200q_shared_prefix_plan")
        return plan

    def plan(self, n_q: int, n_kv: int) -> torch.Tensor:
        """The plan for this many query and kv heads, on the device."""
        plan = self._plans.get((n_q, n_kv))
        if plan is None:
            if self.groups == 0:
                plan = torch.empty(0, dtype=torch.int32, device=self.device)
            else:
                if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("the plan of a shared prefix is made on the host: call once with these heads before the capture")
                with torch.inference_mode(False):           # `update` may be called outside the mode that this call is in
                    plan = self._made(n_q, n_kv)
                    if self.device.type == "cuda":          # on a stream of its own, waited for: the next call may be on any
                        plan = _native.uploaded(plan, torch.cuda.current_device() if self.device.index is None else self.device.index)
            self._plans[n_q, n_kv] = plan
        return plan


def shared_prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                            prefix: SharedPrefix, *, k_amax: torch.Tensor | None = None, v_amax: torch.Tensor | None = None,
                            scale: float | None = None) -> torch.Tensor:
    """`paged_attention` of a batch in which groups of sequences share a prefix: its keys are attended to by all rows of a group at once, and read
    once for each 128 or 256 of them, as the plan finds shorter; the keys behind it through each sequence's own line of the table.  A sequence with fewer tokens than
    its group's prefix is attended to through its own line alone."""
    if prefix.batch != q.shape[0]:
        raise ValueError(f"the prefixes are those of a batch of {prefix.batch}, q is {tuple(q.shape)}")
    if q.dim() != 3 or k_pages.dim() != 4 or k_pages.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k_pages.shape[1]:
        raise ValueError(f"expected q [batch, query heads, D] and pages [pages, kv heads, rows, D], the kv heads dividing the query heads, got {tuple(q.shape)} "
                         f"and {tuple(k_pages.shape)}")
    if prefix.tokens > block_table.shape[-1] * k_pages.shape[2]:
        raise ValueError(f"prefixes of up to {prefix.tokens} tokens do not fit the table's lines of {block_table.shape[-1]} pages of {k_pages.shape[2]} rows")
    scale, plan = 0.0 if scale is None else scale, prefix.plan(q.shape[1], k_pages.shape[1])
    out = _native.shared_prefix_attention(q, k_pages, v_pages, block_table, lens, plan, k_amax, v_amax, scale, prefix.groups, prefix.largest)
    return _shared(q, k_pages, v_pages, block_table, lens, plan, prefix.groups, prefix.largest, k_amax, v_amax, scale) if out is None else out


def _on_device(values, device, dtype=torch.int32) -> torch.Tensor:
    """Values of the host as a tensor on `device`, without a wait for its stream (a copy from pageable memory is one)."""
    t = torch.as_tensor(values, dtype=dtype)
    return t.pin_memory().to(device, non_blocking=True) if device.type == "cuda" else t


def _common(a: list, b: list) -> int:
    """Length of the longest common beginning, by comparisons of whole slices."""
    low, high = 0, min(len(a), len(b))
    while low < high:
        mid = (low + high + 1) // 2
        low, high = (mid, high) if a[low:mid] == b[low:mid] else (low, mid - 1)
    return low


# Keys, times kv heads, that a batch's single-token attention has to read once instead of once more for each who shares them, before a cache takes the
# kernels for shared prefixes.  Three launches, and the parts that they pass on, cost what reading so much costs paged_attention: for up to eight sequences; half
# as much again for more of them, but for one group where paged_attention has 1024 sequences x kv heads to begin and end, which costs it as much; twice that
# with 8-bit pages, whose rows and queries have to be converted first (three times from eight query heads of a kv head on).  What two sequences share counts half,
# and with 8-bit pages, where they do not gain, nothing.  Measured, paged / shared, in us at multiples of 2^17 keys x kv heads:
#   8 kv heads x 4 of 128, 16 bits     4 sequences: 1 24.6 / 23.0, 2 32.9 / 27.7      16: 1 22.5 / 23.5, 1.5 24.6 / 24.2, 2 26.6 / 25.6
#                                      64: 1 24.6 / 27.7, 1.5 26.7 / 27.6, 2 30.1 / 27.6, 4 41.0 / 28.3      256: 0.5 41.0 / 37.9, 1 41.0 / 37.9
#   2 x 4 of 64, 16 bits               4: 1 22.6 / 21.5      16: 1 20.5 / 17.4      64: 1 18.5 / 21.3, 1.5 20.5 / 21.5, 3 26.6 / 21.5
#   8 x 4 of 128, 8 bits               2: 1 30.3 / 29.7, 6 80.0 / 79.8      4: 1 24.6 / 25.6, 2 32.6 / 27.7      16: 1 22.6 / 23.7, 2 28.7 / 30.6, 3 33.1 / 31.5
#                                      64: 1 23.0 / 35.8, 2 31.0 / 36.1, 3 36.4 / 36.1, 4 41.0 / 35.9      256: 1 41.2 / 46.0, 2 46.8 / 45.2
#   8 x 8 of 128, 8 bits               64: 2 32.9 / 40.0, 4 43.0 / 43.9      256: 2 49.9 / 59.0, 3 55.3 / 60.2, 4 59.4 / 60.6
#   1 x 4 of 64, 8 bits                2: 3 38.9 / 46.1, 6 59.0 / 69.8
#   8 x 4 of 128, groups, 16 bits      16 of 4: 1 28.7 / 29.7, 2 37.0 / 34.3      64 of 4: 1 43.0 / 46.3, 2 53.7 / 52.2      32 of 8: 1 41.0 / 39.9
#                                      2 of 2: 2 45.4 / 44.7      16 of 2: 1 32.9 / 37.4, 2 52.8 / 50.2, 5 121 / 89.1      256 of 2: 1 74.0 / 94.3, 5 144 / 132
#   8 x 4 of 128, groups, 8 bits       16 of 4: 2 35.5 / 35.9, 3 41.9 / 37.9      64 of 4: 3 57.6 / 57.6      64 of 2: 2 49.2 / 72.8, 5 82.9 / 101
# Pages that are no multiple of eight rows are copied by threads, which takes what five (8-bit pages: some seventeen) readings by paged_attention take: there, groups
# of fewer than 16 (64) sequences count next to nothing, and larger ones of 8-bit pages half.  Pages of 7 rows, 8 kv heads x 4 of 128:
#   16 bits                            4: 4 51.0 / 64.3, 12 112 / 142      16: 2 28.7 / 29.2, 4 41.0 / 33.8      64: 4 43.0 / 33.8      256: 2 47.1 / 44.8
#   8 bits                             4: 4 47.5 / 140, 12 105 / 364       16: 4 41.0 / 48.2, 40 246 / 271       64: 4 43.2 / 44.1, 12 86.1 / 54.5      256: 4 57.6 / 54.2
_SHARED_KEYS = 1 << 17

_WHOLE = "prompts are attended to as a whole: a sequence that brings tokens must hold no older ones"


class PagedKvCache:
    """The pages of a batch of sequences for every layer of a decoder, and the calls above on them.

    Page p of a sequence is the same page number in every layer; the pools, [pages, kv heads, page_size, head_dim] each, are allocated
    once.  Pages are handed out on the host: `grow` before the layers of a step, with the number of new tokens of each sequence
    (`grow_all`: one of each that goes on), then `append` and `attend` (or `attend_prompt`) once a layer.  Inside a captured CUDA graph
    only these two belong; `grow` outside it, and a graph that is replayed on a fixed table needs the pages of its whole run reserved
    in front (`reserve`).

    dtype bfloat16 or float16 as the tokens are, or float8_e4m3fn with `k_amax`, `v_amax`: per layer one value or one per kv head.
    `weights` True keeps the sums of attention weights by which `evict` chooses.

    `fork` continues a sequence several times: the continuations share its pages, `attend` attends to what a group of them shares at once, and
    a page that is not full is copied when the first of those that share it grows.  `truncate` takes tokens back, `compact` moves the pages in
    use to the front of the pools, `resize` changes how many there are."""

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
        self._uses = [0] * pages                           # sequences that a page is part of
        self._prefix, self._shares, self._saved, self._n_q = None, False, (0, 0, 0), 0      # `_saved`: keys that are read once, sequences and groups that share them
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
        """Pages for sequences of up to `tokens[b]` tokens.  A sequence that is to grow and whose last page is not full gets that page for
        itself: a copy, where others share it."""
        if len(tokens) != self.batch or any(n > self.max_tokens for n in tokens):
            raise ValueError(f"expected {self.batch} counts of up to {self.max_tokens} tokens, got {tokens}")
        need = [max(0, -(-n // self.page_size) - len(p)) for n, p in zip(tokens, self._pages)]
        own, left = [], {}                                 # sequences that need a copy; of a page, those that still share it
        for b, (n, t) in enumerate(zip(tokens, self._tokens)):
            if n > t and t % self.page_size:
                last = self._pages[b][t // self.page_size]
                left.setdefault(last, self._uses[last])
                if left[last] > 1:                         # the last one of them keeps the page
                    left[last] -= 1
                    own.append(b)
        if sum(need) + len(own) > len(self._free):
            raise RuntimeError(f"{sum(need) + len(own)} pages are needed and {len(self._free)} are free")
        rows, cols, vals = [], [], []
        if own:
            at = [self._tokens[b] // self.page_size for b in own]
            fresh = self._free[-len(own):][::-1]
            paged_copy(self.k, self.v, [self._pages[b][i] for b, i in zip(own, at)], fresh, [self._tokens[b] % self.page_size for b in own])
            del self._free[-len(own):]
            for b, i, page in zip(own, at, fresh):
                self._uses[self._pages[b][i]] -= 1
                self._uses[page], self._pages[b][i] = 1, page
            rows, cols, vals = list(own), at, list(fresh)
        for b, n in enumerate(need):
            for _ in range(n):
                rows.append(b), cols.append(len(self._pages[b])), vals.append(self._free.pop())
                self._pages[b].append(vals[-1])
                self._uses[vals[-1]] = 1
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
        """Attention of the newest token of every sequence: q [batch, query heads, head_dim].  Without a window and without weights, what groups
        of forked sequences share is attended to once for all of a group, where that is much.  A captured step stays with the kernels that were
        taken when it was captured, and is right behind any later call."""
        n_q = q.shape[1] if q.dim() == 3 else 0
        if n_q != self._n_q:
            self._n_q = n_q
            self._shares = self._worth()
        if self.weights[layer] is None and window <= 0 and self._shares:
            return shared_prefix_attention(q, self.k[layer], self.v[layer], self.table, self.lens, self._prefix, k_amax=self.k_amax[layer],
                                           v_amax=self.v_amax[layer], scale=scale)
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
        for p in (p for pages in fresh for p in pages):
            self._uses[p] = 1
        for old in self._pages:
            self._give_back(old)
        self._pages, self._tokens = fresh, [min(keep, t) for t in self._tokens]
        self._new, self._rows = [0] * self.batch, 0      # `grow` comes before the next `append`
        self._share()
        return kept

    def _give_back(self, pages: list) -> None:
        for p in pages:
            self._uses[p] -= 1
            if self._uses[p] == 0:
                self._free.append(p)

    def release(self, b: int) -> None:
        """Sequence b is done: its pages are free (those that others share once these are done too), and it is empty until `grow` brings it
        tokens again."""
        shared = any(self._uses[p] > 1 for p in self._pages[b][:1])
        self._give_back(self._pages[b])
        self._pages[b], self._tokens[b], self._new[b] = [], 0, 0
        self._released.add(b % self.batch)
        self.lens[b].zero_()
        self.table[b].fill_(-1)
        for w in self.weights:
            if w is not None:
                w[b].zero_()
        if shared:
            self._share()

    def fork(self, parents: list) -> None:
        """Sequence b goes on from where sequence parents[b] is (b itself: from where it was), for all at once: [0] * batch continues the first one
        `batch` times, and a step of a beam search is `fork` of the beams that were chosen.  Nothing is copied but what `evict` goes by: the
        tokens stay in the pages that they are in.  What sequence b held before is gone, as after `release`; pages reserved for the parent
        stay the parent's."""
        if len(parents) != self.batch or any(p < 0 or p >= self.batch for p in parents):
            raise ValueError(f"expected {self.batch} sequences to go on from, got {parents}")
        moved = [b for b, p in enumerate(parents) if p != b]
        if not moved:
            return
        held = {b: self._pages[parents[b]][:-(-self._tokens[parents[b]] // self.page_size)] for b in moved}
        same = {b: _common(pages, self._pages[b]) for b, pages in held.items()}      # what a beam has in common with the one that it follows
        for b, pages in held.items():
            for p in pages[same[b]:]:
                self._uses[p] += 1
        for b in moved:
            self._give_back(self._pages[b][same[b]:])
        self._released = {b for b, p in enumerate(parents) if p in self._released}
        self._tokens, self._new, self._rows = [self._tokens[p] for p in parents], [0] * self.batch, 0
        for b, pages in held.items():
            self._pages[b] = pages
        width = self.table.shape[1]
        both = _on_device([parents, [len(held[b]) if b in held else width for b in range(self.batch)]], self.table.device, torch.int64)
        line = self.table.index_select(0, both[0])
        self.table.copy_(line.masked_fill_(torch.arange(width, device=line.device) >= both[1][:, None], -1))
        self.lens.copy_(self.lens.index_select(0, both[0]))
        for w in self.weights:
            if w is not None:
                w.copy_(w.index_select(0, both[0]))
        self._share()

    def truncate(self, tokens: list) -> None:
        """Cuts every sequence to its first tokens[b] tokens (those that a verification turned down go, say); the pages behind them are free, reserved
        ones among them."""
        if len(tokens) != self.batch or any(n < 0 or n > t for n, t in zip(tokens, self._tokens)):
            raise ValueError(f"expected {self.batch} counts of up to {self._tokens} tokens, got {tokens}")
        keep = [-(-n // self.page_size) for n in tokens]
        both = _on_device([list(tokens), keep], self.table.device)
        for b, n in enumerate(keep):
            self._give_back(self._pages[b][n:])
            del self._pages[b][n:]
        self._tokens, self._new, self._rows = list(tokens), [0] * self.batch, 0
        self.table.masked_fill_(torch.arange(self.table.shape[1], device=self.table.device) >= both[1][:, None], -1)
        self.lens.copy_(both[0])
        for w in self.weights:
            if w is not None:
                w.masked_fill_(torch.arange(w.shape[2], device=w.device) >= both[0][:, None, None], 0.0)
        self._share()

    def compact(self) -> int:
        """Moves the pages in use to the front of the pools, shared ones once, and returns how many they are."""
        used = sum(1 for n in self._uses if n)
        src = [p for p in range(used, len(self._uses)) if self._uses[p]]
        dst = [p for p in range(used) if not self._uses[p]]
        if src:
            paged_copy(self.k, self.v, src, dst)
            to = dict(zip(src, dst))
            self._pages = [[to.get(p, p) for p in pages] for pages in self._pages]
            for a, b in to.items():
                self._uses[b], self._uses[a] = self._uses[a], 0
            place = list(range(len(self._uses)))
            for a, b in to.items():
                place[a] = b
            place = _on_device(place, self.table.device)
            self.table.copy_(torch.where(self.table < 0, self.table, place[self.table.clamp_min(0).long()]))
        self._free = list(range(len(self._uses) - 1, used - 1, -1))
        return used

    def resize(self, pages: int) -> None:
        """Pools of `pages` pages, at least those in use, in the place of the old ones, one pool after the other: `k` and `v` are other tensors then, and captured
        steps are to be captured again.  Where memory runs out on the way this raises, and the cache has the smaller of the two numbers of pages."""
        used = sum(1 for n in self._uses if n)
        if pages < max(used, 1):
            raise ValueError(f"{used} pages are in use, {pages} are too few")
        self.compact()

        def have(n):
            self._uses = self._uses[:used] + [0] * (n - used)
            self._free = list(range(n - 1, used - 1, -1))

        least = min(pages, len(self._uses))
        have(least)
        try:
            for pools in (self.k, self.v):
                for i, old in enumerate(pools):
                    new = torch.zeros((pages, *old.shape[1:]), dtype=old.dtype, device=old.device)
                    new.view(torch.uint8)[:used] = old.view(torch.uint8)[:used]
                    pools[i] = new
                    del old, new
        except BaseException:
            for pools in (self.k, self.v):
                pools[:] = [p[:least] for p in pools]
            raise
        have(pages)

    def _counts(self, n: int) -> float:
        """How much of what a group of n sequences reads once counts."""
        codes = self.k[0].element_size() == 1
        if self.page_size % 8:
            return (1 / 2 if n >= 64 else 1 / 64) if codes else (1 if n >= 16 else 1 / 32)
        return 1 if n > 2 else (0 if codes else 1 / 2)

    def _worth(self) -> bool:
        keys, n, groups = self._saved
        many, codes = n > 8 and (groups > 1 or n * self.n_kv < 1024), self.k[0].element_size() == 1
        return keys >= _SHARED_KEYS * (1.5 if many else 1) * ((3 if self._n_q >= 8 * self.n_kv else 2) if codes else 1)

    def _share(self) -> None:
        """Finds who shares what, behind each call that changes it: a captured step reads the plan where it is, as it does the table."""
        first: dict = {}
        for b, pages in enumerate(self._pages):
            if self._tokens[b] >= self.page_size and self._uses[pages[0]] > 1:
                first.setdefault(pages[0], []).append(b)
        members = [m for m in first.values() if len(m) > 1]
        # pages that all of a group have in common and that are full
        shared = [self.page_size * min(min(_common(self._pages[m[0]], self._pages[b]), self._tokens[b] // self.page_size) for b in m) for m in members]
        self._saved = self.n_kv * sum((len(m) - 1) * t * self._counts(len(m)) for m, t in zip(members, shared)), sum(len(m) for m in members), len(members)
        self._shares = self._worth()
        if self._prefix is None and members:
            self._prefix = SharedPrefix([], [], self.batch, self.table.device, groups=self.batch // 2, largest=self.batch)
        if self._prefix is not None:
            self._prefix.update(members, shared)
            if self._n_q:                        # the first step behind a fork may be captured
                self._prefix.plan(self._n_q, self.n_kv)


class CachedDecoder:
    """A `DecoderStack` on one rank that generates: prompts and single tokens through its layers, with the attention of a
    `PagedKvCache` in the place of the stack's own (no position encoding, as in the stack).

        decoder = CachedDecoder(stack, cache, window=4096, sinks=4)
        decoder.prompt(h, [n0, n1, ..])      # h [n0 + n1 + .., hidden]: the prompts, one behind the other -> the same shape
        decoder.prompt(h, [0, n1, ..])       # sequences that go on bring none: a released one takes a new prompt
        decoder.step(h)                      # h [batch, hidden]: one token of every sequence that is not released -> the same shape
        decoder.score(h, head, top=4)        # what ranks the continuations: log probabilities, entropy, the most likely tokens
        cache.fork([0, 0, 1, 1])             # and those that are chosen go on
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

    def score(self, h: torch.Tensor, head, tokens: torch.Tensor | None = None, *, top: int = 0, scale: float = 1.0) -> TokenScores:
        """`token_log_probs` of the logits that `head` (an `Fp8Linear`, `Nvfp4Linear` or any other module) makes of h [rows, hidden]."""
        return token_log_probs(head(h), tokens, top=top, scale=scale)
