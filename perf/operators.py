"""What is timed of the key-value cache and its attention: the calls a decoder that generates text makes around its
quantized linears, over the range of sizes it makes them with.

    append    the K and V rows of new tokens go into the pages of the cache (8-bit pages: quantized under a calibrated range)
    decode    attention of one new token of every sequence over its pages, optionally with a sliding window whose first tokens
              (sinks) stay visible, optionally adding each key's attention weight to a running sum
    evict     the keys of the largest sums, the first and the latest ones stay: their rows move to fresh pages
    window    attention of a prompt, or of a chunk of one, with a sliding window and sinks

`run` computes them in plain torch, or through the package where `own` is true; `exact` restates them in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "fp16": 2, "fp8": 1}
_E4M3_MAX = 448.0


def listed():
    return [
        # one sequence of a chat, a few hundred tokens in: latency
        {"name": "decode_token", "kind": "decode", "b": 1, "hq": 32, "hkv": 8, "d": 128, "least": 411, "most": 411, "page": 16,
         "dtype": "bf16", "cache": "bf16", "window": 0, "sinks": 0, "weights": False},
        # a batch of a server, sequences of every age
        {"name": "decode_batch", "kind": "decode", "b": 64, "hq": 64, "hkv": 8, "d": 128, "least": 1, "most": 8190, "page": 16,
         "dtype": "bf16", "cache": "bf16", "window": 0, "sinks": 0, "weights": False},
        # a few sequences over long documents, 8-bit cache
        {"name": "decode_long_fp8", "kind": "decode", "b": 3, "hq": 64, "hkv": 8, "d": 128, "least": 60000, "most": 131071, "page": 64,
         "dtype": "bf16", "cache": "fp8", "window": 0, "sinks": 0, "weights": False},
        # small heads without groups under a sliding window with sinks, half precision
        {"name": "decode_window", "kind": "decode", "b": 32, "hq": 16, "hkv": 16, "d": 64, "least": 900, "most": 16000, "page": 32,
         "dtype": "fp16", "cache": "fp16", "window": 2048, "sinks": 4, "weights": False},
        # a step that keeps the sums by which keys are evicted later
        {"name": "decode_weights", "kind": "decode", "b": 8, "hq": 32, "hkv": 8, "d": 128, "least": 2000, "most": 8200, "page": 16,
         "dtype": "bf16", "cache": "bf16", "window": 0, "sinks": 0, "weights": True},
        # the rows of one decode step, straight from the QKV projection, into 8-bit pages
        {"name": "append_step_fp8", "kind": "append", "b": 64, "hq": 64, "hkv": 8, "d": 128, "new": 1, "least": 100, "most": 500, "page": 16,
         "dtype": "bf16", "cache": "fp8"},
        # the rows of a batch of prompts of different lengths
        {"name": "append_prompts", "kind": "append", "b": 9, "hq": 32, "hkv": 8, "d": 128, "new": 1850, "least": 1850, "most": 4000, "page": 16,
         "dtype": "bf16", "cache": "bf16"},
        # one long sequence cut to a quarter
        {"name": "evict_long", "kind": "evict", "b": 1, "hkv": 8, "d": 128, "least": 32000, "most": 32000, "page": 16, "cache": "bf16",
         "keep": 8192, "recent": 256, "sinks": 4},
        # a batch of sequences, some of them still within their budget
        {"name": "evict_batch_fp8", "kind": "evict", "b": 24, "hkv": 8, "d": 128, "least": 1500, "most": 6000, "page": 32, "cache": "fp8",
         "keep": 2048, "recent": 64, "sinks": 4},
        # the next few tokens of a prompt (a chunk that is checked or filled in) behind what is there already
        {"name": "window_chunk", "kind": "window", "b": 1, "hq": 32, "hkv": 8, "d": 128, "sq": 61, "sk": 1999, "window": 1024, "sinks": 4,
         "dtype": "bf16", "ragged": False},
        # a batch of ragged prompts, heads of 80, half precision
        {"name": "window_ragged", "kind": "window", "b": 8, "hq": 12, "hkv": 12, "d": 80, "sq": 1500, "sk": 1500, "window": 512, "sinks": 1,
         "dtype": "fp16", "ragged": True},
        # long prompts through a layer with grouped heads (the largest case)
        {"name": "window_prompt", "kind": "window", "b": 2, "hq": 32, "hkv": 8, "d": 128, "sq": 8192, "sk": 8192, "window": 4096, "sinks": 4,
         "dtype": "bf16", "ragged": False},
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "append", "evict", "window", "window"])
    hkv = rng.choice([1, 2, 4, 8, 12, 16])
    d = rng.choice([64, 64, 80, 96, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    cache = rng.choice([dtype, "fp8"])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    if kind == "decode":
        most = _log_int(rng, 64, 131072)
        return {"kind": kind, "b": _log_int(rng, 1, 256), "hq": hkv * rng.choice([1, 2, 4, 5, 8, 16]), "hkv": hkv, "d": d,
                "least": rng.choice([1, _log_int(rng, most // 16, most)]), "most": most, "page": page, "dtype": dtype, "cache": cache,
                "window": rng.choice([0, 0, _log_int(rng, 16, 8192)]), "sinks": rng.choice([0, 1, 4, 64]), "weights": rng.random() < 0.25}
    if kind == "append":
        new = rng.choice([1, _log_int(rng, 2, 4000)])
        most = new + _log_int(rng, 1, 2000)
        return {"kind": kind, "b": _log_int(rng, 1, 128), "hq": hkv * rng.choice([1, 4, 8]), "hkv": hkv, "d": d, "new": new, "least": new,
                "most": most, "page": page, "dtype": dtype, "cache": cache}
    if kind == "evict":
        most = _log_int(rng, 256, 65536)
        keep = _log_int(rng, most // 16, most)
        return {"kind": kind, "b": _log_int(rng, 1, 64), "hkv": hkv, "d": d, "least": rng.choice([1, _log_int(rng, most // 16, most)]), "most": most, "page": page,
                "cache": cache, "keep": keep, "recent": rng.randint(0, keep // 2), "sinks": rng.choice([0, 1, 4])}
    sq = _log_int(rng, 32, 8192)
    sk = sq + rng.choice([0, 0, _log_int(rng, 1, 8192)])
    return {"kind": kind, "b": _log_int(rng, 1, 16), "hq": hkv * rng.choice([1, 2, 4, 8]), "hkv": hkv, "d": d, "sq": sq, "sk": sk,
            "window": rng.choice([0, _log_int(rng, 16, 8192)]), "sinks": rng.choice([0, 1, 4, 130]), "dtype": dtype, "ragged": rng.random() < 0.3}


def _plain_elements(c):
    """About how many 32-bit values the plain form holds at once."""
    if c["kind"] == "decode":
        return c["b"] * c["most"] * (2 * c["hkv"] * c["d"] + 2 * c["hq"])
    if c["kind"] == "window":
        return 2 * c["b"] * c["hq"] * c["sq"] * c["sk"]
    if c["kind"] == "evict":
        return c["b"] * c["hkv"] * (8 * c["most"] + c["keep"] * c["d"])
    return c["b"] * c["new"] * (c["hq"] + 2 * c["hkv"]) * c["d"]


def draw(rng):
    cases = listed()
    cost = {key: max(work(c)[key] for c in cases) for key in ("bytes", "flops")}
    room = max(_plain_elements(c) for c in cases)
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= cost["bytes"] and w["flops"] <= cost["flops"] and _plain_elements(case) <= room:
            return case


# ----------------------------------------------------------------------------- sizes
def _lens(c):
    """The lengths of the sequences of a case: from `least` to `most`, in no order."""
    if c["b"] == 1:
        return [c["most"]]
    ranks = sorted(range(c["b"]), key=lambda i: (i * 0.6180339887) % 1.0)
    return [c["least"] + (c["most"] - c["least"]) * r // (c["b"] - 1) for r in ranks]


def _ragged(c):
    """(queries, keys) of each sequence of a window case."""
    if not c["ragged"]:
        return [c["sq"]] * c["b"], [c["sk"]] * c["b"]
    lens = [max(1, c["sq"] - c["sq"] * ((5 * i) % (c["b"] + 1)) // (c["b"] + 2)) for i in range(c["b"])]
    return lens, [n + c["sk"] - c["sq"] for n in lens]


def _new(c):
    """New tokens of each sequence of an append case."""
    if c["new"] == 1:
        return [1] * c["b"]
    return [max(1, c["new"] - c["new"] * ((3 * i) % (c["b"] + 1)) // (c["b"] + 1)) for i in range(c["b"])]


def _visible(n, window, sinks):
    """Keys that the last of n tokens sees."""
    return n if window <= 0 else min(n, window + min(sinks, max(0, n - window)))


def _visible_pairs(nq, nk, window, sinks):
    """The same summed over the last nq of nk tokens."""
    n = torch.arange(max(nk - nq, 0) + 1, nk + 1, dtype=torch.int64)
    if window > 0:
        n = torch.minimum(n, window + (n - window).clamp(0, sinks))
    return int(n.sum())


def work(case):
    c, kind = case, case["kind"]
    if kind == "window":
        nq, nk = _ragged(c)
        pairs = sum(_visible_pairs(a, b, c["window"], c["sinks"]) for a, b in zip(nq, nk))
        used = sum(min(b, a + c["window"] + c["sinks"]) if c["window"] > 0 else b for a, b in zip(nq, nk))
        size = _BYTES[c["dtype"]]
        return {"bytes": size * c["d"] * (sum(nq) + c["b"] * c["sq"]) * c["hq"] + 2 * size * c["d"] * c["hkv"] * used,
                "flops": 4 * c["d"] * c["hq"] * pairs}
    lens, size = _lens(c), _BYTES[c["cache"]]
    row = c["hkv"] * c["d"]
    if kind == "decode":
        seen = sum(_visible(n, c["window"], c["sinks"]) for n in lens)
        pages = sum(-(-n // c["page"]) for n in lens)
        return {"bytes": 2 * seen * row * size + 4 * c["b"] * c["hq"] * c["d"] + 4 * (pages + c["b"]) + (8 * seen * c["hkv"] if c["weights"] else 0),
                "flops": 4 * seen * c["hq"] * c["d"]}
    if kind == "append":
        new = sum(_new(c))
        return {"bytes": 2 * new * row * (_BYTES[c["dtype"]] + size) + 4 * new, "flops": 4 * new * row if c["cache"] == "fp8" else 0}
    kept = sum(min(n, c["keep"]) for n in lens)
    return {"bytes": 4 * kept * row * size + 4 * c["hkv"] * (sum(lens) + c["b"] * (c["most"] + c["keep"])), "flops": c["hkv"] * sum(lens)}


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _channels(g, heads, d):
    """Spread of a head's channels: a few are several times the others, as in trained decoders."""
    return torch.where(torch.rand(heads, 1, d, device="cuda", generator=g) < 0.02, 4.0, 1.0)


def _rows(g, c, tokens, dtype):
    """Q, K and V of `tokens` tokens as they lie in a QKV projection: [tokens, heads, d] views of one buffer."""
    d, hq, hkv = c["d"], c["hq"], c["hkv"]
    qkv = _randn(g, tokens, hq + 2 * hkv, d)
    qkv[:, hq:hq + hkv] *= _channels(g, hkv, d)[:, 0]
    qkv = qkv.to(dtype)
    return qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]


def _pool(g, c, pages, filled):
    """K and V pages [pages, heads, page, d] and the ranges they are held under (8-bit pages)."""
    dtype, shape = _DTYPES[c["cache"]], (pages, c["hkv"], c["page"], c["d"])
    if not filled:
        k, v = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
        amax = [torch.full((1,), a, device="cuda") for a in (20.0, 6.0)] if c["cache"] == "fp8" else [None, None]
        return k.to(dtype), v.to(dtype), amax
    got, amax = [], []
    for spread in (_channels(g, c["hkv"], c["d"]), 1.0):
        x = _randn(g, *shape) * spread
        amax.append(x.abs().amax().reshape(1) if c["cache"] == "fp8" else None)
        got.append((x / (amax[-1] / _E4M3_MAX) if c["cache"] == "fp8" else x).to(dtype))
        del x
    return got[0], got[1], amax


def _tables(g, c, lens, spare=0):
    """Block tables [b, pages of the longest] over a pool in which the sequences' pages lie in no order, and the pool's size;
    the last `spare` pages belong to nobody."""
    per = [-(-n // c["page"]) for n in lens]
    width, total = max(per), sum(per)
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None] < torch.tensor(per, device="cuda")[:, None]
    table[at] = order
    return table, total + spare


def prepare(case, seed):
    c, g, kind = case, _gen(seed), case["kind"]
    if kind == "window":
        dtype = _DTYPES[c["dtype"]]
        nq, nk = _ragged(c)
        q = _rows(g, c, c["b"] * c["sq"], dtype)[0].unflatten(0, (c["b"], c["sq"])).transpose(1, 2)
        k, v = (t.unflatten(0, (c["b"], c["sk"])).transpose(1, 2) for t in _rows(g, c, c["b"] * c["sk"], dtype)[1:])
        lens = [torch.tensor(n, dtype=torch.int32, device="cuda") if c["ragged"] else None for n in (nq, nk)]
        return {"kind": kind, "q": q, "k": k, "v": v, "q_lens": lens[0], "k_lens": lens[1], "window": c["window"], "sinks": c["sinks"]}
    lens = _lens(c)
    out_pages = -(-c["keep"] // c["page"]) * c["b"] if kind == "evict" else 0
    table, pages = _tables(g, c, lens, out_pages)
    k_pages, v_pages, amax = _pool(g, c, pages, kind != "append")
    s = {"kind": kind, "k_pages": k_pages, "v_pages": v_pages, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    if kind == "evict":
        s["out_table"] = torch.arange(pages - out_pages, pages, dtype=torch.int32, device="cuda").view(c["b"], -1)
        for t in (k_pages, v_pages):
            t[pages - out_pages:].view(torch.uint8).zero_()
        # sums of attention weights: most keys have little, some have been looked at again and again; quarters make equal ones
        w = (_randn(g, c["b"], c["hkv"], c["most"]) * 2.0).exp().mul(4).round().div(4)
        s["weights"] = w * (torch.arange(c["most"], device="cuda") < s["lens"][:, None, None])
        s.update(keep=c["keep"], recent=c["recent"], sinks=c["sinks"], first=pages - out_pages)
        return s
    s["k_amax"], s["v_amax"] = amax
    if kind == "append":
        new = _new(c)
        q, s["k"], s["v"] = _rows(g, c, sum(new), _DTYPES[c["dtype"]])
        s["cu_new"] = None if c["new"] == 1 else torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
        return s
    s["q"] = _rows(g, c, c["b"], _DTYPES[c["dtype"]])[0]
    s["weights"] = torch.rand(c["b"], c["hkv"], c["most"], device="cuda", generator=g) if c["weights"] else None
    s.update(window=c["window"], sinks=c["sinks"])
    return s


# ----------------------------------------------------------------------------- the package's operators
def _run_own(s):
    import tensorrt_b200 as b

    kind = s["kind"]
    if kind == "decode":
        out = b.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], k_amax=s["k_amax"], v_amax=s["v_amax"],
                                weights=s["weights"], window=s["window"], sinks=s["sinks"])
        return {"out": out, "weights": s["weights"]}
    if kind == "append":
        b.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu_new"], k_amax=s["k_amax"], v_amax=s["v_amax"])
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if kind == "evict":
        kept, lens, weights = b.paged_evict(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["weights"], s["out_table"], keep=s["keep"],
                                            recent=s["recent"], sinks=s["sinks"])
        return {"kept": kept, "lens": lens, "weights": weights, "k_pages": s["k_pages"][s["first"]:], "v_pages": s["v_pages"][s["first"]:]}
    return {"out": b.window_attention(s["q"], s["k"], s["v"], window=s["window"], sinks=s["sinks"], q_lens=s["q_lens"], k_lens=s["k_lens"])}


# ----------------------------------------------------------------------------- plain forms, 32 bits
def _raw(pages):
    """Pages whose elements can be gathered and written: 8-bit ones as bytes."""
    return pages.view(torch.uint8) if pages.element_size() == 1 else pages


def _scale(amax):
    s = amax / _E4M3_MAX
    return torch.where(s == 0, torch.ones_like(s), s)


def _gathered(pages, table, amax):
    """[b, heads, keys, d] in 32 bits: the pages of every sequence in order."""
    x = _raw(pages)[table.long()].view(pages.dtype).float()
    x = x.transpose(1, 2).flatten(2, 3)
    return x if amax is None else x.mul_(_scale(amax).view(-1, 1, 1))


def _masked_softmax(s, seen):
    """Softmax of s over the keys that are seen; zeros for a row that sees none.  Overwrites s."""
    s.masked_fill_(~seen, -math.inf)
    s -= s.amax(-1, keepdim=True).clamp_min(-3e38)
    s.exp_()
    total = s.sum(-1, keepdim=True)
    return s.div_(torch.where(total == 0, torch.ones_like(total), total))


def _plain_decode(s):
    q, hkv, d = s["q"], s["k_pages"].shape[1], s["q"].shape[2]
    k, v = _gathered(s["k_pages"], s["table"], s["k_amax"]), _gathered(s["v_pages"], s["table"], s["v_amax"])
    at, last = torch.arange(k.shape[2], device="cuda"), s["lens"][:, None] - 1
    seen = at <= last
    if s["window"] > 0:
        seen &= (at > last - s["window"]) | (at < s["sinks"])
    p = q.float().unflatten(1, (hkv, -1)) @ k.transpose(2, 3)
    p = _masked_softmax(p.mul_(1.0 / math.sqrt(d)), seen[:, None, None])
    out = (p @ v).flatten(1, 2).to(q.dtype)
    if s["weights"] is not None:
        s["weights"] += p.sum(2)[:, :, :s["weights"].shape[2]]
    return {"out": out, "weights": s["weights"]}


def _plain_append(s):
    page, tokens = s["k_pages"].shape[2], s["k"].shape[0]
    cu = torch.arange(len(s["lens"]) + 1, device="cuda", dtype=torch.int32) if s["cu_new"] is None else s["cu_new"]
    t = torch.arange(tokens, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(cu, t, right=True) - 1
    at = s["lens"][b] - cu[b + 1] + t
    where = (s["table"][b, at // page].long(), slice(None), (at % page).long())

    def put(pages, x, amax):
        if amax is not None:
            x = (x.float() / _scale(amax).view(-1, 1)).clamp(-_E4M3_MAX, _E4M3_MAX).to(pages.dtype).view(torch.uint8)
        _raw(pages)[where] = x

    put(s["k_pages"], s["k"], s["k_amax"])
    put(s["v_pages"], s["v"], s["v_amax"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_evict(s):
    w, lens, keep, page = s["weights"], s["lens"][:, None, None], s["keep"], s["k_pages"].shape[2]
    at = torch.arange(w.shape[2], device="cuda").expand_as(w)
    rank = torch.where(at >= lens, 0, torch.where((at < s["sinks"]) | (at >= lens - s["recent"]), 2, 1))
    order = torch.where(w.isnan(), -math.inf, w).sort(dim=2, descending=True, stable=True).indices
    order = order.gather(2, rank.gather(2, order).sort(dim=2, descending=True, stable=True).indices)
    count = lens.clamp(max=keep)
    j = torch.arange(keep, device="cuda")
    kept = torch.where(j < count, order[:, :, :keep], w.shape[2]).sort(dim=2).values
    valid = j < count
    at = torch.where(valid, kept, 0)
    new_w = torch.zeros_like(w)
    new_w[:, :, :keep] = torch.where(valid, w.gather(2, at), 0.0)
    b, h = torch.arange(w.shape[0], device="cuda")[:, None, None], torch.arange(w.shape[1], device="cuda")[:, None]
    src = (s["table"][b, at // page].long(), h, at % page)
    dst = (s["out_table"][b, j // page].long(), h, j % page)

    def move(pages):
        pages[dst] = torch.where(valid[..., None], pages[src], pages[dst])

    move(_raw(s["k_pages"]))
    move(_raw(s["v_pages"]))
    return {"kept": torch.where(valid, kept, -1).int(), "lens": count.view(-1).int(), "weights": new_w,
            "k_pages": s["k_pages"][s["first"]:], "v_pages": s["v_pages"][s["first"]:]}


def _plain_window(s):
    q, k, v = s["q"], s["k"], s["v"]
    (b, hq, sq, d), (_, hkv, sk, _) = q.shape, k.shape
    nq = torch.full((b,), sq, device="cuda") if s["q_lens"] is None else s["q_lens"]
    nk = torch.full((b,), sk, device="cuda") if s["k_lens"] is None else s["k_lens"]
    i, j = torch.arange(sq, device="cuda")[:, None], torch.arange(sk, device="cuda")
    at = i + (nk - nq)[:, None, None]
    seen = (j <= at) & (i < nq[:, None, None])
    if s["window"] > 0:
        seen &= (j > at - s["window"]) | (j < s["sinks"])
    p = q.float().unflatten(1, (hkv, -1)) @ k.float().transpose(2, 3)[:, :, None]
    p = _masked_softmax(p.mul_(1.0 / math.sqrt(d)), seen[:, None, None])
    return {"out": (p @ v.float()[:, :, None]).flatten(1, 2).to(q.dtype)}


def run(state):
    if own:
        return _run_own(state)
    return {"decode": _plain_decode, "append": _plain_append, "evict": _plain_evict, "window": _plain_window}[state["kind"]](state)


# ----------------------------------------------------------------------------- the definition, 64 bits
def _attend64(q, k, v, seen, d):
    """q [g, n, d], k and v [keys, d], seen [n, keys] or [keys]: (outputs, weights) of one head group."""
    x = (q @ k.T) / math.sqrt(d)
    x = x.masked_fill(~seen, -math.inf)
    p = torch.softmax(x, -1).nan_to_num(0.0)
    return p @ v, p


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "window":
        q, k, v = s["q"], s["k"], s["v"]
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        g, (nqs, nks) = q.shape[1] // k.shape[1], _ragged(case)
        for b, (nq, nk) in enumerate(zip(nqs, nks)):
            at, j = torch.arange(nk - nq, nk, device="cuda")[:, None], torch.arange(nk, device="cuda")
            seen = j <= at
            if s["window"] > 0:
                seen &= (j > at - s["window"]) | (j < s["sinks"])
            for h in range(q.shape[1]):
                out[b, h, :nq] = _attend64(q[b, h, :nq].double(), k[b, h // g, :nk].double(), v[b, h // g, :nk].double(), seen, case["d"])[0]
        return {"out": out}
    k_pages, v_pages, table, lens, page = s["k_pages"], s["v_pages"], s["table"], _lens(case), case["page"]
    if kind == "decode":
        scale = [1.0 if a is None else float(a) / _E4M3_MAX for a in (s["k_amax"], s["v_amax"])]
        if case["cache"] == "fp8":      # the scale itself is a 32-bit quotient
            scale = [float(torch.tensor(float(a), dtype=torch.float32) / _E4M3_MAX) for a in (s["k_amax"], s["v_amax"])]
        out, weights = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), s["weights"]
        weights = None if weights is None else weights.double()
        g = case["hq"] // case["hkv"]
        for b, n in enumerate(lens):
            rows = table[b, :-(-n // page)].long()
            last = n - 1
            at = torch.arange(n, device="cuda")
            seen = (at > last - s["window"]) | (at < s["sinks"]) if s["window"] > 0 else at >= 0
            for h in range(case["hkv"]):
                k, v = (_raw(t[:, h])[rows].view(t.dtype).double().flatten(0, 1)[:n] * f for t, f in zip((k_pages, v_pages), scale))
                o, p = _attend64(s["q"][b, h * g:(h + 1) * g].double(), k, v, seen, case["d"])
                out[b, h * g:(h + 1) * g] = o
                if weights is not None:
                    weights[b, h, :n] += p.sum(0)
        return {"out": out, "weights": weights}
    if kind == "append":
        got = []
        for pages, x, amax in ((k_pages, s["k"], s["k_amax"]), (v_pages, s["v"], s["v_amax"])):
            full = pages.double()
            x = x.double()
            if amax is not None:
                f = torch.tensor(float(amax), dtype=torch.float32) / _E4M3_MAX
                x = (x.float() / f.cuda()).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn).double()
            t = 0
            for b, (n, new) in enumerate(zip(lens, _new(case))):
                at = torch.arange(n - new, n, device="cuda")
                full[table[b].long()[at // page], :, at % page] = x[t:t + new]
                t += new
            got.append(full)
        return {"k_pages": got[0], "v_pages": got[1]}
    keep, recent, sinks = s["keep"], s["recent"], s["sinks"]
    kept = torch.full((case["b"], case["hkv"], keep), -1, dtype=torch.int32)
    weights = torch.zeros(s["weights"].shape, dtype=torch.float64)
    held = s["weights"].double().cpu()
    pages = [t[s["first"]:].double() for t in (k_pages, v_pages)]
    for b, n in enumerate(lens):
        m = min(n, keep)
        for h in range(case["hkv"]):
            w = held[b, h, :n].clone()
            w[:sinks] = math.inf
            w[max(0, n - recent):] = math.inf
            at = torch.sort(torch.sort(-w, stable=True).indices[:m]).values
            kept[b, h, :m] = at.int()
            weights[b, h, :m] = held[b, h, at]
            at, j = at.cuda(), torch.arange(m, device="cuda")
            for new, old in zip(pages, (k_pages, v_pages)):
                row = _raw(old)[table[b].long()[at // page], h, at % page].view(old.dtype).double()
                new[s["out_table"][b].long()[j // page] - s["first"], h, j % page] = row
    return {"kept": kept.cuda(), "lens": torch.tensor([min(n, keep) for n in lens], dtype=torch.int32, device="cuda"), "weights": weights.cuda(),
            "k_pages": pages[0], "v_pages": pages[1]}
