"""What is timed of several continuations of one prompt over the paged key-value cache: n samples, or the beams of a search.

    copy      pages of every layer's pools are copied to others: the half-filled page of a sequence that is continued twice, a pool
              whose pages move together
    prefix    attention of one new token of every sequence, where groups of sequences share the pages of a long prefix: the keys
              of the prefix are attended to by all of a group at once
    scores    log probability of the token that was taken, entropy and the most likely tokens, from a step's logits

`run` computes them in plain torch, or through the package where `own` is true; `exact` restates them in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp8": 1, "fp32": 4}
_E4M3_MAX = 448.0


def listed():
    return [
        # one sequence is continued a second time: its last page, two layers (latency)
        {"name": "copy_fork_one", "kind": "copy", "layers": 2, "hkv": 8, "d": 128, "page": 16, "cache": "bf16", "pages": 64, "sources": 1,
         "fan": 1, "partial": True, "rows_first": False},
        # a step of a beam search: the last pages of 16 sequences, three more continuations of each, in 32 layers
        {"name": "copy_fork_batch", "kind": "copy", "layers": 32, "hkv": 8, "d": 128, "page": 16, "cache": "bf16", "pages": 256, "sources": 16,
         "fan": 3, "partial": True, "rows_first": False},
        # whole 8-bit pages move to the front of a pool that is stored rows first
        {"name": "copy_compact_fp8", "kind": "copy", "layers": 4, "hkv": 8, "d": 128, "page": 64, "cache": "fp8", "pages": 1000, "sources": 400,
         "fan": 1, "partial": False, "rows_first": True},
        # four samples of a prompt of some hundred tokens (latency)
        {"name": "prefix_few", "kind": "prefix", "groups": 1, "n": 4, "hq": 32, "hkv": 8, "d": 128, "least": 500, "most": 500, "own": 30,
         "page": 16, "dtype": "bf16", "cache": "bf16", "mixed": False},
        # 64 samples of one long prompt: as many rows as a matrix product takes
        {"name": "prefix_samples", "kind": "prefix", "groups": 1, "n": 64, "hq": 64, "hkv": 8, "d": 128, "least": 8192, "most": 8192, "own": 200,
         "page": 16, "dtype": "bf16", "cache": "bf16", "mixed": False},
        # beams of several requests, prompts and groups of different sizes, dealt out over the batch
        {"name": "prefix_beams", "kind": "prefix", "groups": 9, "n": 8, "hq": 32, "hkv": 8, "d": 128, "least": 700, "most": 5000, "own": 400,
         "page": 16, "dtype": "fp16", "cache": "fp16", "mixed": True},
        # 16 questions to one long document, 8-bit cache (the largest case)
        {"name": "prefix_document_fp8", "kind": "prefix", "groups": 1, "n": 16, "hq": 64, "hkv": 8, "d": 128, "least": 100000, "most": 100000,
         "own": 900, "page": 64, "dtype": "bf16", "cache": "fp8", "mixed": False},
        # small heads without groups, a system prompt in front of a hundred conversations
        {"name": "prefix_heads_80", "kind": "prefix", "groups": 1, "n": 100, "hq": 12, "hkv": 12, "d": 80, "least": 1333, "most": 1333, "own": 300,
         "page": 24, "dtype": "fp16", "cache": "fp16", "mixed": False},
        # the beams of one request (latency)
        {"name": "scores_beams", "kind": "scores", "rows": 3, "vocabulary": 32000, "dtype": "bf16", "top": 6, "masked": False, "scale": 1.0},
        # a step of a server that returns alternatives
        {"name": "scores_step", "kind": "scores", "rows": 64, "vocabulary": 128000, "dtype": "bf16", "top": 20, "masked": False, "scale": 1.0},
        # the tokens of a prompt scored, rows that begin at any address
        {"name": "scores_prompt", "kind": "scores", "rows": 2000, "vocabulary": 50001, "dtype": "bf16", "top": 0, "masked": False, "scale": 1.0},
        # 32-bit logits under a grammar that leaves few tokens, at a temperature
        {"name": "scores_grammar", "kind": "scores", "rows": 200, "vocabulary": 100003, "dtype": "fp32", "top": 8, "masked": True, "scale": 1.25},
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    kind = rng.choice(["copy", "prefix", "prefix", "scores"])
    hkv = rng.choice([1, 2, 4, 8, 12])
    d = rng.choice([64, 64, 80, 96, 128, 128])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    cache = rng.choice([dtype, dtype, "fp8"])
    if kind == "copy":
        sources = _log_int(rng, 1, 1000)
        fan = rng.choice([1, 1, 2, 3, 7])
        return {"kind": kind, "layers": _log_int(rng, 1, 32), "hkv": hkv, "d": d, "page": page, "cache": cache,
                "pages": sources * (1 + fan) + _log_int(rng, 1, 300), "sources": sources, "fan": fan, "partial": rng.random() < 0.5,
                "rows_first": rng.random() < 0.4}
    if kind == "prefix":
        most = _log_int(rng, 30, 100000)
        return {"kind": kind, "groups": _log_int(rng, 1, 16), "n": _log_int(rng, 2, 100), "hq": hkv * rng.choice([1, 2, 4, 5, 8]), "hkv": hkv,
                "d": d, "least": rng.choice([most, _log_int(rng, max(1, most // 8), most)]), "most": most, "own": _log_int(rng, 1, 1000),
                "page": page, "dtype": dtype, "cache": cache, "mixed": rng.random() < 0.5}
    return {"kind": kind, "rows": _log_int(rng, 1, 2000), "vocabulary": _log_int(rng, 500, 260000), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
            "top": rng.choice([0, 1, 5, 8, 20, 50]), "masked": rng.random() < 0.25, "scale": rng.choice([1.0, 1.0, 0.5, 1.4])}


def _plain_bytes(c):
    """About how many bytes a case's state and the plain form take."""
    if c["kind"] == "copy":
        return 2 * c["layers"] * c["pages"] * c["hkv"] * c["page"] * c["d"] * _BYTES[c["cache"]]
    if c["kind"] == "prefix":
        return 4 * c["groups"] * c["n"] * (c["most"] + c["own"]) * (4 * c["hkv"] * c["d"] + 3 * c["hq"])
    return 30 * c["rows"] * c["vocabulary"]


def draw(rng):
    cases = listed()
    cost = {key: max(work(c)[key] for c in cases) for key in ("bytes", "flops")}
    room = {kind: max(_plain_bytes(c) for c in cases if c["kind"] == kind) for kind in ("copy", "prefix", "scores")}
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= cost["bytes"] and w["flops"] <= cost["flops"] and _plain_bytes(case) <= room[case["kind"]]:
            return case


# ----------------------------------------------------------------------------- sizes
def _pairs(c):
    """(source, destination, rows) of the pages that are copied: numbers of sources and of free pages, which `prepare` scatters."""
    n = c["sources"] * c["fan"]
    rows = [1 + (i * 7) % c["page"] if c["partial"] else c["page"] for i in range(c["sources"])]
    return [(i % c["sources"], c["sources"] + i, rows[i % c["sources"]]) for i in range(n)]


def _groups(c):
    """(tokens of the prefix, tokens of each sequence behind it) of every group."""
    got = []
    for i in range(c["groups"]):
        n = max(1, c["n"] - c["n"] * ((3 * i) % c["groups"]) // c["groups"])
        tokens = c["least"] if c["groups"] == 1 else c["least"] + (c["most"] - c["least"]) * ((5 * i) % c["groups"]) // (c["groups"] - 1)
        got.append((tokens - tokens % c["page"], [tokens % c["page"] + 1 + (c["own"] - 1) * ((7 * j) % n) // n for j in range(n)]))
    return got


def work(case):
    c = case
    if c["kind"] == "copy":
        pairs = _pairs(c)                                      # a page that is copied several times is read once
        rows = sum(r for _, _, r in pairs) + sum(r for _, _, r in pairs[:c["sources"]])
        return {"bytes": 2 * c["layers"] * rows * c["hkv"] * c["d"] * _BYTES[c["cache"]], "flops": 0}
    if c["kind"] == "prefix":
        groups = _groups(c)
        held = sum(t + sum(tail) for t, tail in groups)
        seen = sum(t * len(tail) + sum(tail) for t, tail in groups)
        b = sum(len(tail) for _, tail in groups)
        return {"bytes": 2 * held * c["hkv"] * c["d"] * _BYTES[c["cache"]] + 4 * b * c["hq"] * c["d"], "flops": 4 * seen * c["hq"] * c["d"]}
    return {"bytes": c["rows"] * (c["vocabulary"] * _BYTES[c["dtype"]] + 12 + 8 * c["top"]), "flops": 6 * c["rows"] * c["vocabulary"]}


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _raw(pages):
    """Pages whose elements can be gathered and written: 8-bit ones as bytes."""
    return pages.view(torch.uint8) if pages.element_size() == 1 else pages


def _pool(g, c, pages, rows_first=False):
    """Pages [pages, heads, page, d], a few channels of each head larger than the others, and their range (8-bit pages)."""
    x = _randn(g, pages, c["hkv"], c["page"], c["d"])
    x *= torch.where(torch.rand(c["hkv"], 1, c["d"], device="cuda", generator=g) < 0.02, 4.0, 1.0)
    amax = x.abs().amax().reshape(1) if c["cache"] == "fp8" else None
    x = (x if amax is None else x / (amax / _E4M3_MAX)).to(_DTYPES[c["cache"]])
    if rows_first:
        x = _raw(x).transpose(1, 2).contiguous().transpose(1, 2).view(x.dtype)
    return x, amax


def prepare(case, seed):
    c, g, kind = case, _gen(seed), case["kind"]
    if kind == "copy":
        at = torch.randperm(c["pages"], device="cuda", generator=g).tolist()
        src, dst, rows = zip(*[(at[a], at[b], n) for a, b, n in _pairs(c)])
        pools = [_pool(g, c, c["pages"], c["rows_first"])[0] for _ in range(2 * c["layers"])]
        return {"kind": kind, "k": pools[::2], "v": pools[1::2], "src": list(src), "dst": list(dst), "rows": list(rows) if c["partial"] else None}
    if kind == "scores":
        n, size = c["rows"], c["vocabulary"]
        x = _randn(g, n, size) * (1.0 + 2.0 * torch.rand(n, 1, device="cuda", generator=g))
        x += torch.where(torch.rand(n, size, device="cuda", generator=g) < 20 / size, 12.0, 0.0)      # what the model thinks likely
        if c["masked"]:
            allowed = torch.rand(n, size, device="cuda", generator=g) < 0.02
            allowed[:, ::997] = True
            x.masked_fill_(~allowed, -math.inf)
        # the token that was taken: of every second row the most likely one, of the others any that may follow
        any_token = torch.rand(n, size, device="cuda", generator=g).masked_fill_(x == -math.inf, -1.0).argmax(1)
        tokens = torch.where(torch.arange(n, device="cuda") % 2 == 0, x.argmax(1), any_token)
        return {"kind": kind, "logits": x.to(_DTYPES[c["dtype"]]), "tokens": tokens, "top": c["top"], "scale": c["scale"]}
    groups, page = _groups(c), c["page"]
    b = sum(len(tail) for _, tail in groups)
    places = list(range(b))                                    # of the batch, group after group
    if c["mixed"]:
        places.sort(key=lambda i: (i * 0.6180339887) % 1.0)
    pages = sum(t // page + sum(-(-n // page) for n in tail) for t, tail in groups)
    width = max(t // page + -(-max(tail) // page) for t, tail in groups)
    numbers = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).cpu()
    table, lens = torch.full((b, width), -1, dtype=torch.int32), [0] * b
    members, shared, used, at = [], [], 0, 0
    for t, tail in groups:
        prefix = numbers[used:used + t // page]
        used += t // page
        for n in tail:
            line = places[at]
            need = -(-n // page)
            table[line, :t // page] = prefix
            table[line, t // page:t // page + need] = numbers[used:used + need]
            lens[line] = t + n
            used, at = used + need, at + 1
        members.append(sorted(places[at - len(tail):at]))
        shared.append(t)
    s = {"kind": kind, "table": table.cuda(), "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    s["k_pages"], s["k_amax"] = _pool(g, c, pages)
    s["v_pages"], s["v_amax"] = _pool(g, c, pages)
    s["q"] = _randn(g, b, c["hq"] + 2 * c["hkv"], c["d"]).to(_DTYPES[c["dtype"]])[:, :c["hq"]]      # as it lies in a QKV projection
    if own:
        import tensorrt_b200

        s["prefix"] = tensorrt_b200.SharedPrefix(members, shared, batch=b)
    return s


# ----------------------------------------------------------------------------- the package's operators
def _run_own(s):
    import tensorrt_b200 as b

    if s["kind"] == "copy":
        b.paged_copy(s["k"], s["v"], s["src"], s["dst"], s["rows"])
        return {"k": s["k"], "v": s["v"]}
    if s["kind"] == "prefix":
        return {"out": b.shared_prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["prefix"], k_amax=s["k_amax"],
                                                 v_amax=s["v_amax"])}
    log_probs, entropy, top_log_probs, top_tokens = b.token_log_probs(s["logits"], s["tokens"], top=s["top"], scale=s["scale"])
    out = {"log_probs": log_probs, "entropy": entropy}
    return {**out, "top_log_probs": top_log_probs, "top_tokens": top_tokens} if s["top"] else out


# ----------------------------------------------------------------------------- plain forms, 32 bits
def _plain_copy(s):
    src, dst = (torch.tensor(t, device="cuda") for t in (s["src"], s["dst"]))
    for pool in s["k"] + s["v"]:
        pool = _raw(pool)
        if s["rows"] is None:
            pool[dst] = pool[src]
        else:
            copied = torch.arange(pool.shape[2], device="cuda") < torch.tensor(s["rows"], device="cuda")[:, None]
            pool[dst] = torch.where(copied[:, None, :, None], pool[src], pool[dst])
    return {"k": s["k"], "v": s["v"]}


def _scale(amax):
    s = amax / _E4M3_MAX
    return torch.where(s == 0, torch.ones_like(s), s)


def _gathered(pages, table, amax):
    """[b, heads, keys, d] in 32 bits: the pages of every sequence in order."""
    x = _raw(pages)[table.clamp_min(0).long()].view(pages.dtype).float()
    x = x.transpose(1, 2).flatten(2, 3)
    return x if amax is None else x.mul_(_scale(amax))


def _plain_prefix(s):
    """Every sequence over all of its own pages: what it shares with others changes nothing but the time."""
    q, hkv, d = s["q"], s["k_pages"].shape[1], s["q"].shape[2]
    k = _gathered(s["k_pages"], s["table"], s["k_amax"])
    x = (q.float().unflatten(1, (hkv, -1)) @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(d))
    x.masked_fill_(torch.arange(k.shape[2], device="cuda") >= s["lens"][:, None, None, None], -math.inf)
    del k
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    x /= x.sum(-1, keepdim=True)
    v = _gathered(s["v_pages"], s["table"], s["v_amax"])
    return {"out": (x @ v).flatten(1, 2).to(q.dtype)}


def _plain_scores(s):
    x = s["logits"].float()
    z = (x - x.amax(1, keepdim=True)) * s["scale"]
    e = z.exp()
    total = e.sum(1)
    lse = total.log()
    z = z.masked_fill(e == 0, 0.0)                       # 0 * -inf: a term without weight
    out = {"log_probs": (x.gather(1, s["tokens"][:, None])[:, 0] - x.amax(1)) * s["scale"] - lse, "entropy": lse - (e * z).sum(1) / total}
    if s["top"]:
        values, at = x.sort(dim=1, descending=True, stable=True)
        out["top_log_probs"] = (values[:, :s["top"]] - values[:, :1]) * s["scale"] - lse[:, None]
        out["top_tokens"] = at[:, :s["top"]].int()
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"copy": _plain_copy, "prefix": _plain_prefix, "scores": _plain_scores}[state["kind"]](state)


# ----------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "copy":
        out, copied = {}, s["rows"] or [case["page"]] * len(s["src"])
        for name in ("k", "v"):
            out[name] = [pool.double() for pool in s[name]]
            for n in set(copied):                              # pages of which n rows are copied
                a, b = (torch.tensor([p for p, m in zip(t, copied) if m == n], device="cuda") for t in (s["src"], s["dst"]))
                for pool in out[name]:
                    pool[b, :, :n] = pool[a, :, :n]
        return out
    if kind == "scores":
        x = s["logits"].double() * s["scale"]
        p = torch.log_softmax(x, 1)
        out = {"log_probs": p[torch.arange(case["rows"], device="cuda"), s["tokens"]], "entropy": -(p.exp() * p.clamp_min(-1e300)).sum(1)}
        if s["top"]:
            out["top_tokens"] = torch.sort(-s["logits"].double(), dim=1, stable=True).indices[:, :s["top"]].int()
            out["top_log_probs"] = p.gather(1, out["top_tokens"].long())
            out = {key: out[key] for key in ("log_probs", "entropy", "top_log_probs", "top_tokens")}
        return out
    page, g = case["page"], case["hq"] // case["hkv"]
    # the scale of 8-bit pages is a 32-bit quotient
    scale = [1.0 if a is None else float(a.cpu() / torch.tensor(_E4M3_MAX)) for a in (s["k_amax"], s["v_amax"])]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, :-(-n // page)].long()
        for h in range(case["hkv"]):
            k, v = (_raw(t[:, h])[pages].view(t.dtype).double().flatten(0, 1)[:n] * f for t, f in zip((s["k_pages"], s["v_pages"]), scale))
            heads = slice(h * g, (h + 1) * g)
            out[b, heads] = torch.softmax((s["q"][b, heads].double() @ k.T) / math.sqrt(case["d"]), -1) @ v
    return {"out": out}
