"""The paged key-value cache on the device: append, attention of one new token, eviction, against 64-bit restatements.

Bounds, from the arithmetic: a result is rounded once to its type (relative u = 2^-8 for bf16, 2^-11 for fp16); the tensor cores take P
rounded to 16 bits, at most u of every term of sum P |V|; exponentials, logits and sums are 32-bit, together below 2^-13 of
it for the logits here (up to some tens, head dimensions up to 128).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E4M3 = torch.float8_e4m3fn


def raw(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def pool(g, pages, heads, rows, d, dtype, layout="hnd"):
    """K and V pages and their ranges; `nhd`: stored [pages, rows, heads, D]."""
    got, amax = [], []
    for spread in (1.5, 1.0):
        x = torch.randn(pages, heads, rows, d, device="cuda", generator=g) * spread
        a = x.abs().amax().reshape(1)
        x = (x / (a / 448)).to(dtype) if dtype == E4M3 else x.to(dtype)
        if layout == "nhd":
            r = raw(x).transpose(1, 2).contiguous().transpose(1, 2)
            x = r.view(E4M3) if dtype == E4M3 else r
        got.append(x)
        amax.append(a if dtype == E4M3 else None)
    return got[0], got[1], amax[0], amax[1]


def table_of(g, lens, rows, width=None):
    per = [-(-max(n, 0) // rows) for n in lens]
    width = max(per + [1]) if width is None else width
    order = torch.randperm(sum(per) + 1, generator=g, device="cuda").to(torch.int32)
    t = torch.full((len(lens), width), -7, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(per):
        n = min(n, width)
        t[b, :n] = order[at:at + n]
        at += n
    return t, sum(per) + 1


def seen_keys(n, window, sinks):
    at = torch.arange(n, device="cuda")
    return at if window <= 0 else at[(at > n - 1 - window) | (at < sinks)]


def attention_ref(q, kp, vp, table, lens, ka, va, window, sinks, scale=None):
    """(out, sum P |V|, weights of every token) in 64 bits."""
    b, hq, d = q.shape
    heads, rows, pages = kp.shape[1], kp.shape[2], kp.shape[0]
    g = hq // heads
    out, mass = torch.zeros(b, hq, d, dtype=torch.float64, device="cuda"), torch.zeros(b, hq, d, dtype=torch.float64, device="cuda")
    most = table.shape[1] * rows
    weights = torch.zeros(b, heads, most, dtype=torch.float64, device="cuda")

    def dequant(pages_, amax, h):
        x = pages_.double()
        if amax is None:
            return x
        s = (amax.float() / 448)
        s = torch.where(s == 0, torch.ones_like(s), s).double()
        return x * (s[h] if s.numel() > 1 else s)

    for i in range(b):
        n = min(max(int(lens[i]), 0), most)
        at = seen_keys(n, window, sinks)
        page = table[i].long()[at // rows]
        ok = (page >= 0) & (page < pages)
        at, page = at[ok], page[ok]
        for h in range(heads):
            k = dequant(raw(kp)[page, h, at % rows].view(kp.dtype), ka, h)
            v = dequant(raw(vp)[page, h, at % rows].view(vp.dtype), va, h)
            s = q[i, h * g:(h + 1) * g].double() @ k.T * (1 / math.sqrt(d) if scale is None else scale)
            p = torch.softmax(s, -1) if len(at) else s
            out[i, h * g:(h + 1) * g] = p @ v
            mass[i, h * g:(h + 1) * g] = p @ v.abs()
            weights[i, h, at] = p.sum(0)
    return out, mass, weights


def check_out(out, ref, mass):
    u = U[out.dtype]
    tol = u * ref.abs() + (u + 2.0 ** -13) * mass + 1e-30
    off = (out.double() - ref).abs()
    assert torch.isfinite(out.float()).all()
    assert (off <= tol).all(), (off / tol).max().item()


CASES = [
    # lens, heads, group, D, rows, token type, page type, window, sinks, layout
    ([1], 1, 1, 64, 16, torch.bfloat16, torch.bfloat16, 0, 0, "hnd"),
    ([0, 1, 2, 15, 16, 17, 63, 64, 65, 129], 2, 4, 128, 16, torch.bfloat16, torch.bfloat16, 0, 0, "hnd"),
    ([0, 1, 2, 15, 16, 17, 63, 64, 65, 129], 2, 4, 128, 16, torch.float16, torch.float16, 0, 0, "nhd"),
    ([0, 1, 31, 32, 33, 700, 1025], 2, 8, 128, 64, torch.bfloat16, E4M3, 0, 0, "hnd"),
    ([5, 333, 1000], 3, 1, 80, 24, torch.float16, E4M3, 0, 0, "nhd"),
    ([5, 333, 1000], 3, 5, 96, 5, torch.bfloat16, torch.bfloat16, 0, 0, "nhd"),
    ([77, 0, 500], 1, 16, 16, 1, torch.float16, torch.float16, 0, 0, "hnd"),
    ([77, 900, 500], 1, 20, 48, 7, torch.bfloat16, E4M3, 0, 0, "hnd"),
    ([400, 1500], 1, 64, 128, 32, torch.bfloat16, torch.bfloat16, 0, 0, "hnd"),
    ([1, 4, 5, 99, 100, 101, 104, 105, 1000], 2, 4, 64, 16, torch.bfloat16, torch.bfloat16, 100, 4, "hnd"),
    ([1, 4, 5, 99, 100, 101, 104, 105, 1000], 2, 4, 64, 16, torch.float16, E4M3, 100, 0, "nhd"),
    ([300, 1000], 2, 2, 112, 16, torch.float16, torch.float16, 1, 0, "hnd"),
    ([300, 1000], 2, 2, 128, 16, torch.float16, torch.float16, 16, 200, "hnd"),
    ([20000, 3, 9000], 2, 4, 128, 16, torch.bfloat16, torch.bfloat16, 0, 0, "hnd"),
    ([20000, 3, 9000], 2, 8, 64, 128, torch.bfloat16, E4M3, 0, 0, "hnd"),
    (list(range(0, 300)), 1, 2, 64, 16, torch.bfloat16, torch.bfloat16, 0, 0, "hnd"),
    ([7] * 1500, 1, 1, 32, 8, torch.float16, torch.float16, 0, 0, "hnd"),
]


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"n{max(c[0])}x{len(c[0])}_h{c[1]}x{c[2]}_d{c[3]}_p{c[4]}_{str(c[6])[6:]}_w{c[7]}")
def test_attention_of_one_token(b200, case, weighted):
    lens, heads, group, d, rows, dt, pt, window, sinks, layout = case
    g = torch.Generator(device="cuda").manual_seed(len(lens) * 7 + d)
    table, pages = table_of(g, lens, rows)
    kp, vp, ka, va = pool(g, pages, heads, rows, d, pt, layout)
    # nothing that is not attended to may matter: rows behind the last token, pages of nobody, keys between sinks and window
    used = torch.zeros(pages, rows, dtype=torch.bool, device="cuda")
    for i, n in enumerate(lens):
        at = seen_keys(n, window, sinks)
        used[table[i].long()[at // rows], at % rows] = True
    for t in (kp, vp):
        r = raw(t)
        r[(~used)[:, None].expand(pages, heads, rows)] = 0x7F if t.element_size() == 1 else float("nan")
    qkv = torch.randn(len(lens), heads * group + 3, d, device="cuda", generator=g).to(dt)
    q = qkv[:, 1:1 + heads * group]
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    before = torch.rand(len(lens), heads, table.shape[1] * rows, device="cuda", generator=g) if weighted else None
    w = None if before is None else before.clone()
    out = b200.paged_attention(q, kp, vp, table, n, k_amax=ka, v_amax=va, weights=w, window=window, sinks=sinks)
    ref, mass, gained = attention_ref(q, kp, vp, table, lens, ka, va, window, sinks)
    assert out.shape == q.shape and out.dtype == dt
    check_out(out, ref, mass)
    if weighted:
        off = (w.double() - (before.double() + gained)).abs()
        assert (off <= 2.0 ** -12 * gained + 2.0 ** -22 * (before + gained)).all(), off.max().item()
    again = b200.paged_attention(q, kp, vp, table, n, k_amax=ka, v_amax=va, window=window, sinks=sinks)
    assert torch.equal(out, again)                      # the same bits on each call, with and without weights


def test_ranges_per_head_and_zero_range(b200):
    g = torch.Generator(device="cuda").manual_seed(3)
    lens, heads, rows, d = [50, 333], 3, 16, 64
    table, pages = table_of(g, lens, rows)
    kp, vp, _, _ = pool(g, pages, heads, rows, d, E4M3)
    ka, va = torch.tensor([3.0, 0.0, 9.0], device="cuda"), torch.tensor([0.5, 7.0, 0.0], device="cuda")
    q = torch.randn(2, 6, d, device="cuda", generator=g).bfloat16() * 0.01
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref, mass, _ = attention_ref(q, kp, vp, table, lens, ka, va, 0, 0, scale=0.5)
    for pages_k, pages_v in ((kp, vp), (kp.view(torch.uint8), vp.view(torch.uint8))):
        check_out(b200.paged_attention(q, pages_k, pages_v, table, n, k_amax=ka, v_amax=va, scale=0.5), ref, mass)


@pytest.mark.parametrize("pt", [torch.float16, torch.bfloat16, E4M3])
def test_queries_of_any_size(b200, pt):
    """Queries far from one and a head of zeros: the products of 8-bit pages must not leave the range of the type that they are
    multiplied in."""
    g = torch.Generator(device="cuda").manual_seed(4)
    dt = torch.float16 if pt == torch.float16 else torch.bfloat16
    lens, rows, d = [200, 31], 16, 128
    table, pages = table_of(g, lens, rows)
    kp, vp, ka, va = pool(g, pages, 1, rows, d, pt)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for size in (1e-6, 1e4) if dt == torch.float16 else (1e-30, 1e20):
        q = (torch.randn(2, 4, d, device="cuda", generator=g) * size).to(dt)
        q[0, 1] = 0
        scale = 0.1 / size
        ref, mass, _ = attention_ref(q, kp, vp, table, lens, ka, va, 0, 0, scale=float(torch.tensor(scale, dtype=torch.float32)))
        check_out(b200.paged_attention(q, kp, vp, table, n, k_amax=ka, v_amax=va, scale=scale), ref, mass)


def test_infinite_and_nan_keys_that_are_seen(b200):
    """-inf products give a weight of zero, a NaN among the keys that are seen gives NaN, and other heads do not notice."""
    lens, heads, rows, d = [100], 2, 16, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    table, pages = table_of(g, lens, rows)
    kp, vp, _, _ = pool(g, pages, heads, rows, d, torch.bfloat16)
    q = torch.rand(1, 2 * heads, d, device="cuda", generator=g).bfloat16() + 0.5
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    where = (int(table[0, 2]), 0, 5)
    kp[where] = -float("inf")
    ref, mass, _ = attention_ref(q, kp, vp, table, lens, None, None, 0, 0)
    check_out(b200.paged_attention(q, kp, vp, table, n), ref, mass)
    vp[where] = float("nan")
    out = b200.paged_attention(q, kp, vp, table, n)
    assert out[0, :2].isnan().all() and torch.isfinite(out[0, 2:].float()).all()
    kp[:, 1] = -float("inf")                             # every key of the other head: 0 / 0, as a softmax gives
    assert b200.paged_attention(q, kp, vp, table, n)[0, 2:].isnan().all()


def test_tables_and_lengths_that_name_less_than_they_say(b200):
    g = torch.Generator(device="cuda").manual_seed(6)
    lens, rows, d = [100, 90, 60, 70], 16, 64
    table, pages = table_of(g, lens, rows)
    kp, vp, _, _ = pool(g, pages, 2, rows, d, torch.bfloat16)
    q = torch.randn(4, 4, d, device="cuda", generator=g).bfloat16()
    table[0, 3] = -1
    table[0, 5] = pages
    table[1, 0] = 0x7FFFFFFF
    table[3] = -1                                        # no row of this sequence is there
    claimed = [100, 5000, -3, 70]                        # beyond the table, negative
    n = torch.tensor(claimed, dtype=torch.int32, device="cuda")
    out = b200.paged_attention(q, kp, vp, table, n)
    ref, mass, _ = attention_ref(q, kp, vp, table, claimed, None, None, 0, 0)
    check_out(out, ref, mass)
    assert not out[2:].any()


def test_pools_beyond_32_bit_offsets(b200):
    rows, d, heads = 16, 128, 8
    pages = (5 << 30) // (rows * d * heads)
    kp = torch.empty(pages, heads, rows, d, dtype=E4M3, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(7)
    lens = [40]
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device="cuda")
    a = torch.tensor([4.0], device="cuda")
    k, v = (torch.randn(40, heads, d, device="cuda", generator=g).bfloat16() for _ in range(2))
    vp = torch.empty_like(kp)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    b200.paged_append(k, v, kp, vp, table, n, cu, k_amax=a, v_amax=a)
    q = torch.randn(1, heads, d, device="cuda", generator=g).bfloat16()
    ref, mass, _ = attention_ref(q, kp, vp, table, lens, a, a, 0, 0)
    assert (raw(kp)[pages - 1] != 0).any()
    check_out(b200.paged_attention(q, kp, vp, table, n, k_amax=a, v_amax=a), ref, mass)
    w = torch.rand(1, heads, 48, device="cuda", generator=g)
    fresh = torch.tensor([[pages // 2, pages - 3]], dtype=torch.int32, device="cuda")
    kept, m, _ = b200.paged_evict(kp, vp, table, n, w, fresh, keep=20)
    assert m.tolist() == [20]
    ref, mass, _ = attention_ref(q[:, :1], kp[:, :1], vp[:, :1], fresh, [20], a, a, 0, 0)
    check_out(b200.paged_attention(q, kp, vp, fresh, m, k_amax=a, v_amax=a)[:, :1], ref, mass)
    rows_of = raw(kp)[table[0].long()[kept[0, 5].long() // rows], 5, kept[0, 5].long() % rows]
    assert torch.equal(raw(kp)[fresh[0].long()[torch.arange(20, device="cuda") // rows], 5, torch.arange(20, device="cuda") % rows], rows_of)


def test_other_streams_and_graphs(b200):
    """Calls on a stream of its own, and a captured step replayed on changed inputs."""
    g = torch.Generator(device="cuda").manual_seed(8)
    lens, rows, d = [513, 2000, 77], 16, 128
    table, pages = table_of(g, lens, rows)
    kp, vp, _, _ = pool(g, pages, 2, rows, d, torch.bfloat16)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(3, 8, d, device="cuda", generator=g).bfloat16()
    k, v = (torch.randn(3, 2, d, device="cuda", generator=g).bfloat16() for _ in range(2))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        on_stream = b200.paged_attention(q, kp, vp, table, n)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(on_stream, b200.paged_attention(q, kp, vp, table, n))
    w = torch.zeros(3, 2, table.shape[1] * rows, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b200.paged_append(k, v, kp, vp, table, n)
        out = b200.paged_attention(q, kp, vp, table, n, weights=w)
    for _ in range(3):
        k.normal_(generator=g), v.normal_(generator=g), q.normal_(generator=g), w.zero_()
        graph.replay()
        ref, mass, gained = attention_ref(q, kp, vp, table, lens, None, None, 0, 0)
        check_out(out, ref, mass)
        assert (w.double() - gained).abs().max() <= 2.0 ** -11
        last = n.long() - 1
        assert torch.equal(kp[table[torch.arange(3), last // rows].long(), :, last % rows], k)


@pytest.mark.parametrize("tiles,heads,group,d,pt", [([16], 1, 8, 128, torch.bfloat16), ([17], 1, 1, 64, torch.bfloat16), ([25, 18], 1, 16, 80, E4M3),
                                                    ([128], 1, 4, 128, E4M3), ([129], 1, 3, 128, torch.bfloat16), ([130, 1, 140], 1, 9, 64, torch.bfloat16),
                                                    ([1600], 1, 2, 128, torch.bfloat16), ([700, 3, 500], 2, 5, 64, E4M3)])
def test_attention_joined_from_many_parts(b200, tiles, heads, group, d, pt):
    """Sequences whose keys many CTAs share: the parts are joined at once or in two steps, some of them of no key, and twice the same bits."""
    g = torch.Generator(device="cuda").manual_seed(sum(tiles))
    rows, lens = 32, [64 * t - 5 for t in tiles]
    table, pages = table_of(g, lens, rows)
    kp, vp, ka, va = pool(g, pages, heads, rows, d, pt)
    table[:, 6:10] = -1                                   # two tiles and two halves without a page
    table[0, 20:32] = -1
    q = torch.randn(len(lens), heads * group, d, device="cuda", generator=g).bfloat16()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    w = torch.zeros(len(lens), heads, table.shape[1] * rows, device="cuda")
    out = b200.paged_attention(q, kp, vp, table, n, k_amax=ka, v_amax=va, weights=w)
    ref, mass, gained = attention_ref(q, kp, vp, table, lens, ka, va, 0, 0)
    check_out(out, ref, mass)
    assert (w.double() - gained).abs().max() <= 2.0 ** -11
    for _ in range(5):
        again = b200.paged_attention(q, kp, vp, table, n, k_amax=ka, v_amax=va)
        assert torch.equal(out.view(torch.int16), again.view(torch.int16))


# ----------------------------------------------------------------------------- append
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("heads,d,rows,new,layout", [(1, 16, 1, None, "hnd"), (8, 128, 16, None, "hnd"), (3, 80, 7, [5, 0, 40, 1], "nhd"),
                                                     (2, 64, 16, [300, 17, 16], "hnd"), (12, 96, 24, [1, 1, 999], "nhd")])
def test_append(b200, dt, codes, heads, d, rows, new, layout):
    import oracle as o

    g = torch.Generator(device="cuda").manual_seed(heads * d)
    counts = [1] * 5 if new is None else new
    lens = [c + 13 * i for i, c in enumerate(counts)]
    table, pages = table_of(g, lens, rows)
    kp, vp, _, _ = pool(g, pages, heads, rows, d, E4M3 if codes else dt, layout)
    tokens = sum(counts)
    qkv = torch.randn(tokens, 3 * heads, d, device="cuda", generator=g).to(dt)
    k, v = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]
    k[-1, 0, :4] = torch.tensor([float("inf"), -float("inf"), 0.0, -0.0])
    amax = [torch.rand(heads, device="cuda", generator=g) + 0.5 for _ in range(2)] if codes else [None, None]
    if codes and heads > 1:
        amax[0][1] = 0.0
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = None if new is None else torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
    want = []
    for pages_, x, a in ((kp, k, amax[0]), (vp, v, amax[1])):
        full = raw(pages_).clone()
        t = 0
        for b, c in enumerate(counts):
            for i in range(c):
                at = lens[b] - c + i
                row = x[t].cpu()
                if codes:
                    row = o.fp8_quantize(row, a.cpu().view(-1, 1))[0].view(heads, d)
                full[int(table[b, at // rows]), :, at % rows] = row.cuda()
                t += 1
        want.append(full)
    b200.paged_append(k, v, kp, vp, table, n, cu, k_amax=amax[0], v_amax=amax[1])
    for pages_, full in zip((kp, vp), want):
        r = raw(pages_)
        assert torch.equal(r.view(torch.uint8) if codes else r.view(torch.int16), full.view(torch.uint8) if codes else full.view(torch.int16))


@pytest.mark.parametrize("heads,most", [(1, 40), (2, 1), (1, 3000)])
def test_append_of_many_sequences(b200, heads, most):
    """A CTA's tokens are of many sequences, some of which bring nothing, or all of one."""
    g = torch.Generator(device="cuda").manual_seed(most)
    fresh = torch.randint(0, most + 1, (60000 // (most + 1) + 2,), device="cuda", generator=g)
    old = torch.randint(0, 20, fresh.shape, device="cuda", generator=g)
    lens, rows, d = fresh + old, 8, 16
    table, pages = table_of(g, lens.tolist(), rows)
    kp, vp, _, _ = pool(g, pages, heads, rows, d, torch.bfloat16)
    want_k, want_v = kp.clone(), vp.clone()
    cu = torch.nn.functional.pad(fresh.cumsum(0), (1, 0)).to(torch.int32)
    k, v = (torch.randn(int(cu[-1]), heads, d, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(2))
    b = torch.repeat_interleave(torch.arange(fresh.numel(), device="cuda"), fresh)
    at = old[b] + torch.arange(b.numel(), device="cuda") - cu[b]
    page = table[b, at // rows].long()
    want_k[page, :, at % rows], want_v[page, :, at % rows] = k, v
    b200.paged_append(k, v, kp, vp, table, lens.to(torch.int32), cu)
    assert torch.equal(kp.view(torch.int16), want_k.view(torch.int16)) and torch.equal(vp.view(torch.int16), want_v.view(torch.int16))


def test_append_leaves_what_it_is_not_given_alone(b200):
    """Tokens without a page, before the first token or beyond the table are left out; unaligned rows are copied first."""
    heads, d, rows = 2, 64, 8
    kp, vp = (torch.zeros(6, heads, rows, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.tensor([[0, -1], [1, 6], [2, 3]], dtype=torch.int32, device="cuda")
    n = torch.tensor([9, 16, 2], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 3, 6, 10], dtype=torch.int32, device="cuda")
    flat = torch.randn(10 * heads * d + 1, device="cuda").bfloat16()
    k = flat[1:].view(10, heads, d)
    b200.paged_append(k, k, kp, vp, table, n, cu)
    want = torch.zeros_like(kp)
    want[0, :, 6], want[0, :, 7] = k[0], k[1]            # tokens 6 and 7 of sequence 0; 8 has no page
    want[2, :, 0], want[2, :, 1] = k[8], k[9]            # sequence 2 claims two tokens for four rows: the last two
    assert torch.equal(kp, want) and torch.equal(vp, want)
    b200.paged_append(k[:0], k[:0], kp, vp, table[:0], n[:0])
    assert torch.equal(kp, want)


# ----------------------------------------------------------------------------- eviction
def evict_ref(w, n, keep, recent, sinks):
    """Kept tokens of one sequence and head; w on the host."""
    w = [-math.inf if x != x else x for x in w[:n].tolist()]
    fixed = [t for t in range(n) if t < sinks or t >= n - recent]
    rest = sorted((t for t in range(n) if sinks <= t < n - recent), key=lambda t: (-w[t], t))
    m = min(n, keep)
    return sorted(fixed + rest[:m - len(fixed)]) if m < n else list(range(n))


@pytest.mark.parametrize("values", ["quarters", "equal", "zeros", "wild"])
@pytest.mark.parametrize("lens,heads,d,rows,dt,keep,recent,sinks", [
    ([0, 1, 5, 8, 9, 40], 2, 64, 8, torch.bfloat16, 8, 2, 1),
    ([300, 64, 65, 1000], 3, 80, 5, E4M3, 64, 0, 0),
    ([300, 64, 65, 1000], 3, 128, 16, torch.float16, 64, 60, 4),
    ([2000, 2000], 1, 16, 1, torch.float16, 1999, 0, 0),
    ([5000, 100, 257], 8, 128, 24, torch.bfloat16, 256, 16, 4),
    ([20000, 9], 2, 64, 32, E4M3, 5000, 100, 4),
    ([500], 1, 64, 16, torch.bfloat16, 0, 0, 0),
    ([70000], 1, 32, 64, E4M3, 30000, 1, 0),
])
def test_evict(b200, lens, heads, d, rows, dt, keep, recent, sinks, values):
    g = torch.Generator(device="cuda").manual_seed(keep + d)
    table, pages = table_of(g, lens, rows)
    spare = max(1, -(-keep // rows))
    kp, vp, _, _ = pool(g, pages + spare * len(lens), heads, rows, d, dt)
    fresh = (pages + torch.randperm(spare * len(lens), device="cuda", generator=g)).to(torch.int32).view(len(lens), spare)
    L = max(max(lens), keep) + 3
    w = {"quarters": lambda: (torch.randn(len(lens), heads, L, device="cuda", generator=g) * 2).exp().mul(4).round().div(4),
         "equal": lambda: torch.full((len(lens), heads, L), 0.5, device="cuda"),
         "zeros": lambda: torch.where(torch.rand(len(lens), heads, L, device="cuda", generator=g) < 0.5, -0.0, 0.0),
         "wild": lambda: torch.randn(len(lens), heads, L, device="cuda", generator=g) * 1e30}[values]()
    if values == "wild":
        pick = torch.rand(w.shape, device="cuda", generator=g)
        w[pick < 0.1] = float("nan")
        w[(pick >= 0.1) & (pick < 0.15)] = float("inf")
        w[(pick >= 0.15) & (pick < 0.2)] = -float("inf")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    old_k, old_v, old_w = raw(kp).clone(), raw(vp).clone(), w.clone()
    kept, m, nw = b200.paged_evict(kp, vp, table, n, w, fresh, keep=keep, recent=recent, sinks=sinks)
    assert m.tolist() == [min(x, keep) for x in lens] and kept.shape == (len(lens), heads, keep)
    assert torch.equal(w.view(torch.int32), old_w.view(torch.int32))
    want_k, want_v = old_k.clone(), old_v.clone()
    for b, x in enumerate(lens):
        for h in range(heads):
            ref = evict_ref(old_w[b, h].cpu(), x, keep, recent, sinks)
            assert kept[b, h].tolist() == ref + [-1] * (keep - len(ref))
            at, j = torch.tensor(ref, dtype=torch.long, device="cuda"), torch.arange(len(ref), device="cuda")
            assert torch.equal(nw[b, h, :len(ref)].view(torch.int32), old_w[b, h, at].view(torch.int32)) and not nw[b, h, len(ref):].any()
            for want, old in ((want_k, old_k), (want_v, old_v)):
                want[fresh[b].long()[j // rows], h, j % rows] = old[table[b].long()[at // rows], h, at % rows]
    as_bits = lambda t: t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int16)  # noqa: E731
    assert torch.equal(as_bits(raw(kp)), as_bits(want_k)) and torch.equal(as_bits(raw(vp)), as_bits(want_v))


# ----------------------------------------------------------------------------- refusals
def test_what_is_refused(b200):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    kp, table, n, q, k = z(4, 2, 16, 64), z(3, 4, dtype=torch.int32), z(3, dtype=torch.int32), z(3, 4, 64), z(3, 2, 64)
    amax, w = torch.ones(1, device="cuda"), z(3, 2, 64, dtype=torch.float32)

    def refused(call, *a, match=None, **kw):
        with pytest.raises((RuntimeError, ValueError), match=match):
            call(*a, **kw)

    attend, append, evict = b200.paged_attention, b200.paged_append, b200.paged_evict
    refused(attend, q.float(), kp, kp, table, n, match="float16 | bfloat16")
    refused(attend, q.half(), kp, kp, table, n, match="share a type")
    refused(attend, q, kp, kp, table, n, k_amax=amax, v_amax=amax, match="FP8")
    refused(attend, q, kp.to(E4M3), kp.to(E4M3), table, n, match="FP8")
    refused(attend, q, kp.to(E4M3), kp.to(E4M3), table, n, k_amax=amax.expand(3), v_amax=amax.expand(3), match="per kv head")
    refused(attend, q.float(), kp.float(), kp.float(), table, n, match="pages of")
    refused(attend, q, kp, kp[:, :1], table, n, match="one type")
    refused(attend, z(3, 3, 64), kp, kp, table, n, match="multiple of the kv heads")
    refused(attend, z(2, 4, 64), kp, kp, table, n, match="expected q")
    refused(attend, q, kp, kp, table.long(), n, match="int32")
    refused(attend, q, kp, kp, table, n.long(), match="int32")
    refused(attend, q, kp, kp, table, n[:2], match="lens")
    refused(attend, q, kp, kp, table.cpu(), n, match="device")
    refused(attend, q, kp, kp, table, n, weights=w[:, :1], match="weights")
    refused(attend, q, kp, kp, table, n, weights=w.half(), match="weights")
    refused(attend, q, kp, kp, table, n, sinks=-1, match="sinks")
    refused(attend, q, kp, kp, table, n, scale=-1.0, match="scale")
    refused(attend, z(3, 4, 24), z(4, 2, 16, 24), z(4, 2, 16, 24), table, n, match="multiple of 16")
    refused(attend, z(3, 4, 144), z(4, 2, 16, 144), z(4, 2, 16, 144), table, n, match="multiple of 16")
    refused(attend, q, z(4, 2, 16, 128)[..., ::2], z(4, 2, 16, 128)[..., ::2], table, n, match="contiguous")
    refused(append, k.half(), k.half(), kp, kp, table, n, match="share a type")
    refused(append, k[:2], k[:2], kp, kp, table, n, match="one token of every sequence")
    refused(append, z(3, 3, 64), z(3, 3, 64), kp, kp, table, n, match="expected k and v")
    refused(append, k, k, kp, kp, table, n, n, match="cu_new")
    refused(evict, kp, kp, table, n, w, table, keep=8, recent=8, sinks=1, match="recent")
    refused(evict, kp, kp, table, n, w, table[:, :1], keep=32, match="room")
    refused(evict, kp, kp, table, n, w[..., :8], table, keep=32, match="weights")
    refused(evict, kp, kp, table, n, w.double(), table, keep=8, match="weights")
    f = b200.window_attention
    q, k = z(1, 4, 8, 64), z(1, 2, 8, 64)
    refused(f, q.float(), k.float(), k.float(), match="float16 | bfloat16")
    refused(f, q, k.half(), k, match="share a type")
    refused(f, q, z(1, 3, 8, 64), z(1, 3, 8, 64), match="Hq % Hkv")
    refused(f, q, k, k, sinks=-1, match="sinks")
    refused(f, q, k, k, scale=float("inf"), match="scale")
    refused(f, q, k, k, q_lens=torch.zeros(2, dtype=torch.int32, device="cuda"), match="q_lens")
    refused(f, q, k, k, k_lens=torch.zeros(1, device="cuda"), match="k_lens")
    refused(f, q[0], k[0], k[0], match="expected q")


# ----------------------------------------------------------------------------- sizes of the other forms
@pytest.mark.parametrize("lens,heads,keep", [([120000, 30], 1, 50000), ([13000, 12000], 160, 700), ([5000] * 3, 4, 4999), ([100000], 8, 257), ([400001, 7], 1, 30000), ([49000, 48999], 160, 300)])
def test_evict_long_rows_against_a_sort(b200, lens, heads, keep):
    """Rows over clusters, whose keys are held in shared memory or read again on each walk."""
    g = torch.Generator(device="cuda").manual_seed(keep)
    rows, d, L = 64, 16, max(lens)
    table, pages = table_of(g, lens, rows)
    spare = -(-keep // rows)
    kp, vp, _, _ = pool(g, pages + spare * len(lens), heads, rows, d, E4M3)
    fresh = torch.arange(pages, pages + spare * len(lens), dtype=torch.int32, device="cuda").view(len(lens), spare)
    w = (torch.randn(len(lens), heads, L, device="cuda", generator=g) * 2).exp()
    w = torch.where(torch.rand(w.shape, device="cuda", generator=g) < 0.5, (w * 2).round() / 2, w)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kept, m, nw = b200.paged_evict(kp, vp, table, n, w, fresh, keep=keep, recent=keep // 8, sinks=3)
    for b, x in enumerate(lens):
        held = w[b, :, :x].clone()
        held[:, :3] = math.inf
        held[:, max(0, x - keep // 8):] = math.inf
        at = held.sort(dim=1, descending=True, stable=True).indices[:, :min(x, keep)].sort(dim=1).values
        assert torch.equal(kept[b, :, :at.shape[1]].long(), at) and (kept[b, :, at.shape[1]:] == -1).all()
        assert torch.equal(nw[b, :, :at.shape[1]], w[b].gather(1, at)) and not nw[b, :, at.shape[1]:].any()
        j = torch.arange(at.shape[1], device="cuda")
        for h in (0, heads - 1):
            assert torch.equal(raw(vp)[fresh[b].long()[j // rows], h, j % rows], raw(vp)[table[b].long()[at[h] // rows], h, at[h] % rows])


def test_the_ops_and_the_functions_are_one(b200):
    """The torch.library ops, which a graph holds, and the functions give the same bits; inference tensors and other dtypes of scale pass."""
    g = torch.Generator(device="cuda").manual_seed(9)
    lens = [70, 300]
    table, pages = table_of(g, lens, 16)
    kp, vp, ka, va = pool(g, pages, 2, 16, 64, E4M3)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(2, 6, 64, device="cuda", generator=g).bfloat16()
    w1, w2 = (torch.zeros(2, 2, 320, device="cuda") for _ in range(2))
    a = b200.paged_attention(q, kp, vp, table, n, k_amax=ka, v_amax=va, weights=w1, scale=0.25, window=100, sinks=2)
    b = torch.ops.tensorrt.b200_paged_attention(q, kp, vp, table, n, w2, ka, va, 0.25, 100, 2)
    assert torch.equal(a, b) and torch.equal(w1, w2)
    assert torch.equal(a, b200.paged_attention(q, kp, vp, table, n, k_amax=ka.double(), v_amax=va.half().float().fill_(va.item()), scale=0.25, window=100, sinks=2))
    with torch.inference_mode():
        assert torch.equal(b200.paged_attention(q.clone(), kp, vp, table, n, k_amax=ka, v_amax=va, scale=1), torch.ops.tensorrt.b200_paged_attention(
            q, kp, vp, table, n, None, ka, va, 1.0, 0, 0))
    x = torch.randn(1, 4, 40, 64, device="cuda", generator=g).half()
    assert torch.equal(b200.window_attention(x, x, x, window=9), torch.ops.tensorrt.b200_window_attention(x, x, x, None, None, 0.0, 9, 0))


def test_graphs_share_no_workspace_with_their_stream(b200):
    """Two graphs captured on one stream, replayed side by side on others while that stream goes on: each has a workspace of its own."""
    g = torch.Generator(device="cuda").manual_seed(10)
    lens = [5000, 3000]
    table, pages = table_of(g, lens, 16)
    kp, vp, _, _ = pool(g, pages, 2, 16, 128, torch.bfloat16)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs = [torch.randn(2, 8, 128, device="cuda", generator=g).bfloat16() for _ in range(3)]
    want = [b200.paged_attention(q, kp, vp, table, n) for q in qs]
    home, others = torch.cuda.Stream(), [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for q in qs[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=home):
            outs.append([b200.paged_attention(q, kp, vp, table, n) for _ in range(4)])
    torch.cuda.synchronize()
    for _ in range(20):
        for st, graph in zip(others, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        with torch.cuda.stream(home):
            eager = [b200.paged_attention(qs[2], kp, vp, table, n) for _ in range(4)]
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(o, want[i]) for o in outs[i])
        assert all(torch.equal(o, want[2]) for o in eager)


# ----------------------------------------------------------------------------- tokens that are not there
@pytest.mark.parametrize("lens,heads,rows,keep,recent,sinks,gone", [
    ([40, 40, 17], 2, 8, 16, 4, 2, 0.4),                 # some more, some fewer than `keep` are there
    ([40, 0, 7], 2, 8, 40, 30, 10, 0.5),                 # all that are there stay
    ([300, 64, 1000], 3, 5, 64, 0, 0, 0.3),
    ([700, 650], 1, 1, 650, 64, 8, 0.05),
    ([33, 64], 1, 64, 20, 3, 3, 1.0),                    # none is there
    ([20000, 9], 2, 32, 5000, 100, 4, 0.3),              # over a cluster
    ([400001, 70], 1, 64, 30000, 300, 10, 0.2),          # whose keys are read again on each walk
    ([400001, 70], 1, 64, 30000, 0, 0, 0.95),
])
@pytest.mark.parametrize("values", ["quarters", "lowest"])
def test_evict_of_tokens_without_a_page(b200, lens, heads, rows, keep, recent, sinks, gone, values):
    """A page that the table does not name (given back behind a window) holds no tokens that could stay: what stays is attended to as
    the same tokens were before."""
    g = torch.Generator(device="cuda").manual_seed(keep + rows)
    d, L = 16, max(max(lens), keep)
    table, pages = table_of(g, lens, rows)
    spare = -(-keep // rows)
    kp, vp, _, _ = pool(g, pages + spare * len(lens), heads, rows, d, torch.bfloat16)
    kp[pages:], vp[pages:] = float("nan"), float("nan")   # what the fresh pages hold beyond the rows that move is nobody's
    fresh = (pages + torch.randperm(spare * len(lens), device="cuda", generator=g)).to(torch.int32).view(len(lens), spare)
    holes = torch.rand(table.shape, device="cuda", generator=g) < gone
    table[holes] = torch.where(torch.rand(table.shape, device="cuda", generator=g) < 0.5, -1, kp.shape[0])[holes].to(torch.int32)
    w = (torch.randn(len(lens), heads, L, device="cuda", generator=g) * 2).exp().mul(4).round().div(4)
    if values == "lowest":
        w = torch.where(w < 1.0, w, -float("inf"))
        w[torch.rand(w.shape, device="cuda", generator=g) < 0.3] = float("nan")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kept, m, nw = b200.paged_evict(kp, vp, table, n, w, fresh, keep=keep, recent=recent, sinks=sinks)
    for b, x in enumerate(lens):
        at = torch.arange(x, device="cuda")
        there = ((table[b] >= 0) & (table[b] < kp.shape[0]))[at // rows]
        stays = min(int(there.sum()), keep)
        assert int(m[b]) == stays
        for h in range(heads):
            rank = torch.where(w[b, h, :x].isnan(), -math.inf, w[b, h, :x])
            order = rank.sort(descending=True, stable=True).indices
            group = torch.where(there, torch.where((at < sinks) | (at >= x - recent), 2, 1), 0)
            order = order[group[order].sort(descending=True, stable=True).indices]
            ref = order[:stays].sort().values
            assert torch.equal(kept[b, h, :stays].long(), ref) and (kept[b, h, stays:] == -1).all()
            assert torch.equal(nw[b, h, :stays].view(torch.int32), w[b, h, ref].view(torch.int32)) and not nw[b, h, stays:].any()
            j = torch.arange(stays, device="cuda")
            for p in (kp, vp):
                assert torch.equal(p[fresh[b].long()[j // rows], h, j % rows], p[table[b].long()[ref // rows], h, ref % rows])
    q = torch.randn(len(lens), heads, d, device="cuda", generator=g).bfloat16()
    ref, mass, _ = attention_ref(q, kp, vp, fresh, m.tolist(), None, None, 0, 0)
    check_out(b200.paged_attention(q, kp, vp, fresh, m), ref, mass)


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("counts,rows_given", [([1, 1, 1], 5), ([3, 0, 6], 40), ([0, 0, 0], 4), ([70, 1, 300], 1000)])
def test_append_of_rows_that_no_sequence_brings(b200, counts, rows_given, codes):
    """Rows behind the last sequence's (tokens padded to a fixed number) are written nowhere, whatever the table names there."""
    g = torch.Generator(device="cuda").manual_seed(rows_given)
    heads, d, rows = 2, 64, 16
    lens = [c + 5 * i for i, c in enumerate(counts)]
    table, pages = table_of(g, lens, rows, width=200)
    table[table < 0] = 0                                  # entries not in use: page 0, which belongs to somebody
    kp, vp, ka, va = pool(g, pages, heads, rows, d, E4M3 if codes else torch.bfloat16)
    k, v = (torch.randn(rows_given, heads, d, device="cuda", generator=g).bfloat16() for _ in range(2))
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
    want_k, want_v = kp.clone(), vp.clone()
    b200.paged_append(k[:sum(counts)], v[:sum(counts)], want_k, want_v, table, n, cu, k_amax=ka, v_amax=va)
    b200.paged_append(k, v, kp, vp, table, n, cu, k_amax=ka, v_amax=va)
    for got, want in ((kp, want_k), (vp, want_v)):
        assert torch.equal(raw(got).view(torch.uint8), raw(want).view(torch.uint8))
    later = cu + 2                                        # rows in front of the first sequence's are nobody's either
    kp2, vp2 = want_k.clone(), want_v.clone()
    pad = lambda t: torch.cat([torch.full_like(t[:2], 7.0), t[:sum(counts)]])  # noqa: E731
    b200.paged_append(pad(k), pad(v), kp2, vp2, table, n, later, k_amax=ka, v_amax=va)
    assert torch.equal(raw(kp2).view(torch.uint8), raw(want_k).view(torch.uint8)) and torch.equal(raw(vp2).view(torch.uint8), raw(want_v).view(torch.uint8))


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("nats", [8.0, 12.0, 16.0])
@pytest.mark.parametrize("dt,pt,heads,group,d,n", [
    (torch.float16, torch.float16, 2, 4, 64, 700), (torch.float16, torch.float16, 1, 16, 128, 40), (torch.float16, E4M3, 2, 1, 128, 700),
    (torch.bfloat16, E4M3, 1, 8, 64, 5000), (torch.bfloat16, torch.bfloat16, 1, 2, 80, 700), (torch.bfloat16, E4M3, 1, 12, 96, 20)])
def test_keys_far_below_the_heaviest(b200, dt, pt, heads, group, d, n, nats, weighted):
    """A first key with nearly all of the weight and no value: the result is made of the others, whose weights are far below one.  P is
    held in 16 bits with the heaviest of its keys at 2^11 or above, so that a weight of e^-17 is still a normal number of fp16; the values
    are large, so that the result is one too."""
    g = torch.Generator(device="cuda").manual_seed(n + d)
    rows = 16
    table, pages = table_of(g, [n], rows)
    k, v = torch.randn(n, heads, d, device="cuda", generator=g) * 0.02, (torch.rand(n, heads, d, device="cuda", generator=g) + 0.5) * 4096
    q = torch.randn(1, heads * group, d, device="cuda", generator=g)
    q[..., 0], k[..., 0] = 4.0, 0.0
    k[0], v[0] = 0.0, 0.0
    k[0, :, 0] = nats / 4
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    kp, vp = (torch.zeros(pages, heads, rows, d, device="cuda", dtype=pt) for _ in range(2))
    ka, va = (torch.tensor([a], device="cuda") if pt == E4M3 else None for a in (4.0, 8192.0))
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    b200.paged_append(k, v, kp, vp, table, lens, torch.tensor([0, n], dtype=torch.int32, device="cuda"), k_amax=ka, v_amax=va)
    w = torch.zeros(1, heads, n, device="cuda") if weighted else None
    out = b200.paged_attention(q, kp, vp, table, lens, k_amax=ka, v_amax=va, weights=w, scale=1.0)
    ref, mass, gained = attention_ref(q, kp, vp, table, [n], ka, va, 0, 0, scale=1.0)
    assert (ref[..., 1:].abs() > 0).all() and gained[0, :, 0].min() > 0.5
    check_out(out, ref, mass)
    if weighted:
        assert ((w.double() - gained[:, :, :n]).abs() <= 2.0 ** -12 * gained[:, :, :n]).all()


@pytest.mark.parametrize("dt,pt", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, E4M3)])
@pytest.mark.parametrize("size", [2.0 ** e for e in (4, 12, 20, 23, 24, 25, 26, 27, 28, 30, 60)], ids=str)
def test_logits_that_32_bits_hold_coarsely(b200, dt, pt, size):
    """Logits whose neighbours in 32 bits are up to many nats apart, rising along the keys: P stays in the range of its type, the result a mean
    of the values."""
    g = torch.Generator(device="cuda").manual_seed(31)
    n, d, rows = 1500, 64, 16
    table, pages = table_of(g, [n], rows)
    kp, vp, ka, va = pool(g, pages, 1, rows, d, pt)
    rising = torch.linspace(3.0, 4.0, n, device="cuda")
    where = (table[0].long()[torch.arange(n, device="cuda") // rows], 0, torch.arange(n, device="cuda") % rows)
    if pt == E4M3:
        ka = torch.tensor([448.0], device="cuda")
        raw(kp)[where] = (rising[:, None] * torch.ones(d, device="cuda")).to(E4M3).view(torch.uint8)
    else:
        kp[where] = (rising[:, None] * torch.ones(d, device="cuda")).to(dt)
    q = (torch.rand(1, 4, d, device="cuda", generator=g) + 0.5).to(dt)
    out = b200.paged_attention(q, kp, vp, table, torch.tensor([n], dtype=torch.int32, device="cuda"), k_amax=ka, v_amax=va, scale=size / (4 * d)).float()
    values = raw(vp)[where].view(vp.dtype).float() * (1.0 if va is None else va / 448)
    room = 2.0 ** -6 * values.abs().amax()               # roundings of P, of its sum and of the result
    assert torch.isfinite(out).all() and (out >= values.amin(0) - room).all() and (out <= values.amax(0) + room).all()


def test_inputs_that_require_gradients(b200):
    """No gradient is defined: a result of such inputs says so as that of the op does, and is not a constant without a word."""
    from torch.autograd import forward_ad

    g = torch.Generator(device="cuda").manual_seed(21)
    table, pages = table_of(g, [40, 9], 16)
    kp, vp, _, _ = pool(g, pages, 2, 16, 64, torch.bfloat16)
    n = torch.tensor([40, 9], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda", generator=g).bfloat16()
    x = torch.randn(1, 2, 40, 64, device="cuda", generator=g).bfloat16()
    ops = torch.ops.tensorrt
    calls = [(lambda t: b200.paged_attention(t, kp, vp, table, n), lambda t: ops.b200_paged_attention(t, kp, vp, table, n, None, None, None, 0.0, 0, 0), q),
             (lambda t: b200.window_attention(t, x, x), lambda t: ops.b200_window_attention(t, x, x, None, None, 0.0, 0, 0), x),
             (lambda t: b200.window_attention(x, x, t), lambda t: ops.b200_window_attention(x, x, t, None, None, 0.0, 0, 0), x)]
    for f, op, t in calls:
        plain = f(t)
        assert not plain.requires_grad
        leaf = t.clone().requires_grad_()
        assert f(leaf).requires_grad and op(leaf).requires_grad and torch.equal(f(leaf), plain)
        with torch.no_grad():
            assert not f(leaf).requires_grad and torch.equal(f(leaf), plain)

        def dual(call):
            with forward_ad.dual_level():
                try:
                    return forward_ad.unpack_dual(call(forward_ad.make_dual(t, torch.ones_like(t)))).tangent is None
                except (RuntimeError, NotImplementedError) as e:
                    return str(e)

        assert dual(f) == dual(op)
        assert "b200_" in str(torch.jit.trace(f, (t,), check_trace=False).graph)


@pytest.mark.parametrize("window,sinks", [(100, 4), (0, 0)])
def test_wide_tables_and_weights_take_no_more_room_than_what_is_seen(b200, window, sinks):
    g = torch.Generator(device="cuda").manual_seed(22)
    lens, heads, group, rows, d = [3000, 40, 0, 101], 4, 8, 16, 64
    width = 8192 if window else 200                       # 131072 tokens, of which a window sees 104
    table, pages = table_of(g, lens, rows, width=width)
    kp, vp, _, _ = pool(g, pages, heads, rows, d, torch.bfloat16)
    q = torch.randn(4, heads * group, d, device="cuda", generator=g).bfloat16()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    w = torch.zeros(4, heads, 131072, device="cuda")
    b200.paged_attention(q, kp, vp, table, n, weights=w, window=window, sinks=sinks)      # the workspace is there
    w.zero_()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = b200.paged_attention(q, kp, vp, table, n, weights=w, window=window, sinks=sinks)
    assert torch.cuda.max_memory_allocated() - before <= 4 * 32 * 4 * ((104 if window else 3200) + 4) + (1 << 20)
    ref, mass, gained = attention_ref(q, kp, vp, table[:, :200], lens, None, None, window, sinks)
    check_out(out, ref, mass)
    assert (w[..., :3200].double() - gained).abs().max() <= 2.0 ** -10 and not w[..., 3200:].any()
