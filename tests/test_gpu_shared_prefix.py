"""Attention of one new token where groups of sequences share a prefix, against a 64-bit restatement.  Bounds as in
tests/test_gpu_paged_cache.py: one rounding of the result, one of P to 16 bits, 32-bit sums."""
import math

import pytest
import torch

from test_gpu_paged_cache import E4M3, check_out, pool, raw

pytestmark = pytest.mark.gpu


def batch(g, groups, alone, rows, mixed):
    """Tables of groups (tokens of the prefix, tokens of each sequence behind it) and of sequences by themselves: (table, lens, members,
    tokens, [(line, first token that is its own)], pages).  Pages lie in no order; a page that the prefix ends in is each sequence's own."""
    n = sum(len(own) for _, own in groups) + len(alone)
    places = list(range(n))
    if mixed:
        places.sort(key=lambda i: (i * 0.618) % 1.0)
    need = sum(-(-t // rows) for t, _ in groups) + sum(-(-(t % rows + k) // rows) for t, own in groups for k in own) + sum(-(-k // rows) for k in alone)
    numbers = torch.randperm(need + 1, generator=g, device="cuda").to(torch.int32).cpu().tolist()
    width = max([-(-(t + max(own)) // rows) for t, own in groups] + [-(-k // rows) for k in alone] + [1])
    table, lens, members, at = torch.full((n, width), -1, dtype=torch.int32), [0] * n, [], 0
    leaders = list(range(n))
    for t, own in groups:
        prefix = [numbers.pop() for _ in range(-(-t // rows))]
        m = sorted(places[at:at + len(own)])
        at += len(own)
        for b, k in zip(m, own):
            mine = [numbers.pop() for _ in range(-(-(t % rows + k) // rows))]
            line = prefix[:t // rows] + mine
            if b == m[0]:                                      # the leader's line names the page that the prefix ends in
                line = prefix + mine[1:] if t % rows else prefix + mine
                if k and t % rows:
                    pass
            table[b, :len(line)] = torch.tensor(line, dtype=torch.int32)
            lens[b], leaders[b] = t + k, m[0]
        members.append(m)
    for k in alone:
        b = places[at]
        at += 1
        line = [numbers.pop() for _ in range(-(-k // rows))]
        table[b, :len(line)] = torch.tensor(line, dtype=torch.int32)
        lens[b] = k
    return table.cuda(), lens, members, [t for t, _ in groups], leaders, need + 1


def reference(q, kp, vp, table, lens, members, tokens, ka, va, scale=None):
    """(out, sum P |V|) in 64 bits; also which rows of the pools are read."""
    n, hq, d = q.shape
    heads, rows, pages = kp.shape[1], kp.shape[2], kp.shape[0]
    g = hq // heads
    out, mass = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda"), torch.zeros(n, hq, d, dtype=torch.float64, device="cuda")
    used = torch.zeros(pages, rows, dtype=torch.bool, device="cuda")
    line, shared = list(range(n)), [0] * n
    for m, t in zip(members, tokens):
        for b in m:
            if t <= lens[b]:
                line[b], shared[b] = m[0], t
    for b in range(n):
        at = torch.arange(lens[b], device="cuda")
        page = torch.where(at < shared[b], table[line[b]].long()[at // rows], table[b].long()[at // rows])
        ok = (page >= 0) & (page < pages)
        at, page = at[ok], page[ok]
        used[page, at % rows] = True
        for h in range(heads):
            scales = [1.0 if a is None else (a.float() / 448).double()[h if a.numel() > 1 else 0] for a in (ka, va)]
            k, v = (raw(p)[page, h, at % rows].view(p.dtype).double() * f for p, f in zip((kp, vp), scales))
            s = q[b, h * g:(h + 1) * g].double() @ k.T * (1 / math.sqrt(d) if scale is None else scale)
            p = torch.softmax(s, -1) if len(at) else s
            out[b, h * g:(h + 1) * g], mass[b, h * g:(h + 1) * g] = p @ v, p @ v.abs()
    return out, mass, used


CASES = [
    # groups, alone, heads, query heads of each, D, rows, token type, page type, layout, dealt out
    ([(1, [1, 1])], [], 1, 1, 64, 16, torch.bfloat16, torch.bfloat16, "hnd", False),
    ([(16, [0, 1, 2])], [5], 2, 4, 128, 16, torch.bfloat16, torch.bfloat16, "hnd", False),
    ([(17, [3, 0, 40]), (127, [1, 1])], [0, 300], 2, 4, 128, 16, torch.float16, torch.float16, "nhd", True),
    ([(128, [5] * 4), (129, [7] * 3), (0, [4, 5])], [64], 2, 8, 128, 32, torch.bfloat16, torch.bfloat16, "hnd", True),
    ([(500, list(range(1, 40))), (257, [9, 8])], [], 1, 5, 96, 5, torch.bfloat16, torch.bfloat16, "nhd", False),
    ([(384, [30, 1, 77])], [], 3, 1, 80, 24, torch.float16, torch.float16, "hnd", True),
    ([(333, [30, 1, 77])], [], 3, 1, 80, 24, torch.float16, E4M3, "nhd", True),
    ([(700, [1] * 20), (64, [2] * 2)], [1], 2, 8, 128, 64, torch.bfloat16, E4M3, "hnd", False),
    ([(1000, [1, 500])], [], 1, 16, 16, 1, torch.float16, torch.float16, "hnd", False),
    ([(1000, [3, 50])], [], 1, 20, 48, 7, torch.bfloat16, E4M3, "hnd", False),
    ([(4096, [100] * 70)], [], 2, 8, 64, 16, torch.bfloat16, torch.bfloat16, "hnd", False),
    ([(9000, [1, 2, 3])], [9000], 2, 4, 112, 128, torch.float16, torch.float16, "nhd", False),
    ([(30000, [1] * 6), (300, [1] * 40)], [2] * 5, 1, 64, 128, 64, torch.bfloat16, E4M3, "hnd", True),
    ([(16 * (1 + i % 5), [1 + i % 3] * 2) for i in range(300)], [3] * 10, 1, 2, 64, 16, torch.bfloat16, torch.bfloat16, "hnd", True),
    ([(0, [5, 6])], [7], 1, 2, 64, 16, torch.bfloat16, torch.bfloat16, "hnd", False),
]


def made(case, seed=3):
    groups, alone, heads, group, d, rows, dt, pt, layout, mixed = case
    g = torch.Generator(device="cuda").manual_seed(seed + d)
    table, lens, members, tokens, leaders, pages = batch(g, groups, alone, rows, mixed)
    kp, vp, ka, va = pool(g, pages, heads, rows, d, pt, layout)
    q = torch.randn(len(lens), heads * group + 3, d, device="cuda", generator=g).to(dt)[:, 1:1 + heads * group]
    return q, kp, vp, ka, va, table, lens, members, tokens


def on_device(lens):
    return torch.tensor(lens, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"g{len(c[0])}_n{len(c[0][0][1])}_t{c[0][0][0]}_h{c[2]}x{c[3]}_d{c[4]}_p{c[5]}_{str(c[7])[6:]}")
def test_shared_prefix(b200, case):
    q, kp, vp, ka, va, table, lens, members, tokens = made(case)
    used = reference(q, kp, vp, table, lens, members, tokens, ka, va)[2]
    for t in (kp, vp):                                     # what is not attended to does not matter
        raw(t)[(~used)[:, None].expand(t.shape[:3])] = 0x7F if t.element_size() == 1 else float("nan")
    ref, mass, _ = reference(q, kp, vp, table, lens, members, tokens, ka, va)
    prefix = b200.SharedPrefix(members, tokens, len(lens))
    out = b200.shared_prefix_attention(q, kp, vp, table, on_device(lens), prefix, k_amax=ka, v_amax=va)
    check_out(out, ref, mass)
    for _ in range(3):                                     # no order of CTAs decides anything
        assert torch.equal(out, b200.shared_prefix_attention(q, kp, vp, table, on_device(lens), prefix, k_amax=ka, v_amax=va))
    op = torch.ops.tensorrt.b200_shared_prefix_attention(q, kp, vp, table, on_device(lens), prefix.plan(q.shape[1], kp.shape[1]), prefix.groups, prefix.largest, ka, va, 0.0)
    assert torch.equal(out, op)
    # the same from a plan that leaves room for others
    wide = b200.SharedPrefix(members, tokens, len(lens), groups=len(lens), largest=len(lens))
    check_out(b200.shared_prefix_attention(q, kp, vp, table, on_device(lens), wide, k_amax=ka, v_amax=va), ref, mass)


def test_sequences_that_are_shorter_than_their_prefix(b200):
    """One that was cut or released is attended to through its own line alone; holes in the lines are keys that are not there."""
    case = ([(64, [3, 5, 9, 2]), (160, [1, 1, 1])], [20], 2, 4, 64, 16, torch.bfloat16, torch.bfloat16, "hnd", True)
    q, kp, vp, ka, va, table, lens, members, tokens = made(case)
    a, b = members
    for line in (a[1], a[2]):                              # own lines name their whole text
        table[line, :4] = table[a[0], :4]
    lens[a[1]], lens[a[2]], lens[b[2]] = 40, 0, -3
    table[b[0], 2], table[b[0], 5], table[b[1], 10] = -1, 1 << 20, -5      # holes: in the prefix (the leader's line), and behind it
    lens = [max(n, 0) for n in lens]
    ref, mass, _ = reference(q, kp, vp, table, lens, members, tokens, ka, va)
    n = on_device(lens)
    n[b[2]] = -3
    out = b200.shared_prefix_attention(q, kp, vp, table, n, b200.SharedPrefix(members, tokens, len(lens)))
    check_out(out, ref, mass)
    assert not out[a[2]].any() and not out[b[2]].any()
    # no page at all
    out = b200.shared_prefix_attention(q, kp[:0], vp[:0], table, n, b200.SharedPrefix(members, tokens, len(lens)))
    assert not out.any()
    # lines that cannot hold the prefix
    with pytest.raises(ValueError):
        b200.shared_prefix_attention(q, kp, vp, table[:, :9], n, b200.SharedPrefix(members, tokens, len(lens)))


@pytest.mark.parametrize("dt,pt", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, E4M3), (torch.float16, E4M3)], ids=str)
def test_values_that_are_not_finite(b200, dt, pt):
    """Where they are seen they show in the rows that see them, and nowhere else."""
    case = ([(256, [4, 4]), (128, [4, 4])], [9], 2, 2, 64, 16, dt, pt, "hnd", False)
    q, kp, vp, ka, va, table, lens, members, tokens = made(case)
    clean = b200.shared_prefix_attention(q, kp, vp, table, on_device(lens), b200.SharedPrefix(members, tokens, 5), k_amax=ka, v_amax=va)
    raw(vp)[table[0, 3], 1, 2] = 0x7F if pt == E4M3 else float("nan")      # token 50 of the first prefix, kv head 1
    out = b200.shared_prefix_attention(q, kp, vp, table, on_device(lens), b200.SharedPrefix(members, tokens, 5), k_amax=ka, v_amax=va)
    assert out[:2, 2:].isnan().all()
    assert torch.equal(out[:2, :2], clean[:2, :2]) and torch.equal(out[2:], clean[2:])
    raw(kp)[table[2, 1], 0, 5] = 0x7F if pt == E4M3 else float("nan")
    out = b200.shared_prefix_attention(q, kp, vp, table, on_device(lens), b200.SharedPrefix(members, tokens, 5), k_amax=ka, v_amax=va)
    assert out[2:4, :2].isnan().all() and torch.equal(out[2:4, 2:], clean[2:4, 2:]) and torch.equal(out[4], clean[4])


@pytest.mark.parametrize("pt", [torch.float16, E4M3, torch.bfloat16], ids=str)
@pytest.mark.parametrize("size", [3.0, 40.0])
def test_logits_of_every_size(b200, pt, size):
    """Maxima that keep rising along the keys, and logits of some hundreds: references are followed, in parts too."""
    dt = torch.bfloat16 if pt == torch.bfloat16 else torch.float16
    case = ([(5000, [40, 3, 200])], [100], 1, 8, 128, 16, dt, pt, "hnd", False)
    q, kp, vp, ka, va, table, lens, members, tokens = made(case)
    rise = torch.linspace(-1, 1, 5008, device="cuda")[:, None] * torch.ones(128, device="cuda")
    at = table[0, :313].long()
    k = rise.view(313, 1, 16, 128) * 4
    raw(kp)[at] = raw((k / (ka / 448) if pt == E4M3 else k).to(pt))
    q = (q.float() * 0.05 + 0.1).to(dt)
    scale = size / 40
    ref, mass, _ = reference(q, kp, vp, table, lens, members, tokens, ka, va, scale)
    check_out(b200.shared_prefix_attention(q, kp, vp, table, on_device(lens), b200.SharedPrefix(members, tokens, 4), k_amax=ka, v_amax=va, scale=scale), ref, mass)


@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 28, 2.0 ** 60])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=str)
def test_logits_that_32_bits_hold_coarsely(b200, dt, size):
    """A mean of the values that are seen, whatever the size of the logits, and no infinity on the way."""
    case = ([(700, [5, 9])], [], 1, 2, 64, 16, dt, dt, "hnd", False)
    q, kp, vp, ka, va, table, lens, members, tokens = made(case)
    out = b200.shared_prefix_attention(q, kp, vp, table, on_device(lens), b200.SharedPrefix(members, tokens, 2), scale=size).float()
    assert torch.isfinite(out).all() and out.abs().max() <= vp.float().abs().max() * (1 + 2.0 ** -7)


def test_ranges_of_each_head_and_their_types(b200):
    case = ([(300, [7, 8])], [33], 3, 4, 96, 32, torch.bfloat16, E4M3, "nhd", False)
    q, kp, vp, _, _, table, lens, members, tokens = made(case)
    ka, va = torch.tensor([3.0, 0.0, 5.5], device="cuda"), torch.tensor([1.0, 2.0, 0.25], device="cuda")
    ref, mass, _ = reference(q, kp, vp, table, lens, members, tokens, torch.where(ka == 0, 448.0, ka), va)
    prefix = b200.SharedPrefix(members, tokens, 3)
    for k, v in ((ka, va), (ka.double(), va.half())):
        check_out(b200.shared_prefix_attention(q, kp, vp, table, on_device(lens), prefix, k_amax=k, v_amax=v), ref, mass)
    check_out(b200.shared_prefix_attention(q, kp.view(torch.uint8), vp.view(torch.uint8), table, on_device(lens), prefix, k_amax=ka, v_amax=va), ref, mass)


def test_queries_far_from_one(b200):
    """8-bit pages: queries are scaled into the range of the products' type, row by row."""
    case = ([(400, [7, 8, 9, 1, 1])], [33], 2, 4, 64, 16, torch.bfloat16, E4M3, "hnd", False)
    q, kp, vp, ka, va, table, lens, members, tokens = made(case)
    for big in (2.0 ** 40, 2.0 ** -40):
        qq = q.clone()
        qq[1], qq[3] = qq[1] * big, 0
        ref, mass, _ = reference(qq, kp, vp, table, lens, members, tokens, ka, va, 1 / big if big > 1 else 0.125)
        out = b200.shared_prefix_attention(qq, kp, vp, table, on_device(lens), b200.SharedPrefix(members, tokens, 6), k_amax=ka, v_amax=va,
                                           scale=1 / big if big > 1 else 0.125)
        check_out(out[[1, 3]], ref[[1, 3]], mass[[1, 3]])


def test_pools_of_two_layouts_and_overlapping_rows(b200):
    """K and V stored differently; pools that no tensor map can hold (every head the same rows) go row by row."""
    g = torch.Generator(device="cuda").manual_seed(4)
    case = ([(300, [7, 8])], [33], 2, 4, 64, 16, torch.bfloat16, torch.bfloat16, "hnd", False)
    q, kp, vp, ka, va, table, lens, members, tokens = made(case)
    vp = vp.transpose(1, 2).contiguous().transpose(1, 2)
    prefix = b200.SharedPrefix(members, tokens, 3)
    ref, mass, _ = reference(q, kp, vp, table, lens, members, tokens, None, None)
    check_out(b200.shared_prefix_attention(q, kp, vp, table, on_device(lens), prefix), ref, mass)
    one = torch.randn(kp.shape[0], 1, 16, 64, device="cuda", generator=g).bfloat16().expand(-1, 2, -1, -1)
    ref, mass, _ = reference(q, one, one, table, lens, members, tokens, None, None)
    check_out(b200.shared_prefix_attention(q, one, one, table, on_device(lens), prefix), ref, mass)


def test_streams_graphs_and_plans_in_place(b200):
    """A captured call goes by the lengths, the table and the plan as they are when it is replayed; two graphs share nothing."""
    case = ([(320, [3, 4, 5])], [40, 50, 60], 2, 4, 64, 16, torch.bfloat16, torch.bfloat16, "hnd", False)
    q, kp, vp, _, _, table, lens, members, tokens = made(case)
    table = torch.nn.functional.pad(table, (0, 4), value=-1)
    n, other = on_device(lens), q.flip(0).contiguous()
    prefix = b200.SharedPrefix(members, tokens, 6, groups=3, largest=6)
    f = lambda x: b200.shared_prefix_attention(x, kp, vp, table, n, prefix)  # noqa: E731
    want = [f(q), f(other)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        there = [f(q), f(other)]
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(there, want))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, x in zip(graphs, (q, other)):
        with torch.cuda.graph(graph):
            outs.append([f(x) for _ in range(3)])
    for _ in range(5):
        for graph, s in zip(graphs, (torch.cuda.current_stream(), stream)):
            with torch.cuda.stream(s):
                graph.replay()
        eager = f(q)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0]) and all(torch.equal(o, w) for got, w in zip(outs, want) for o in got)
    # other groups, other lengths
    table[4, :20], table[5, :20] = table[3, :20], table[3, :20]
    n.copy_(on_device([320, 323, 330, 40, 47, 41]))
    prefix.update([[5, 3, 4], [0, 2]], [32, 160])
    table[2, :20] = table[0, :20]
    torch.cuda.synchronize()
    graphs[0].replay()
    torch.cuda.synchronize()
    ref, mass, _ = reference(q, kp, vp, table, n.tolist(), [[5, 3, 4], [0, 2]], [32, 160], None, None)
    check_out(outs[0][0], ref, mass)
    prefix.update([], [])                                  # nothing is shared any more
    graphs[0].replay()
    torch.cuda.synchronize()
    ref, mass, _ = reference(q, kp, vp, table, n.tolist(), [], [], None, None)
    check_out(outs[0][0], ref, mass)
    fresh = b200.SharedPrefix([[0, 1]], [16], 6)
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            f(q)
            b200.shared_prefix_attention(q, kp, vp, table, n, fresh)


def test_refusals(b200):
    case = ([(64, [3, 5])], [], 2, 4, 64, 16, torch.bfloat16, torch.bfloat16, "hnd", False)
    q, kp, vp, _, _, table, lens, members, tokens = made(case)
    n, prefix = on_device(lens), b200.SharedPrefix(members, tokens, 2)
    f = b200.shared_prefix_attention
    a = torch.ones(1, device="cuda")
    for call in (lambda: f(q[:, :7], kp, vp, table, n, prefix), lambda: f(q, kp, vp, table, n, prefix, scale=-1.0), lambda: f(q.float(), kp, vp, table, n, prefix),
                 lambda: f(q, kp, vp, table, n, prefix, k_amax=a, v_amax=a), lambda: f(q.half(), kp, vp, table, n, prefix), lambda: f(q[:1], kp, vp, table[:1], n[:1], prefix),
                 lambda: f(q, kp, vp, table[:, :3], n, prefix), lambda: f(q, kp.view(torch.uint8), vp.view(torch.uint8), table, n, prefix)):
        with pytest.raises(ValueError):
            call()
    plan = prefix.plan(8, 2)
    op = torch.ops.tensorrt.b200_shared_prefix_attention
    for call in (lambda: op(q, kp, vp, table, n, plan[:-1], 1, 2, None, None, 0.0), lambda: op(q, kp, vp, table, n, plan.cpu(), 1, 2, None, None, 0.0),
                 lambda: op(q, kp, vp, table, n, plan.long(), 1, 2, None, None, 0.0),
                 lambda: op(q, kp, vp, table, n, plan, 3, 2, None, None, 0.0), lambda: op(q, kp, vp, table, n, plan, 1, 0, None, None, 0.0),
                 lambda: f(q, kp, vp[:3], table, n, prefix), lambda: f(q, kp, vp, table.long(), n, prefix), lambda: f(q, kp, vp, table, n.cpu(), prefix)):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    assert f(q[:0], kp, vp, table[:0], n[:0], b200.SharedPrefix([], [], 0)).shape == (0, 8, 64)
    # a plan that was made for larger groups and has as many values: whom it has no room for is left out, nothing is written out of bounds
    assert op(q, kp, vp, table, n, plan, 1, 1, None, None, 0.0).shape == q.shape
