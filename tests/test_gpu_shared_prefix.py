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
