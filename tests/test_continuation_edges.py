"""CPU checks of continuations at their edges: groups that hold nothing, calls that fail on the way."""
import random

import pytest
import torch

from test_continuations import CTAS, ITEM_STEPS, make_plan, model  # noqa: F401


@pytest.mark.parametrize("batch,members,tokens", [(4, [], []), (4, [[0]], [64]), (4, [[1, 2]], [0]), (1, [], []), (0, [], [])])
def test_an_update_where_nothing_is_shared(b200, batch, members, tokens):
    prefix = b200.SharedPrefix(members, tokens, batch, device="cpu")
    plan = prefix.plan(8, 2)
    assert prefix.groups == 0 and plan.numel() == 0
    for now in ((members, tokens), ([], []), ([[0]] * min(batch, 1), [9] * min(batch, 1))):
        prefix.update(*now)
        assert prefix.tokens == 0 and prefix.plan(8, 2) is plan
    if batch > 1:
        with pytest.raises(ValueError):
            prefix.update([[0, 1]], [8])
        assert prefix.tokens == 0


@pytest.mark.parametrize("largest", [None, 0, 1])
def test_room_for_groups_of_nobody(b200, largest):
    """Groups of up to one sequence hold nothing that is shared: a call has to be possible all the same."""
    prefix = b200.SharedPrefix([], [], 4, device="cpu", groups=2, largest=largest)
    assert prefix.groups == 0 and prefix.plan(8, 2).numel() == 0
    prefix.update([[1]], [50])
    with pytest.raises(ValueError):
        prefix.update([[0, 1]], [50])


@pytest.mark.parametrize("pages", [60, 14])
@pytest.mark.parametrize("nth", [0, 1, 2, 3])
def test_no_memory_for_the_pools_of_another_size(model, monkeypatch, pages, nth):  # noqa: F811
    """A cache that could not be given all of its new pools has the smaller of the two numbers of pages in every layer, and goes on."""
    m = model(pages=40, layers=2)
    c = m.cache
    m.grow([10, 2, 0, 5, 0])
    c.release(3)
    m.texts = [m.texts[0], m.texts[1], list(m.texts[0]), [], list(m.texts[0])]
    c.fork([0, 1, 0, 3, 0])
    made, zeros = [0], torch.zeros

    def no_room(*a, **kw):
        made[0] += 1
        if made[0] > nth:
            raise torch.OutOfMemoryError("no room")
        return zeros(*a, **kw)

    monkeypatch.setattr(torch, "zeros", no_room)
    with pytest.raises(torch.OutOfMemoryError):
        c.resize(pages)
    monkeypatch.setattr(torch, "zeros", zeros)
    assert [p.shape[0] for p in c.k + c.v] == [min(40, pages)] * 4 and len(c._uses) == min(40, pages)
    m.check()
    m.grow([2, 3, 1, 0, 1])                                  # with copies of the page that is shared and not full
    c.compact()
    m.check()
    c.resize(30)
    assert [p.shape[0] for p in c.k + c.v] == [30] * 4
    m.grow([1, 1, 1, 4, 1])


@pytest.mark.parametrize("n,n_kv,tokens,codes,shares", [
    (64, 8, 256, False, False), (64, 8, 272, False, False), (64, 8, 400, False, True), (16, 8, 1104, False, False), (16, 8, 1648, False, True), (64, 2, 1056, False, False),
    (128, 8, 144, False, True), (8, 8, 2352, False, True), (2, 8, 32752, False, False), (2, 8, 32784, False, True), (8, 8, 2352, True, False), (8, 8, 4688, True, True), (64, 8, 528, True, False),
    (64, 8, 800, True, True), (256, 8, 144, True, True), (256, 8, 112, True, False), (2, 1, 800000, True, False), (3, 1, 140000, True, True)])
def test_the_choice_goes_by_what_was_measured(b200, n, n_kv, tokens, codes, shares):
    amax = dict(dtype=torch.float8_e4m3fn, k_amax=[torch.ones(1)], v_amax=[torch.ones(1)]) if codes else {}
    cache = b200.PagedKvCache(1, n, n_kv, 16, pages=1, max_tokens=tokens + 16, page_size=16, device="cpu", **amax)
    cache._uses, cache._free = [0] * (tokens // 16 + 1), list(range(tokens // 16 + 1))      # numbers of pages only
    cache.grow([tokens] + [0] * (n - 1))
    cache.fork([0] * n)
    assert cache._shares == shares


def test_the_choice_goes_by_the_query_heads_too(b200, monkeypatch):
    import tensorrt_b200.kv_cache as kv

    calls = []
    for name in ("shared_prefix_attention", "paged_attention"):
        monkeypatch.setattr(kv, name, lambda q, *a, name=name, **kw: calls.append(name))
    one = [torch.ones(1)]
    cache = b200.PagedKvCache(1, 64, 8, 16, pages=1, max_tokens=1000, page_size=16, device="cpu", dtype=torch.float8_e4m3fn, k_amax=one, v_amax=one)
    cache._uses, cache._free = [0] * 70, list(range(70))
    cache.grow([800] + [0] * 63)
    cache.fork([0] * 64)
    for n_q in (32, 64, 8, 64):
        cache.attend(0, torch.zeros(64, n_q, 16))
        cache.fork([1] + [0] * 63)
        cache.attend(0, torch.zeros(64, n_q, 16))
    assert calls == ["shared_prefix_attention"] * 2 + ["paged_attention"] * 2 + ["shared_prefix_attention"] * 2 + ["paged_attention"] * 2


def places_of_parts(plan, members, tokens, batch, n_q, n_kv, groups, items_most):
    """Rows of the scratch that each CTA writes, as the kernel finds them, and those that the join reads for each row of an item, as it finds them."""
    up, group, paired = (lambda n: (n + 3) // 4 * 4), n_q // n_kv, plan[0]
    ctas = 4 + 4 * batch + up(batch) + 4 * groups
    items = ctas + 12 * CTAS
    places = items + up(2 * items_most)
    size = 256 if paired else 128
    line = [(g, h, b) for g in range(len(members)) if tokens[g] for h in range(n_kv) for b in range(-(-len(members[g]) * group // size))]
    tiles = lambda g: -(-tokens[g] // 128)  # noqa: E731
    steps = lambda g: tiles(g) if paired else -(-tiles(g) // 2)  # noqa: E731
    written, read = {}, {}
    for c in range(CTAS):
        left, item, _, _, _, step = plan[ctas + 12 * c:ctas + 12 * c + 6]
        while left > 0:
            g, h, b = line[item]
            rows = len(members[g]) * group
            half_rows = [min(rows - b * size - (s * 128 if paired else 0), 128) for s in range(2)]
            whole = min(rows - b * size, 256) if paired else 2 * half_rows[0]
            for s in range(2):
                for r in range(half_rows[s]):
                    at = plan[places + 2 * item] + c * whole + s * half_rows[0] + r
                    assert at >= 0 and at not in written
                    written[at] = item, b * size + (s * 128 if paired else 0) + r
            left, step, item = left - min(left, steps(g) - step) - ITEM_STEPS, 0, item + 1
    for i, (g, h, b) in enumerate(line):
        base, rows = plan[places + 2 * i:places + 2 * i + 2]
        c0, n = plan[items + 2 * i:items + 2 * i + 2]
        for row in range(b * size, min((b + 1) * size, len(members[g]) * group)):
            apart = rows if paired else rows // 2
            for k in range(n if paired else 2 * n):
                read[base + c0 * rows + (row & 128 if paired else 0) + (row & 127) + k * apart] = i, row
    assert written == read
    return max(written, default=-1) + 1


@pytest.mark.parametrize("seed", range(24))
def test_parts_have_places_of_their_own(b200, seed):
    r = random.Random(seed)
    n_kv = r.choice([1, 2, 8])
    n_q, sizes = n_kv * r.choice([1, 2, 5, 8, 16]), [r.choice([1, 2, 3, 8, 40]) for _ in range(r.randint(1, 20))]
    batch = sum(sizes) + r.randint(0, 3)
    names = r.sample(range(batch), sum(sizes))
    members = [[names.pop() for _ in range(n)] for n in sizes]
    tokens = [r.choice([0, 1, 127, 128, 129, r.randint(1, 5000), r.randint(1, 100000)]) for _ in sizes]
    groups, largest = (batch, batch) if r.random() < 0.5 else (len(members), max(sizes))
    rc, plan = make_plan(members, tokens, batch, n_q, n_kv, groups, largest)
    assert rc == 0
    group = n_q // n_kv
    items = n_kv * min(groups * -(-largest * group // 128), batch * group // 128 + groups)
    rows = places_of_parts(plan, members, tokens, batch, n_q, n_kv, groups, items)
    from tensorrt_b200 import _lib

    room = 2 * min(groups * largest, batch) * n_q + CTAS * min(2 * largest * group, 256)
    assert rows <= room
    own = _lib.load().b200q_shared_prefix_workspace_bytes(batch, n_q, n_kv, 128, 0, 0)      # what there is beside parts and their sums
    assert room * (512 + 8) <= _lib.load().b200q_shared_prefix_workspace_bytes(batch, n_q, n_kv, 128, groups, largest) - own <= room * (512 + 8) + 1024


@pytest.mark.parametrize("batch,n_q,n_kv,most", [(64, 64, 8, 45), (256, 64, 8, 90), (1024, 64, 8, 260), (1024, 32, 32, 260)])
def test_the_scratch_of_a_cache_goes_by_its_batch(b200, batch, n_q, n_kv, most):
    """A cache has room for any groups: megabytes, and no more of them than its sequences' rows and a tile of each CTA need."""
    from tensorrt_b200 import _lib

    assert _lib.load().b200q_shared_prefix_workspace_bytes(batch, n_q, n_kv, 128, batch // 2, batch) <= most << 20


@pytest.mark.parametrize("n,tokens,codes,shares", [(4, 22000, False, False), (4, 65000, False, False), (16, 2191, False, True), (64, 518, False, True), (4, 65000, True, False),
                                                   (16, 43680, True, False), (64, 1036, True, False), (64, 3115, True, True), (256, 259, True, True)])
def test_the_choice_goes_by_the_rows_of_a_page_too(b200, n, tokens, codes, shares):
    """Pages of seven rows, which no tensor map takes."""
    amax = dict(dtype=torch.float8_e4m3fn, k_amax=[torch.ones(1)], v_amax=[torch.ones(1)]) if codes else {}
    cache = b200.PagedKvCache(1, n, 8, 16, pages=1, max_tokens=tokens + 16, page_size=7, device="cpu", **amax)
    cache._uses, cache._free = [0] * (tokens // 7 + 1), list(range(tokens // 7 + 1))
    cache.grow([tokens] + [0] * (n - 1))
    cache.fork([0] * n)
    assert cache._shares == shares


@pytest.mark.parametrize("groups,per,tokens,codes,shares", [(16, 4, 336, False, False), (16, 4, 528, False, True), (64, 4, 80, False, False), (64, 4, 160, False, True), (16, 2, 2048, False, False),
                                                           (16, 2, 3200, False, True), (16, 4, 672, True, False), (16, 4, 1040, True, True), (64, 2, 1280, True, False)])
def test_the_choice_goes_by_the_groups_too(b200, groups, per, tokens, codes, shares):
    amax = dict(dtype=torch.float8_e4m3fn, k_amax=[torch.ones(1)], v_amax=[torch.ones(1)]) if codes else {}
    n, pages = groups * per, groups * (tokens // 16)
    cache = b200.PagedKvCache(1, n, 8, 16, pages=1, max_tokens=tokens + 16, page_size=16, device="cpu", **amax)
    cache._uses, cache._free = [0] * pages, list(range(pages))
    cache.grow([0 if b % per else tokens for b in range(n)])
    cache.fork([b - b % per for b in range(n)])
    assert cache._shares == shares


def test_a_plan_made_in_inference_mode_can_be_updated(b200):
    """A step in inference mode, the fork behind it outside."""
    prefix = b200.SharedPrefix([[0, 1]], [16], 4, device="cpu")
    with torch.inference_mode():
        plan = prefix.plan(8, 2)
    prefix.update([[2, 3]], [640])
    assert prefix.plan(8, 2) is plan and plan.tolist() == make_plan([[2, 3]], [640], 4, 8, 2)[1]
    with torch.inference_mode():
        prefix.update([[0, 3]], [64])
    assert plan.tolist() == make_plan([[0, 3]], [64], 4, 8, 2)[1]


def test_nothing_is_appended_behind_an_eviction_without_room(b200, monkeypatch):
    import tensorrt_b200.kv_cache as kv

    monkeypatch.setattr(kv, "paged_evict", lambda k, v, table, lens, weights, out, *, keep, recent, sinks: (torch.zeros(3, 2, keep, dtype=torch.int32), lens.clamp(max=keep), weights))
    cache = b200.PagedKvCache(1, 3, 2, 16, pages=60, max_tokens=64, page_size=8, weights=True, device="cpu")
    cache.grow([5, 4, 3])
    cache.evict(2)
    rows = torch.zeros(12, 2, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="expected the rows of 0 new tokens"):
        cache.append(0, rows, rows)
