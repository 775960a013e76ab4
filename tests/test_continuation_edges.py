"""CPU checks of continuations at their edges: groups that hold nothing, calls that fail on the way."""
import pytest
import torch

from test_continuations import model  # noqa: F401


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
    (128, 8, 144, False, True), (8, 8, 2352, False, True), (2, 8, 16400, False, True), (8, 8, 2352, True, False), (8, 8, 4688, True, True), (64, 8, 528, True, False),
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
