"""CPU checks of what continues a prompt several times: refusals that need no device, schemas, fake kernels, the plan of shared prefixes, and the pages
of a cache that forks, truncates and compacts, against a model of plain lists."""
import ctypes
import random

import pytest
import torch

from test_kv_cache import cache_of, host_cache, p  # noqa: F401

CTAS, ITEM_STEPS = 148, 2


def ints(v):
    return (ctypes.c_int32 * max(1, len(v)))(*v)


def make_plan(members, tokens, batch, n_q, n_kv, groups=None, largest=None):
    from tensorrt_b200 import _lib

    lib, flat, cu = _lib.load(), [b for m in members for b in m], [0]
    for m in members:
        cu.append(cu[-1] + len(m))
    groups = len(members) if groups is None else groups
    cu += cu[-1:] * (groups - len(members))
    sizes = batch, n_q, n_kv, groups, max([len(m) for m in members] + [0]) if largest is None else largest
    plan = torch.full((max(1, lib.b200q_shared_prefix_plan_values(*sizes)),), -7, dtype=torch.int32)
    rc = lib.b200q_shared_prefix_plan(ints(flat), ints(cu), ints(list(tokens) + [0] * (groups - len(tokens))), *sizes, plan.data_ptr())
    return rc, plan.tolist()


def walk(plan, members, tokens, batch, n_q, n_kv, groups):
    """Who works on which step of which item, read from the plan as the kernel reads it."""
    up, group, paired = (lambda n: (n + 3) // 4 * 4), n_q // n_kv, plan[0]
    order = 4 + 4 * batch
    ctas = order + up(batch) + 4 * groups
    items = ctas + 12 * CTAS
    tiles = lambda g: -(-tokens[g] // 128)  # noqa: E731
    steps = lambda g: tiles(g) if paired else -(-tiles(g) // 2)  # noqa: E731
    blocks = lambda g: -(-len(members[g]) * group // (256 if paired else 128)) if tokens[g] else 0  # noqa: E731
    line = [(g, h, b) for g in range(len(members)) for h in range(n_kv) for b in range(blocks(g))]
    done, longest = {}, 0
    for c in range(CTAS):
        left, item, g, h, b, step, _, _, first, n, t, leader = plan[ctas + 12 * c:ctas + 12 * c + 12]
        if left == 0:
            continue
        longest = max(longest, left + ITEM_STEPS)
        assert line[item] == (g, h, b) and (n, t, leader) == (len(members[g]), tokens[g], members[g][0])
        assert plan[order + first:order + first + n] == members[g]
        while left > 0:
            count = min(left, steps(line[item][0]) - step)
            assert count > 0
            for k in range(step, step + count):
                assert done.setdefault((item, k), c) == c
            left, step, item = left - count - ITEM_STEPS, 0, item + 1
    assert len(done) == sum(steps(g) for g, _, _ in line)
    for i, (g, _, _) in enumerate(line):
        of = [done[i, k] for k in range(steps(g))]
        assert of == sorted(of) and plan[items + 2 * i:items + 2 * i + 2] == [of[0], of[-1] - of[0] + 1]
    for g, m in enumerate(members):
        for place, b in enumerate(m):
            assert plan[4 + 4 * b] == tokens[g] and plan[4 + 4 * b + 3] == place * group
            if tokens[g]:
                assert line[plan[4 + 4 * b + 1]] == (g, 0, 0) and plan[4 + 4 * b + 2] == blocks(g)
    work = sum(steps(g) + ITEM_STEPS for g, _, _ in line)
    assert longest <= -(-work // CTAS) + max([steps(g) for g, _, _ in line], default=0) + ITEM_STEPS
    return paired, longest


@pytest.mark.parametrize("seed", range(20))
def test_plans_give_every_step_to_one_cta(b200, seed):
    r = random.Random(seed)
    n_kv = r.choice([1, 2, 4, 8, 12])
    n_q, sizes = n_kv * r.choice([1, 2, 4, 5, 8, 16]), [r.choice([1, 2, 3, 8, 40]) for _ in range(r.randint(1, 20))]
    batch = sum(sizes) + r.randint(0, 3)
    places = r.sample(range(batch), sum(sizes))
    members = [[places.pop() for _ in range(n)] for n in sizes]
    tokens = [r.choice([0, 1, 127, 128, 129, r.randint(1, 5000), r.randint(1, 100000)]) for _ in sizes]
    wide = r.random() < 0.5
    groups, largest = (batch, batch) if wide else (len(members), max(sizes))
    rc, plan = make_plan(members, tokens, batch, n_q, n_kv, groups, largest)
    assert rc == 0
    walk(plan, members, tokens, batch, n_q, n_kv, groups)


def test_plans_are_balanced(b200):
    for members, tokens, n_q, n_kv, want in (([list(range(64))], [8192], 64, 8, (1, 10)), ([list(range(16))], [100000], 64, 8, (0, 24)), ([[0, 1, 2, 3]], [496], 32, 8, (1, 3))):
        batch = len(members[0])
        rc, plan = make_plan(members, tokens, batch, n_q, n_kv)
        assert rc == 0 and walk(plan, members, tokens, batch, n_q, n_kv, 1) == want


def test_plans_that_are_refused(b200):
    bad = lambda members, tokens, batch=6, n_q=8, n_kv=2, **kw: make_plan(members, tokens, batch, n_q, n_kv, **kw)[0]  # noqa: E731
    assert bad([[0, 1], [2, 1]], [16, 16]) == bad([[0, 0]], [16]) == bad([[0, 6]], [16]) == bad([[-1, 1]], [16]) == -1
    assert bad([[0, 1]], [-1]) == bad([[0, 1, 2]], [5], largest=2) == bad([[0, 1]], [5], n_q=7) == bad([[0, 1]], [5], n_kv=0) == -1
    assert bad([[0, 1]], [5], batch=70000) == bad([[0, 1]], [5], groups=7) == bad([[0, 1]], [5], largest=7) == -1
    assert bad([[0, 1]], [5]) == bad([[]], [5]) == bad([], []) == 0
    with pytest.raises(ValueError):
        b200.SharedPrefix([[0, 1], [1, 2]], [8, 8], 4, device="cpu")
    for members, tokens, kw in (([[0, 4]], [8], {}), ([[0, 1]], [8, 8], {}), ([[0, 1]], [-8], {}), ([[0, 1]], [1 << 31], {}), ([[0, 1]], [8], dict(groups=0)),
                                ([[0, 1, 2]], [8], dict(groups=1, largest=2)), ([[0, 1]], [8], dict(groups=5)), ([[0, 1]], [8], dict(largest=5))):
        with pytest.raises(ValueError):
            b200.SharedPrefix(members, tokens, 4, device="cpu", **kw)
    prefix = b200.SharedPrefix([[0, 1], [2], [3]], [8, 100, 0], 4, device="cpu")       # nothing is shared by one, nor where there is nothing
    assert (prefix.groups, prefix.largest, prefix.tokens) == (1, 2, 8)
    plan = prefix.plan(8, 2)
    at = plan.data_ptr()
    prefix.update([[2, 3]], [640])
    assert prefix.plan(8, 2).data_ptr() == at and plan.tolist() == make_plan([[2, 3]], [640], 4, 8, 2)[1]      # in place
    with pytest.raises(ValueError):
        prefix.update([[0, 1], [2, 3]], [8, 8])
    assert b200.SharedPrefix([], [], 0, device="cpu").plan(8, 2).numel() == 0


def test_arguments_that_are_refused(b200, p):  # noqa: F811
    from tensorrt_b200 import _lib

    lib, i64 = _lib.load(), ctypes.c_int64
    pools, strides = (ctypes.c_void_p * 2)(p, p + 1024), (i64 * 3)(2048, 1024, 128)
    copy = lambda pools=pools, n=2, pages=4, heads=2, size=8, row=128, s=strides, src=(0,), dst=(1,), rows=None, pairs=None: lib.b200q_paged_copy(  # noqa: E731
        pools, n, pages, heads, size, row, s, ints(src), ints(dst), None if rows is None else ints(rows), len(src) if pairs is None else pairs, None)
    assert copy(src=(4,)) == copy(src=(-1,)) == copy(dst=(4,)) == copy(dst=(0,)) == copy(src=(0, 0), dst=(1, 1)) == copy(src=(0, 1), dst=(1, 2)) == -1
    many = list(range(20))
    assert copy(pages=64, src=many, dst=[20 + i % 19 for i in many]) == copy(pages=64, src=many, dst=[19 + i for i in many]) == -1
    assert copy(rows=(9,)) == copy(rows=(-1,)) == copy(pools=None) == copy(s=None) == copy(n=-1) == copy(pairs=-1) == copy(pages=-1, pairs=0) == copy(heads=0) == -1
    assert copy(size=0) == copy(row=0) == copy(row=512) == copy(pairs=5) == copy(pools=(ctypes.c_void_p * 2)(p, None)) == -1
    assert copy(row=120) == copy(s=(i64 * 3)(2048, 1024, 120)) == copy(s=(i64 * 3)(-2048, 1024, 128)) == copy(pools=(ctypes.c_void_p * 2)(p, p + 8)) == -2
    assert copy(n=0) == copy(pairs=0) == copy(src=(), dst=()) == 0            # nothing to copy: no device is needed

    c, s2, big = ctypes.byref(cache_of(p)), (i64 * 2)(128, 64), 1 << 40
    attend = lambda q=p, dt=2, s=s2, cc=c, b=3, hq=4, plan=p, groups=1, largest=2, scale=1.0, out=p, aw=p, an=big, ws=p, n=big: lib.b200q_shared_prefix_attention(  # noqa: E731
        q, dt, s, cc, p, 4, 4, p, b, hq, plan, groups, largest, scale, out, aw, an, ws, n, None)
    assert attend(q=None) == attend(out=None) == attend(s=None) == attend(plan=None) == attend(hq=3) == attend(hq=0) == attend(dt=1) == attend(dt=0) == -1
    assert attend(scale=float("nan")) == attend(groups=-1) == attend(groups=4) == attend(largest=4) == attend(largest=0) == attend(b=0) == -1
    assert attend(cc=ctypes.byref(cache_of(p, D=24))) == attend(cc=ctypes.byref(cache_of(p, dtype=3))) == -1
    assert attend(q=p + 8) == attend(s=(i64 * 2)(128, 60)) == attend(ws=p + 4) == attend(aw=p + 4) == attend(plan=p + 4) == -2
    assert attend(ws=None) == attend(n=8) == attend(aw=None) == attend(an=8) == -5
    assert attend(groups=0, b=0) == 0
    assert lib.b200q_shared_prefix_workspace_bytes(3, 4, 2, 64, 1, 2) > 0 == lib.b200q_shared_prefix_workspace_bytes(3, 5, 2, 64, 1, 2)

    score = lambda x=p, dt=2, rows=3, v=50, stride=50, t=p, tb=8, scale=1.0, lp=p, e=p, top=4, tl=p, tt=p: lib.b200q_token_log_probs(  # noqa: E731
        x, dt, rows, v, stride, t, tb, scale, lp, e, top, tl, tt, None)
    assert score(x=None) == score(dt=3) == score(rows=-1) == score(v=0) == score(stride=-1) == score(t=None) == score(lp=None) == score(tb=2) == -1
    assert score(top=-1) == score(top=65) == score(v=3, top=4) == score(tl=None) == score(tt=None) == -1
    assert score(scale=0.0) == score(scale=-1.0) == score(scale=float("nan")) == score(scale=float("inf")) == -1
    assert score(x=p + 1) == score(t=p + 4) == score(x=p + 2, dt=0) == -2
    assert score(rows=0) == 0


def test_schemas_and_fake_kernels(b200):
    ops = torch.ops.tensorrt
    written = {name: [a.name for a in getattr(ops, name).default._schema.arguments if a.alias_info and a.alias_info.is_write]
               for name in ("b200_paged_copy", "b200_shared_prefix_attention", "b200_token_log_probs")}
    assert written == {"b200_paged_copy": ["k_pages", "v_pages"], "b200_shared_prefix_attention": [], "b200_token_log_probs": []}
    m = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    kp = m(10, 2, 16, 64)
    prefix = b200.SharedPrefix([[0, 1]], [16], 3, device="cpu")
    out = b200.shared_prefix_attention(m(3, 8, 64), kp, kp, m(3, 4, dtype=torch.int32), m(3, dtype=torch.int32), prefix)
    assert out.shape == (3, 8, 64) and out.dtype == torch.bfloat16
    assert b200.paged_copy([kp], [kp], [0], [1]) is None
    got = b200.token_log_probs(m(2, 5, 100), m(2, 5, dtype=torch.int64), top=7)
    assert got.log_probs.shape == got.entropy.shape == (2, 5) and got.top_log_probs.shape == got.top_tokens.shape == (2, 5, 7)
    assert got.top_tokens.dtype == torch.int32 and got.entropy.dtype == torch.float32
    for bad in (dict(batch=4), dict(width=0)):
        with pytest.raises(ValueError):
            n, w = bad.get("batch", 3), bad.get("width", 4)
            b200.shared_prefix_attention(m(n, 8, 64), kp, kp, m(n, w, dtype=torch.int32), m(n, dtype=torch.int32), prefix)
    with pytest.raises(ValueError):
        b200.shared_prefix_attention(m(3, 7, 64), kp, kp, m(3, 4, dtype=torch.int32), m(3, dtype=torch.int32), prefix)


def test_cpu_tensors_are_refused(b200):
    x, pages, table, n = torch.zeros(2, 2, 64).bfloat16(), torch.zeros(4, 1, 16, 64).bfloat16(), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    prefix = b200.SharedPrefix([[0, 1]], [16], 2, device="cpu")
    for call in (lambda: b200.paged_copy(pages, pages, [0], [1]), lambda: b200.token_log_probs(torch.zeros(2, 50)),
                 lambda: b200.shared_prefix_attention(x, pages, pages, table, n, prefix)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


# ----------------------------------------------------------------------------- the pages of a cache that forks
def copy_on_the_host(k_pages, v_pages, src, dst, rows=None):
    assert len(set(dst)) == len(dst) and not set(dst) & set(src)
    for pool in k_pages + v_pages:
        for i, (a, b) in enumerate(zip(src, dst)):
            n = pool.shape[2] if rows is None else rows[i]
            pool[b, :, :n] = pool[a, :, :n]


class Model:
    """A cache on the host whose tokens are numbers, written to where `append` would, beside plain lists of them."""

    def __init__(self, b200, monkeypatch, **kw):
        import tensorrt_b200.kv_cache as kv

        monkeypatch.setattr(kv, "paged_copy", copy_on_the_host)
        self.cache = host_cache(b200, **{**dict(batch=5, pages=40, max_tokens=60, page_size=4, dtype=torch.float16), **kw})
        self.texts, self.next = [[] for _ in range(self.cache.batch)], 1

    def grow(self, new):
        c = self.cache
        c.grow(new)
        for b, n in enumerate(new):
            for _ in range(n):
                t = len(self.texts[b])
                self.texts[b].append(self.next % 2000)
                page = c._pages[b][t // c.page_size]
                assert c._uses[page] == 1                  # nobody writes to what others read
                for pool in c.k + c.v:
                    pool[page, :, t % c.page_size] = self.next % 2000
                self.next += 1
        self.check()

    def check(self):
        c = self.cache
        assert c.tokens() == [len(t) for t in self.texts] == c.lens.tolist()
        uses = [0] * len(c._uses)
        for b, text in enumerate(self.texts):
            assert c.table[b, :len(c._pages[b])].tolist() == c._pages[b] and (c.table[b, len(c._pages[b]):] == -1).all()
            for page in c._pages[b]:
                uses[page] += 1
            for pool in c.k + c.v:
                for t, token in enumerate(text):
                    assert (pool[c._pages[b][t // c.page_size], :, t % c.page_size] == token).all()
        assert uses == c._uses and sorted(c._free) == [p for p, n in enumerate(uses) if n == 0]
        if c._shares:
            members, tokens = c._prefix.last
            for m, t in zip(members, tokens):
                assert t % c.page_size == 0 and len(m) > 1 and all(self.texts[b][:t] == self.texts[m[0]][:t] for b in m)
                assert all(c._pages[b][:t // c.page_size] == c._pages[m[0]][:t // c.page_size] for b in m)


@pytest.fixture
def model(b200, monkeypatch):
    def update(self, members, tokens, inner=b200.SharedPrefix.update):
        self.last = members, tokens
        inner(self, members, tokens)

    import tensorrt_b200.kv_cache as kv

    monkeypatch.setattr(b200.SharedPrefix, "update", update)
    monkeypatch.setattr(kv, "_SHARED_KEYS", 1)
    return lambda **kw: Model(b200, monkeypatch, **kw)


@pytest.mark.parametrize("seed", range(12))
def test_forks_cuts_and_moves_keep_every_text(model, seed):
    r, m = random.Random(seed), model()
    c = m.cache
    for _ in range(40):
        kind = r.choice(["grow", "grow", "grow", "step", "fork", "fork", "truncate", "release", "compact", "resize", "reserve"])
        before = m.texts
        try:
            if kind == "grow":
                m.grow([r.choice([0, 0, 1, 3, 9]) if len(t) < 45 else 0 for t in m.texts])
            elif kind == "step":
                m.grow([int(len(t) < 55) for t in m.texts])
            elif kind == "reserve":
                c.reserve([min(60, len(t) + r.choice([0, 6])) for t in m.texts])
            elif kind == "fork":
                parents = [r.randrange(5) if r.random() < 0.6 else b for b in range(5)]
                m.texts = [list(m.texts[p]) for p in parents]
                c.fork(parents)
            elif kind == "truncate":
                m.texts = [t[:r.randint(0, len(t))] if r.random() < 0.3 else t for t in m.texts]
                c.truncate([len(t) for t in m.texts])
            elif kind == "release":
                b = r.randrange(5)
                m.texts[b] = []
                c.release(b)
            elif kind == "compact":
                used = c.compact()
                assert used == len(c._uses) - c.free_pages() and all(c._uses[:used]) and not any(c._uses[used:])
            else:
                c.resize(max(len(c._uses) - c.free_pages(), r.randint(20, 50)))
        except RuntimeError as e:
            assert "are needed" in str(e)
            m.texts = before
        m.check()


def test_a_page_is_copied_for_all_but_the_last_that_grow(model, monkeypatch):
    import tensorrt_b200.kv_cache as kv

    m, copies = model(weights=False), []
    monkeypatch.setattr(kv, "paged_copy", lambda k, v, src, dst, rows: (copies.append((src, rows)), copy_on_the_host(k, v, src, dst, rows)))
    m.grow([10, 0, 0, 0, 0])
    free = m.cache.free_pages()
    m.texts = [list(m.texts[0]) for _ in range(5)]
    m.cache.fork([0] * 5)
    assert m.cache.free_pages() == free and not copies       # nothing is copied yet
    m.grow([1, 1, 0, 0, 0])
    assert [len(s) for s, _ in copies] == [2] and copies[0][1] == [2, 2] and m.cache.free_pages() == free - 2
    m.grow([0, 0, 1, 1, 1])
    assert len(copies[1][0]) == 2 and m.cache.free_pages() == free - 4
    assert m.cache._shares and m.cache._prefix.last == ([[0, 1, 2, 3, 4]], [8])
    with pytest.raises(RuntimeError, match="are needed"):
        m.cache.reserve([60] * 5)
    m.check()


def test_eviction_of_shared_pages(b200, model, monkeypatch):
    import tensorrt_b200.kv_cache as kv

    m = model(weights=True)
    c = m.cache

    def evict(k, v, table, lens, weights, out, *, keep, recent, sinks):       # the first `keep` tokens, into fresh pages
        for b, t in enumerate(m.texts):
            for i in range(min(keep, len(t))):
                for pool in (k, v):
                    pool[out[b, i // c.page_size], :, i % c.page_size] = t[i]
        return torch.zeros(5, 2, keep, dtype=torch.int32), lens.clamp(max=keep), torch.zeros_like(weights)

    monkeypatch.setattr(kv, "paged_evict", evict)
    m.grow([12, 5, 0, 0, 0])
    for w in c.weights:
        w[0] += 1.0
    m.texts = [list(m.texts[p]) for p in (0, 1, 0, 0, 1)]
    c.fork([0, 1, 0, 0, 1])
    assert all((w[2] == 1).all() and not w[1].any() for w in c.weights)
    c.evict(7)
    m.texts = [t[:7] for t in m.texts]
    m.check()
    c.truncate([6, 5, 0, 7, 2])
    m.texts = [t[:n] for t, n in zip(m.texts, [6, 5, 0, 7, 2])]
    m.check()
    m.grow([1, 1, 1, 1, 1])


@pytest.mark.parametrize("call", [lambda c: c.fork([0, 1]), lambda c: c.fork([0, 1, 2, 3, 5]), lambda c: c.fork([0, 1, 2, 3, -1]), lambda c: c.truncate([3] * 4),
                                  lambda c: c.truncate([11, 0, 0, 0, 0]), lambda c: c.truncate([-1, 0, 0, 0, 0]), lambda c: c.resize(2), lambda c: c.resize(0)])
def test_refused_calls_change_nothing(model, call):
    m = model()
    m.grow([10, 2, 0, 0, 0])
    with pytest.raises(ValueError):
        call(m.cache)
    m.check()


def test_a_refused_copy_changes_nothing(b200, monkeypatch):
    import tensorrt_b200.kv_cache as kv

    def refuse(*_):
        raise RuntimeError("no device")

    monkeypatch.setattr(kv, "paged_copy", refuse)
    cache = host_cache(b200)
    cache.grow([10, 0, 0])
    cache.fork([0, 0, 0])
    before = cache.tokens(), cache.table.tolist(), list(cache._free), list(cache._uses), [list(x) for x in cache._pages]
    with pytest.raises(RuntimeError, match="no device"):
        cache.grow([1, 1, 1])
    assert (cache.tokens(), cache.table.tolist(), list(cache._free), list(cache._uses), [list(x) for x in cache._pages]) == before


def test_released_parents(model):
    m = model()
    m.grow([5, 4, 0, 0, 0])
    m.cache.release(1)
    m.texts[1] = []
    m.texts = [list(m.texts[p]) for p in (1, 1, 0, 3, 4)]
    m.cache.fork([1, 1, 0, 3, 4])                            # what goes on from a released sequence is released
    m.check()
    m.cache.grow_all()
    assert m.cache.tokens() == [0, 0, 6, 1, 1]


@pytest.mark.parametrize("n,shares", [((1 << 17) // 6, False), ((1 << 17) // 6 + 8, True)])
def test_what_is_shared_must_be_worth_it(b200, monkeypatch, n, shares):
    """(sequences - 1) x tokens in full pages x kv heads, against 2^17."""
    cache = b200.PagedKvCache(1, 4, 2, 16, pages=6000, max_tokens=n + 8, page_size=8, device="cpu")
    cache.grow([n, 0, 0, 0])
    assert not cache._shares
    cache.fork([0] * 4)
    assert cache._shares == shares
    cache.release(1)
    assert not cache._shares and cache._prefix._lists[0][:] == [0, 2, 3]      # a captured step goes by the plan all the same
    cache.release(2), cache.release(0)
    assert cache._prefix.tokens == 0


def test_a_plan_is_at_hand_for_a_first_step_that_is_captured(b200, monkeypatch):
    """Once a step has told how many query heads there are, the plan is made where a fork changes it."""
    import tensorrt_b200.kv_cache as kv

    monkeypatch.setattr(kv, "paged_attention", lambda q, *a, **kw: q)
    cache = b200.PagedKvCache(1, 4, 2, 16, pages=60, max_tokens=64, page_size=8, device="cpu")
    cache.grow([20, 1, 0, 0])
    cache.attend(0, torch.zeros(4, 6, 16))
    cache.fork([0, 1, 0, 0])
    assert list(cache._prefix._plans) == [(6, 2)]
    before = cache._prefix.plan(6, 2).clone()
    cache.truncate([9, 1, 9, 9])
    assert cache._prefix.tokens == 8 and not torch.equal(before, cache._prefix._plans[6, 2])


def test_nothing_is_appended_behind_a_fork_or_a_cut_without_room(b200, monkeypatch):
    """The newest rows are shared then, or gone."""
    rows = torch.zeros(3, 2, 16, dtype=torch.bfloat16)
    for change in (lambda c: c.fork([0, 0, 1]), lambda c: c.truncate([3, 2, 1])):
        cache = b200.PagedKvCache(1, 3, 2, 16, pages=60, max_tokens=64, page_size=8, device="cpu")
        cache.grow([5, 4, 3])
        change(cache)
        with pytest.raises(ValueError, match="expected the rows of 0 new tokens"):
            cache.append(0, rows, rows)


def test_a_plan_is_not_updated_in_a_capture(b200, monkeypatch):
    prefix = b200.SharedPrefix([[0, 1]], [16], 4, device="cpu")
    prefix.plan(4, 2)
    prefix.device = torch.device("cuda")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="outside the capture"):
        prefix.update([[0, 1]], [8])
