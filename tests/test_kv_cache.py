"""CPU checks of the paged key-value cache's boundary: refusals that need no device, schemas, fake kernels."""
import ctypes

import pytest
import torch


def cache_of(p, **kw):
    from tensorrt_b200 import _lib

    c = _lib.PagedCache(p, p, 2, 16, 4, 2, 64, (2 * 16 * 64, 16 * 64, 64), (2 * 16 * 64, 16 * 64, 64), None, None, 0)
    for k, v in kw.items():
        if k.endswith("strides"):
            v = (ctypes.c_int64 * 3)(*v)
        setattr(c, k, v)
    return c


@pytest.fixture
def p():
    buf = ctypes.create_string_buffer(8192)
    yield (ctypes.addressof(buf) + 255) & ~255


BAD_CACHES = [(dict(dtype=0), -1), (dict(dtype=1), -1), (dict(dtype=3), -1), (dict(dtype=9), -1), (dict(page_size=0), -1), (dict(page_size=-4), -1),
              (dict(num_pages=-1), -1), (dict(num_pages=1 << 33), -1), (dict(heads=0), -1), (dict(D=0), -1), (dict(D=24), -1), (dict(D=144), -1),
              (dict(k_pages=None), -1), (dict(v_pages=None), -1), (dict(k_strides=(2048, 1024, 60)), -2), (dict(v_strides=(2048, -1024, 64)), -2)]


@pytest.mark.parametrize("change,status", BAD_CACHES, ids=str)
def test_caches_that_are_refused(b200, p, change, status):
    from tensorrt_b200 import _lib

    lib, i64 = _lib.load(), ctypes.c_int64
    c = ctypes.byref(cache_of(p, **change))
    s4, s2 = (i64 * 4)(128, 64, 128, 64), (i64 * 2)(128, 64)
    assert lib.b200q_paged_append(p, p, 2, s4, 3, None, c, p, 4, 4, p, 3, None) == status
    assert lib.b200q_paged_attention(p, 2, s2, c, p, 4, 4, p, 3, 4, 1.0, 0, 0, p, None, 0, p, 1 << 40, None, 0, None) == status
    if change.get("dtype") not in (1, 3):               # rows that only move need neither a type in common nor a range
        assert lib.b200q_paged_evict(c, p, 4, 4, p, p, 64, p, 4, 4, 3, 32, 2, 2, p, p, p + 16, None) == status


def test_arguments_that_are_refused(b200, p):
    from tensorrt_b200 import _lib

    lib, i64 = _lib.load(), ctypes.c_int64
    c = ctypes.byref(cache_of(p))
    codes = lambda **kw: ctypes.byref(cache_of(p, **{**dict(dtype=3, k_amax=p, v_amax=p, amax_numel=1), **kw}))  # noqa: E731
    s4, s2 = (i64 * 4)(128, 64, 128, 64), (i64 * 2)(128, 64)
    append = lambda k=p, v=p, dt=2, s=s4, t=3, cu=None, cc=c, tab=p, width=4, lens=p, b=3: lib.b200q_paged_append(  # noqa: E731
        k, v, dt, s, t, cu, cc, tab, 4, width, lens, b, None)
    assert append(k=None) == append(v=None) == append(s=None) == append(lens=None) == append(tab=None) == append(cc=None) == -1
    assert append(dt=0) == append(dt=3) == append(t=2) == append(t=-1) == append(width=-1) == append(b=-1) == -1
    assert append(k=p + 2) == append(s=(i64 * 4)(128, 60, 128, 64)) == -2
    assert append(cc=codes(amax_numel=3)) == append(cc=codes(k_amax=None)) == append(cc=codes(v_amax=None)) == -1
    assert append(t=0, cu=p) == append(width=0) == 0     # nothing to write: no device is needed

    big = 1 << 40
    attend = lambda q=p, dt=2, s=s2, cc=c, b=3, hq=4, scale=1.0, sinks=0, out=p, w=None, wl=0, ws=p, n=big, sc=None, sn=0: lib.b200q_paged_attention(  # noqa: E731
        q, dt, s, cc, p, 4, 4, p, b, hq, scale, 0, sinks, out, w, wl, ws, n, sc, sn, None)
    assert attend(q=None) == attend(out=None) == attend(s=None) == attend(hq=3) == attend(hq=0) == attend(sinks=-1) == attend(dt=1) == -1
    assert attend(scale=float("nan")) == attend(w=p, wl=-1, sc=p, sn=big) == -1
    assert attend(q=p + 8) == attend(s=(i64 * 2)(128, 60)) == attend(ws=p + 4) == -2
    assert attend(ws=None) == attend(n=8) == attend(w=p, wl=64) == attend(w=p, wl=64, sc=p, sn=8) == -5
    assert attend(b=0) == 0

    evict = lambda w=p, wl=64, out=p, width=4, b=3, keep=32, recent=2, sinks=2, kept=p, lens=p, nw=p + 16: lib.b200q_paged_evict(  # noqa: E731
        c, p, 4, 4, p, w, wl, out, 4, width, b, keep, recent, sinks, kept, lens, nw, None)
    assert evict(w=None) == evict(out=None) == evict(kept=None) == evict(lens=None) == evict(nw=None) == evict(nw=p) == -1
    assert evict(keep=-1) == evict(recent=-1) == evict(sinks=-1) == evict(recent=31) == evict(wl=31) == evict(width=1) == -1
    assert evict(b=0) == 0

    s9, s3 = (i64 * 9)(*[4096, 1024, 64] * 3), (i64 * 3)(4096, 1024, 64)
    window = lambda q=p, k=p, v=p, dt=2, s=s9, out=p, so=s3, b=1, hq=4, hkv=2, sq=16, sk=16, d=64, scale=1.0, sinks=0: lib.b200q_window_attention(  # noqa: E731
        q, k, v, dt, s, out, so, None, None, b, hq, hkv, sq, sk, d, scale, 0, sinks, None)
    assert window(q=None) == window(k=None) == window(v=None) == window(out=None) == window(s=None) == window(so=None) == -1
    assert window(dt=0) == window(hq=3) == window(hkv=0) == window(sq=-1) == window(d=72) == window(d=144) == window(sinks=-1) == -1
    assert window(scale=float("nan")) == window(b=40000) == -1
    assert window(q=p + 2) == window(k=p + 2) == window(out=p + 4) == window(s=(i64 * 9)(*[4096, 1024, 60] * 3)) == -2
    assert window(so=(i64 * 3)(4096, 1024, 60)) == -2
    assert window(b=0) == window(sq=0) == 0


def test_fake_kernels(b200):
    m = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    kp, table, lens = m(10, 2, 16, 64), m(3, 4, dtype=torch.int32), m(3, dtype=torch.int32)
    w = m(3, 2, 64, dtype=torch.float32)
    out = b200.paged_attention(m(3, 8, 64), kp, kp, table, lens, weights=w)
    assert out.shape == (3, 8, 64) and out.dtype == torch.bfloat16
    assert b200.paged_append(m(3, 2, 64), m(3, 2, 64), kp, kp, table, lens) is None
    kept, n, nw = b200.paged_evict(kp, kp, table, lens, w, table, keep=32, recent=4, sinks=1)
    assert kept.shape == (3, 2, 32) and kept.dtype == torch.int32 and n.shape == (3,) and nw.shape == w.shape
    q = m(2, 100, 8, 64).transpose(1, 2)
    assert b200.window_attention(q, m(2, 2, 100, 64), m(2, 2, 100, 64)).stride() == q.stride()


def test_schemas_say_what_is_written(b200):
    written = {name: [a.name for a in getattr(torch.ops.tensorrt, name).default._schema.arguments if a.alias_info and a.alias_info.is_write]
               for name in ("b200_paged_append", "b200_paged_attention", "b200_paged_evict", "b200_window_attention")}
    assert written == {"b200_paged_append": ["k_pages", "v_pages"], "b200_paged_attention": ["weights"],
                       "b200_paged_evict": ["k_pages", "v_pages"], "b200_window_attention": []}


def test_cpu_tensors_are_refused(b200):
    x, n = torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.ones(1, dtype=torch.int32)
    pages, table = torch.zeros(1, 1, 16, 64, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: b200.paged_append(x, x, pages, pages, table, n), lambda: b200.paged_attention(x, pages, pages, table, n),
                 lambda: b200.window_attention(x[None], x[None], x[None])):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


# ----------------------------------------------------------------------------- PagedKvCache on the host
def host_cache(b200, **kw):
    return b200.PagedKvCache(**{**dict(layers=2, batch=3, n_kv=2, head_dim=16, pages=14, max_tokens=64, page_size=8, weights=True, device="cpu"), **kw})


def state(cache):
    return cache.tokens(), cache.lens.tolist(), cache.table.tolist(), sorted(cache._free), [list(p) for p in cache._pages]


@pytest.mark.parametrize("bad", [dict(keep=16, recent=10, sinks=7), dict(keep=65), dict(keep=-1), dict(keep=8, recent=-1), dict(keep=8, sinks=-1)], ids=str)
def test_a_refused_eviction_loses_no_pages(b200, bad):
    cache = host_cache(b200)
    cache.grow([20, 9, 0])
    before = state(cache)
    with pytest.raises(ValueError):
        cache.evict(**bad)
    assert state(cache) == before
    with pytest.raises((RuntimeError, NotImplementedError)):      # no device: refused by the call behind
        cache.evict(8, 2, 1)
    assert state(cache) == before


def test_eviction_asks_for_the_pages_that_it_takes(b200, monkeypatch):
    """Short sequences need room for what they have, not for `keep` tokens; one page less is too few."""
    import tensorrt_b200.kv_cache as kv

    def evict(k, v, table, lens, weights, out, *, keep, recent, sinks):
        return torch.zeros(3, 2, keep, dtype=torch.int32), lens.clamp(max=keep), torch.zeros_like(weights)

    monkeypatch.setattr(kv, "paged_evict", evict)
    cache = host_cache(b200)
    cache.grow([40, 9, 3])                               # 5 + 2 + 1 of 14 pages; of 32 tokens 4 + 2 + 1 would be fresh
    with pytest.raises(RuntimeError, match="7 pages are needed and 6 are free"):
        cache.evict(32)
    cache.evict(24)                                      # 3 + 2 + 1
    assert cache.tokens() == [24, 9, 3] == cache.lens.tolist() and cache.free_pages() == 8
    assert [(r >= 0).sum().item() for r in cache.table] == [3, 2, 1]


def test_the_cache_takes_the_rows_that_were_announced(b200):
    cache = host_cache(b200)
    rows = lambda n: (torch.zeros(n, 2, 16, dtype=torch.bfloat16),) * 2  # noqa: E731
    cache.grow([4, 0, 2])
    for n in (3, 5, 7):
        with pytest.raises(ValueError, match="6 new tokens"):
            cache.append(0, *rows(n))
    cache.grow([1, 1, 1])
    with pytest.raises(ValueError, match="3 new tokens"):
        cache.append(0, *rows(6))


class NoLayers:
    """What CachedDecoder asks of a stack, without its kernels."""
    world = 1

    def __init__(self, **kw):
        from types import SimpleNamespace

        self.cfg = SimpleNamespace(**{**dict(hidden=64, n_q=4, n_kv=2, head_dim=16), **kw})
        self.layers = [None, None]


def test_what_the_decoder_refuses_changes_nothing(b200):
    cache = host_cache(b200)
    decoder = b200.CachedDecoder(NoLayers(), cache)
    cache.grow([4, 0, 2])
    before = state(cache)
    h = lambda n, hidden=64: torch.zeros(n, hidden, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(ValueError, match="as a whole"):
        decoder.prompt(h(5), [0, 3, 2])
    with pytest.raises(ValueError, match="expected"):
        decoder.prompt(h(5, 32), [0, 5, 0])
    with pytest.raises(ValueError, match="expected"):
        decoder.step(h(3, 32))
    with pytest.raises(ValueError, match="counts"):
        decoder.prompt(h(5), [0, 5])
    assert state(cache) == before
    with pytest.raises(ValueError, match="type"):
        b200.CachedDecoder(NoLayers(), host_cache(b200, dtype=torch.float16))


def test_prompts_of_some_sequences(b200):
    cache = host_cache(b200)
    cache.grow([4, 0, 2])
    cache.release(2)
    cache.check_prompt([0, 3, 5])
    for new in ([1, 0, 0], [1, 3, 0]):
        with pytest.raises(ValueError, match="as a whole"):
            cache.check_prompt(new)


def test_a_released_sequence_takes_no_token_of_a_step(b200):
    cache = host_cache(b200)
    cache.grow([4, 9, 2])
    cache.release(1)
    for _ in range(40):
        cache.grow_all()
    assert cache.tokens() == [44, 0, 42] == cache.lens.tolist() and cache.free_pages() == 14 - 12
    cache.grow([0, 3, 0])                                # until it is asked for by name
    cache.grow_all()
    assert cache.tokens() == [45, 4, 43] == cache.lens.tolist() and cache.free_pages() == 14 - 13


def test_scratch_is_for_the_keys_that_can_be_seen(b200, p):
    from tensorrt_b200 import _lib

    lib, i64 = _lib.load(), ctypes.c_int64
    c, s2 = ctypes.byref(cache_of(p)), (i64 * 2)(128, 64)     # pages of 16 rows
    attend = lambda sn, width, window, sinks, wl: lib.b200q_paged_attention(  # noqa: E731
        p, 2, s2, c, p, width, width, p, 3, 4, 1.0, window, sinks, p, p, wl, p, 1 << 40, p, sn, None)
    for width, window, sinks, wl, keys in ((4, 0, 0, 64, 64), (4, 0, 0, 1 << 17, 64), (1 << 13, 0, 0, 500, 500), (1 << 13, 100, 20, 1 << 17, 120),
                                           (1 << 13, 100, 1 << 62, 1 << 17, 1 << 17), (4, 1 << 62, 3, 1 << 17, 64), (0, 0, 0, 64, 0)):
        n = lib.b200q_paged_attention_scratch_bytes(3, 4, keys)
        assert attend(n - 1, width, window, sinks, wl) == -5
        if not torch.cuda.is_available():
            assert attend(n, width, window, sinks, wl) not in (0, -1, -2, -5)     # as far as the device
