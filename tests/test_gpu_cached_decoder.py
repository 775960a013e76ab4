"""The cache's calls as a generating decoder makes them: prompts, single tokens, eviction, release.

What is compared walks the same quantized linears, so the bounds are those of two orders of the same sums behind a bf16 residual
stream: rel-L2 2e-2, as for the stack's other forms."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def rel(a, b):
    a, b = a.double(), b.double()
    return ((a - b).norm() / b.norm()).item()


def make(b200, layers=2, batch=3, dtype=torch.bfloat16, **kw):
    from tensorrt_b200.stack import DecoderStack, StackConfig, random_layer_weights

    cfg = StackConfig(hidden=512, n_q=8, n_kv=2, head_dim=64, ffn=1024, layers=layers)
    stack = DecoderStack(cfg, random_layer_weights(cfg, 3))
    if dtype == E4M3:
        kw["k_amax"] = kw["v_amax"] = [torch.tensor([4.0], device="cuda")] * layers
    return stack, b200.PagedKvCache(layers, batch, 2, 64, pages=200, max_tokens=600, page_size=8, dtype=dtype, **kw)


@pytest.mark.parametrize("dtype,bound", [(torch.bfloat16, 2e-2), (E4M3, 6e-2)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
def test_tokens_one_by_one_equal_the_prompt_at_once(b200, dtype, bound, window, sinks):
    """With 8-bit pages the keys and values of a step carry one rounding of 2^-4 that those of a prompt in hand do not."""
    g = torch.Generator(device="cuda").manual_seed(1)
    lens, steps = [40, 7, 90], 5
    h = [torch.randn(n + steps, 512, device="cuda", generator=g).bfloat16() for n in lens]
    stack, cache = make(b200, dtype=dtype)
    whole = b200.CachedDecoder(stack, cache, window, sinks).prompt(torch.cat(h), [n + steps for n in lens])
    want = torch.cat([t[-steps:] for t in whole.split([n + steps for n in lens])])
    stack, cache = make(b200, dtype=dtype)
    decoder = b200.CachedDecoder(stack, cache, window, sinks)
    decoder.prompt(torch.cat([t[:n] for t, n in zip(h, lens)]), lens)
    got = torch.stack([decoder.step(torch.stack([t[n + s] for t, n in zip(h, lens)])) for s in range(steps)], 1).flatten(0, 1)
    assert cache.tokens() == [n + steps for n in lens] and cache.lens.tolist() == cache.tokens()
    assert rel(got, want) <= bound


def test_prompts_of_one_length_and_the_core_by_hand(b200):
    """One layer's attention inside the walk against the formula on the projection that the layer makes."""
    g = torch.Generator(device="cuda").manual_seed(2)
    stack, cache = make(b200, layers=1)
    h = torch.randn(3 * 33, 512, device="cuda", generator=g).bfloat16()
    seen = {}
    inner = cache.attend_prompt

    def attend_prompt(layer, q, k, v, **kw):
        seen["q"], seen["k"], seen["v"], seen["out"] = q, k, v, inner(layer, q, k, v, **kw)
        return seen["out"]

    cache.attend_prompt = attend_prompt
    b200.CachedDecoder(stack, cache).prompt(h, [33, 33, 33])
    q, k, v = (seen[n].double().view(3, 33, -1, 64).transpose(1, 2) for n in "qkv")
    s = q @ k.repeat_interleave(4, 1).transpose(2, 3) / math.sqrt(64)
    s = s.masked_fill(~torch.ones(33, 33, dtype=torch.bool, device="cuda").tril(), -math.inf)
    want = (torch.softmax(s, -1) @ v.repeat_interleave(4, 1)).transpose(1, 2).reshape(99, 8, 64)
    assert rel(seen["out"], want) <= 2.0 ** -7


def test_eviction_keeps_what_the_weights_say_and_generation_goes_on(b200):
    g = torch.Generator(device="cuda").manual_seed(3)
    stack, cache = make(b200, weights=True)
    decoder = b200.CachedDecoder(stack, cache)
    decoder.prompt(torch.randn(200, 512, device="cuda", generator=g).bfloat16(), [100, 60, 40])
    for _ in range(4):
        decoder.step(torch.randn(3, 512, device="cuda", generator=g).bfloat16())
    before = [w.clone() for w in cache.weights]
    assert all(abs(w[b].sum().item() / (8 * 4) - 1) < 1e-3 for w in before for b in range(3))     # 8 query heads, 4 steps: each a sum of one
    used = cache.free_pages()
    kept = cache.evict(50, recent=10, sinks=2)
    assert cache.tokens() == [50, 50, 44] and cache.lens.tolist() == [50, 50, 44] and cache.free_pages() > used
    for w, which in zip(before, kept):
        for b, n in enumerate((104, 64, 44)):
            for head in range(2):
                mid = w[b, head, 2:n - 10]
                best = set((2 + mid.sort(descending=True, stable=True).indices[:min(n, 50) - 12]).tolist()) | {0, 1} | set(range(n - 10, n))
                assert set(which[b, head].tolist()) - {-1} == best
    out = decoder.step(torch.randn(3, 512, device="cuda", generator=g).bfloat16())
    assert torch.isfinite(out.float()).all() and cache.tokens() == [51, 51, 45]
    cache.release(1)
    assert cache.tokens()[1] == 0 and cache.lens.tolist()[1] == 0 and not cache.weights[0][1].any()


def test_a_step_in_a_graph(b200):
    """Pages reserved in front, the tokens' part of a step captured once and replayed as the sequences grow."""
    g = torch.Generator(device="cuda").manual_seed(4)
    _, cache = make(b200, layers=1)
    _, plain = make(b200, layers=1)
    k = torch.randn(3, 2, 64, device="cuda", generator=g).bfloat16()
    v, q = k.clone(), torch.randn(3, 8, 64, device="cuda", generator=g).bfloat16()
    for c in (cache, plain):
        c.reserve([30, 30, 30])
        c.grow([1, 1, 1])
        c.append(0, k, v)
        c.attend(0, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(0, k, v)
        out = cache.attend(0, q)
    for _ in range(20):
        k.normal_(generator=g), v.normal_(generator=g), q.normal_(generator=g)
        cache.grow([1, 1, 1]), plain.grow([1, 1, 1])
        graph.replay()
        plain.append(0, k, v)
        assert torch.equal(out, plain.attend(0, q))


def test_what_the_classes_refuse(b200):
    stack, cache = make(b200)
    for bad in (dict(dtype=torch.float32), dict(dtype=E4M3), dict(pages=0), dict(k_amax=[1.0], v_amax=[1.0])):
        with pytest.raises(ValueError):
            b200.PagedKvCache(**{**dict(layers=1, batch=1, n_kv=1, head_dim=64, pages=4, max_tokens=64), **bad})
    with pytest.raises(ValueError, match="kv heads"):
        b200.CachedDecoder(stack, b200.PagedKvCache(2, 3, 4, 64, pages=4, max_tokens=64))
    decoder = b200.CachedDecoder(stack, cache)
    with pytest.raises(ValueError, match="expected"):
        decoder.prompt(torch.zeros(5, 512, dtype=torch.bfloat16, device="cuda"), [1, 1, 1])
    with pytest.raises(ValueError, match="expected"):
        decoder.step(torch.zeros(5, 512, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="counts"):
        cache.grow([1, 1])
    with pytest.raises(ValueError, match="counts"):
        cache.reserve([601, 1, 1])
    with pytest.raises(RuntimeError, match="free"):
        cache.grow([600, 600, 600])
    with pytest.raises(ValueError, match="weights"):
        cache.evict(4)
    cache.grow([4, 4, 4])
    cache.grow([1, 1, 1])
    with pytest.raises(ValueError, match="as a whole"):
        cache.attend_prompt(0, *(torch.zeros(3, n, 64, dtype=torch.bfloat16, device="cuda") for n in (8, 2, 2)))


# ----------------------------------------------------------------------------- slots that are freed and filled again
def test_a_refused_prompt_changes_nothing(b200):
    stack, cache = make(b200)
    g = torch.Generator(device="cuda").manual_seed(5)
    decoder = b200.CachedDecoder(stack, cache)
    h = torch.randn(60, 512, device="cuda", generator=g).bfloat16()
    decoder.prompt(h[:30], [10, 12, 8])
    before = cache.tokens(), cache.lens.tolist(), cache.free_pages(), cache.table.clone(), [t.clone() for t in cache.k + cache.v]
    for lens in ([20, 20, 20], [0, 60, 0]):
        with pytest.raises(ValueError, match="as a whole"):
            decoder.prompt(h, lens)
        with pytest.raises(ValueError, match="expected"):
            decoder.prompt(h[:, :256], lens)
    assert (cache.tokens(), cache.lens.tolist(), cache.free_pages()) == before[:3] and torch.equal(cache.table, before[3])
    assert all(torch.equal(a, b) for a, b in zip(cache.k + cache.v, before[4]))


@pytest.mark.parametrize("lens", [[0, 25, 0], [13, 0, 0]])
def test_a_freed_slot_takes_a_new_prompt(b200, lens):
    """Beside sequences that go on: the same as in a cache of its own, and the others do not notice."""
    g = torch.Generator(device="cuda").manual_seed(6)
    stack, cache = make(b200)
    decoder = b200.CachedDecoder(stack, cache, 16, 2)
    decoder.prompt(torch.randn(90, 512, device="cuda", generator=g).bfloat16(), [40, 20, 30])
    b = [i for i, n in enumerate(lens) if n][0]
    cache.release(b)
    h = torch.randn(sum(lens), 512, device="cuda", generator=g).bfloat16()
    kept = [i for i in range(3) if i != b]
    rows = {i: cache.k[1][cache.table[i, :2].long()].clone() for i in kept}
    got = decoder.prompt(h, lens)
    own_stack, own = make(b200, batch=1)
    alone = b200.CachedDecoder(own_stack, own, 16, 2)
    assert rel(got, alone.prompt(h, [sum(lens)])) <= 2e-2
    assert all(torch.equal(cache.k[1][cache.table[i, :2].long()], rows[i]) for i in kept)
    step = torch.randn(3, 512, device="cuda", generator=g).bfloat16()
    assert rel(decoder.step(step)[b], alone.step(step[b:b + 1])[0]) <= 2e-2
    assert cache.tokens() == [n + 1 if n else (40, 20, 30)[i] + 1 for i, n in enumerate(lens)] == cache.lens.tolist()


def test_steps_leave_freed_slots_alone(b200):
    """A freed slot takes no token and no page; its row of a step is nobody's."""
    g = torch.Generator(device="cuda").manual_seed(7)
    h = torch.randn(60, 512, device="cuda", generator=g).bfloat16()
    steps = torch.randn(20, 3, 512, device="cuda", generator=g).bfloat16()
    outs = []
    for freed in (False, True):
        stack, cache = make(b200, weights=True)
        decoder = b200.CachedDecoder(stack, cache)
        decoder.prompt(h, [10, 30, 20])
        if freed:
            cache.release(1)
        free = cache.free_pages()
        outs.append([decoder.step(s) for s in steps])
        if freed:
            assert cache.tokens() == [30, 0, 40] == cache.lens.tolist() and (cache.table[1] == -1).all()
            assert free - cache.free_pages() == (4 - 2) + (5 - 3) and not cache.weights[0][1].any()
    for a, b in zip(*outs):
        assert torch.isfinite(b.float()).all() and torch.equal(a[0::2], b[0::2])


@pytest.mark.parametrize("lens", [[21, 21, 21], [40, 7, 90], [0, 9, 300]])
def test_prompts_and_steps_do_not_wait_for_the_device(b200, lens):
    g = torch.Generator(device="cuda").manual_seed(8)
    h = torch.randn(sum(lens), 512, device="cuda", generator=g).bfloat16()
    step = torch.randn(3, 512, device="cuda", generator=g).bfloat16()
    for _ in range(2):                                    # once for what is set up on first use
        stack, cache = make(b200)
        decoder = b200.CachedDecoder(stack, cache, 30, 1)
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error" if _ else "default")
        try:
            decoder.prompt(h, lens)
            cache.release(1)
            decoder.step(step)
        finally:
            torch.cuda.set_sync_debug_mode("default")
    assert cache.tokens() == [lens[0] + 1, 0, lens[2] + 1] == cache.lens.tolist()
