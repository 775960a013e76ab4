"""Several continuations of one prompt through a decoder: fork, steps over shared pages, scores, and the beams that are chosen go on.  What is compared
walks the same quantized linears: rel-L2 2e-2 behind a bf16 residual stream, as for the cached decoder's other forms."""
import pytest
import torch

from test_gpu_cached_decoder import E4M3, make, rel

pytestmark = pytest.mark.gpu


def singles(b200, texts, dtype):
    """The newest hidden state of every text by itself: a prompt to all but its last token, then a step; no page is shared."""
    stack, cache = make(b200, batch=len(texts), dtype=dtype)
    decoder = b200.CachedDecoder(stack, cache)
    decoder.prompt(torch.cat([t[:-1] for t in texts]), [len(t) - 1 for t in texts])
    return decoder.step(torch.stack([t[-1] for t in texts]))


@pytest.mark.parametrize("dtype,bound", [(torch.bfloat16, 2e-2), (E4M3, 6e-2)])
@pytest.mark.parametrize("length", [3, 64, 171])
def test_beams_are_what_each_would_be_alone(b200, monkeypatch, dtype, bound, length):
    """Six beams of two prompts: forked, stepped, scored and chosen five times over, with a compaction in between."""
    import tensorrt_b200.kv_cache as kv

    monkeypatch.setattr(kv, "_SHARED_KEYS", 1)
    g = torch.Generator(device="cuda").manual_seed(length)
    embed = torch.randn(300, 512, device="cuda", generator=g).bfloat16()
    head = b200.Fp8Linear.from_float((torch.randn(300, 512, device="cuda", generator=g) * 0.05).bfloat16())
    prompts = [torch.randn(n, 512, device="cuda", generator=g).bfloat16() for n in (length, 33)]
    stack, cache = make(b200, batch=6, dtype=dtype)
    decoder = b200.CachedDecoder(stack, cache)
    decoder.prompt(torch.cat(prompts), [length, 33, 0, 0, 0, 0])
    cache.fork([0, 1, 0, 0, 1, 1])
    texts = [prompts[i] for i in (0, 1, 0, 0, 1, 1)]
    tokens, total = torch.tensor([1, 2, 3, 4, 5, 6], device="cuda"), torch.zeros(6, device="cuda")
    shares = []
    for step in range(5):
        texts = [torch.cat([t, embed[tokens[b]][None]]) for b, t in enumerate(texts)]
        h = decoder.step(embed[tokens])
        shares.append(cache._shares)
        assert rel(h, singles(b200, texts, dtype)) <= bound
        scores = decoder.score(h, head, top=3)
        logits = head(h).double()
        assert torch.equal(scores.top_tokens.long(), logits.sort(dim=1, descending=True, stable=True).indices[:, :3])
        assert (scores.top_log_probs - torch.log_softmax(logits, 1).gather(1, scores.top_tokens.long())).abs().max() <= 2.0 ** -14
        # the three best of each prompt's beams go on
        parents, chosen = [0] * 6, [0] * 6
        for beams in ([0, 2, 3], [1, 4, 5]):
            at = (total[beams, None] + scores.top_log_probs[beams]).flatten().topk(3).indices.tolist()
            for b, i in zip(beams, at):
                parents[b], chosen[b] = beams[i // 3], int(scores.top_tokens[beams[i // 3], i % 3])
        total = torch.stack([total[p] + scores.top_log_probs[p][(scores.top_tokens[p] == t).nonzero()[0, 0]] for p, t in zip(parents, chosen)])
        cache.fork(parents)
        texts, tokens = [texts[p] for p in parents], torch.tensor(chosen, device="cuda")
        if step == 2:
            used = cache.compact()
            assert used == 200 - cache.free_pages() and int(cache.table.max()) < used
            cache.resize(used + 40)
    assert shares[0] and all(shares)                       # the second prompt is longer than a page
    cache.truncate([len(t) - 2 for t in texts])             # and two tokens back
    texts = [torch.cat([t[:-2], embed[7][None]]) for t in texts]
    assert rel(decoder.step(embed[[7] * 6]), singles(b200, texts, dtype)) <= bound
    for b in range(6):
        cache.release(b)
    assert cache.free_pages() == used + 40


def test_attend_goes_through_the_shared_pages(b200, monkeypatch):
    import tensorrt_b200.kv_cache as kv

    calls = []
    monkeypatch.setattr(kv, "_SHARED_KEYS", 1)
    for name in ("shared_prefix_attention", "paged_attention"):
        def call(*a, name=name, inner=getattr(kv, name), **kw):
            calls.append(name)
            return inner(*a, **kw)
        monkeypatch.setattr(kv, name, call)
    g = torch.Generator(device="cuda").manual_seed(8)
    cache = b200.PagedKvCache(1, 4, 2, 64, pages=100, max_tokens=300, page_size=16)
    k, v = (torch.randn(200, 2, 64, device="cuda", generator=g).bfloat16() for _ in range(2))
    q = torch.randn(4, 8, 64, device="cuda", generator=g).bfloat16()

    def step():
        cache.grow_all()
        cache.append(0, k[:4] + len(calls), v[:4])
        return cache.attend(0, q)

    cache.grow([200, 0, 0, 0])
    cache.append(0, k, v)
    step()
    cache.fork([0, 0, 0, 0])
    shared = step()
    assert calls == ["paged_attention", "shared_prefix_attention"]
    apart = kv.paged_attention(q, cache.k[0], cache.v[0], cache.table, cache.lens)
    assert rel(shared, apart) <= 2.0 ** -7
    cache.attend(0, q, window=50)                           # a window: every sequence by itself
    assert calls[-1] == "paged_attention"
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(0, q)
    cache.release(2)                                        # the graph goes by the table, the lengths and the plan as they are
    graph.replay()
    assert rel(out, kv.paged_attention(q, cache.k[0], cache.v[0], cache.table, cache.lens)) <= 2.0 ** -7 and not out[2].any()
    step()
    graph.replay()
    assert torch.equal(out, cache.attend(0, q)) and not out[2].any()
    cache.release(0)                                        # the one whose line named the prefix
    graph.replay()
    assert rel(out, kv.paged_attention(q, cache.k[0], cache.v[0], cache.table, cache.lens)) <= 2.0 ** -7 and not out[0].any()
    cache.release(1)
    step()
    assert calls[-1] == "paged_attention"                   # nothing is shared any more
    graph.replay()
    assert rel(out[3], cache.attend(0, q)[3]) <= 2.0 ** -7 and not out[:3].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, E4M3], ids=str)
def test_many_continuations_of_a_long_text(b200, dtype):
    """What a batch shares is read once where that is much; both kernels agree to the roundings of P and of the result, 2 x 2^-8 in bf16."""
    g = torch.Generator(device="cuda").manual_seed(8)
    n, B, token = 50000, 5, torch.float16 if dtype == torch.float16 else torch.bfloat16
    amax = dict(k_amax=[torch.tensor([5.0], device="cuda")], v_amax=[torch.tensor([5.0], device="cuda")]) if dtype == E4M3 else {}
    cache = b200.PagedKvCache(1, B, 2, 64, pages=n // 32 + 20, max_tokens=n + 100, page_size=32, dtype=dtype, **amax)
    cache.grow([n] + [0] * (B - 1))
    cache.append(0, *(torch.randn(n, 2, 64, device="cuda", generator=g).to(token) for _ in range(2)))
    cache.fork([0] * B)
    for step in range(3):
        cache.grow_all()
        cache.append(0, *(torch.randn(B, 2, 64, device="cuda", generator=g).to(token) * 3 for _ in range(2)))
        q = torch.randn(B, 6, 64, device="cuda", generator=g).to(token)
        assert cache._shares
        out = cache.attend(0, q)
        assert rel(out, b200.paged_attention(q, cache.k[0], cache.v[0], cache.table, cache.lens, k_amax=cache.k_amax[0], v_amax=cache.v_amax[0])) <= 2.0 ** -7
        cache.fork([0, 0, 1, 3, 3])
    assert cache.free_pages() >= 20 - B - 3
