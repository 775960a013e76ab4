"""Continuations under torch's inference mode: a step in it, the cache's changes outside, and the other way round."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inside", [True, False])
def test_steps_in_inference_mode_and_forks_outside(b200, monkeypatch, inside):
    import tensorrt_b200.kv_cache as kv

    monkeypatch.setattr(kv, "_SHARED_KEYS", 1)
    g = torch.Generator(device="cuda").manual_seed(4)
    k, q = torch.randn(70, 2, 64, device="cuda", generator=g).bfloat16(), torch.randn(4, 8, 64, device="cuda", generator=g).bfloat16()
    cache = b200.PagedKvCache(1, 4, 2, 64, pages=60, max_tokens=128, page_size=16)
    cache.grow([70, 0, 0, 0])
    cache.append(0, k, k)
    outs = []
    for parents in ([0, 0, 0, 0], [0, 1, 1, 2], [3, 3, 3, 3]):
        with torch.inference_mode(not inside):
            cache.fork(parents)
        with torch.inference_mode(inside):
            cache.grow_all()
            cache.append(0, k[:4] * (1 + len(outs)), k[4:8])
            assert cache._shares
            outs.append((cache.attend(0, q), b200.paged_attention(q, cache.k[0], cache.v[0], cache.table, cache.lens)))
            scores = b200.token_log_probs(q.flatten(1), top=3)
            assert scores.top_tokens.shape == (4, 3)
        with torch.inference_mode(not inside):
            cache.truncate([n - 1 if b == 3 else n for b, n in enumerate(cache.tokens())])
            cache.compact()
            cache.resize(60)
    for a, b in outs:
        assert (a.float() - b.float()).norm() <= 2.0 ** -7 * b.float().norm()
