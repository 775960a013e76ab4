"""Pages of the key-value cache copied to others, in the pools of all layers at once: every byte as indexing gives it, no other byte touched."""
import pytest
import torch

from test_gpu_paged_cache import E4M3

pytestmark = pytest.mark.gpu


def raw(t):
    """The bits: random ones are NaN here and there, which equals nothing."""
    return t.view(torch.uint8 if t.element_size() == 1 else torch.int16)


def pools(g, layers, pages, heads, rows, d, dt, layout):
    got = []
    for _ in range(2 * layers):
        shape = (pages, rows, heads, d) if layout == "nhd" else (pages, heads, rows, d)
        bytes_ = torch.randint(0, 256, (*shape[:3], d * (1 if dt in (E4M3, torch.uint8) else 2)), dtype=torch.uint8, device="cuda", generator=g)
        t = bytes_.view(dt)
        if layout == "apart":                              # pages, heads and rows with room between them
            room = torch.zeros(pages, heads + 1, rows + 2, d + 16, dtype=torch.uint8 if t.element_size() == 1 else dt, device="cuda")
            room = room.view(dt)[:, :heads, :rows, :d]
            room.view(torch.uint8 if t.element_size() == 1 else torch.int16).copy_(raw(t))
            t = room
        got.append(t.transpose(1, 2) if layout == "nhd" else t)
    return got[:layers], got[layers:]


def want(pool, src, dst, rows):
    out = raw(pool).clone()
    for i, (a, b) in enumerate(zip(src, dst)):
        n = pool.shape[2] if rows is None else rows[i]
        out[b, :, :n] = raw(pool)[a, :, :n]
    return out


@pytest.mark.parametrize("layers,pages,heads,rows,d,dt,layout,pairs,partial", [
    (1, 2, 1, 1, 16, torch.bfloat16, "hnd", 1, False), (1, 3, 1, 16, 64, E4M3, "hnd", 1, True), (2, 40, 8, 16, 128, torch.bfloat16, "hnd", 17, True),
    (3, 40, 3, 24, 80, torch.float16, "nhd", 20, True), (2, 40, 3, 5, 96, E4M3, "nhd", 9, False), (2, 30, 2, 7, 48, torch.uint8, "apart", 15, True),
    (80, 12, 2, 16, 64, torch.bfloat16, "hnd", 5, True), (2, 300, 2, 16, 64, torch.float16, "hnd", 70, False), (140, 6, 1, 4, 16, E4M3, "hnd", 3, True),
    (1, 5000, 1, 2, 32, torch.float16, "nhd", 2400, True), (1, 6, 4, 1000, 128, torch.bfloat16, "hnd", 2, True), (1, 4, 300, 3, 112, torch.bfloat16, "apart", 2, False)],
    ids=str)
def test_copies(b200, layers, pages, heads, rows, d, dt, layout, pairs, partial):
    g = torch.Generator(device="cuda").manual_seed(pages + d)
    k, v = pools(g, layers, pages, heads, rows, d, dt, layout)
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    dst = order[:pairs]
    left = order[pairs:]
    src = [left[(i * i) % len(left)] for i in range(pairs)]                # some are read more than once
    n = [(i * 5 + 1) % (rows + 1) for i in range(pairs)] if partial else None
    expected = [want(p, src, dst, n) for p in k + v]
    b200.paged_copy(k, v, src, dst, n)
    assert all(torch.equal(raw(p), e) for p, e in zip(k + v, expected))
    b200.paged_copy(k, v, src, dst, n)                                     # again: the same
    assert all(torch.equal(raw(p), e) for p, e in zip(k + v, expected))


def test_pools_of_two_layouts_tensors_and_the_op(b200):
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = pools(g, 2, 9, 4, 8, 64, torch.bfloat16, "hnd")[0], pools(g, 2, 9, 4, 8, 64, torch.bfloat16, "nhd")[1]
    expected = [want(p, [0, 0], [5, 7], [3, 8]) for p in k + v]
    b200.paged_copy(tuple(k), tuple(v), (0, 0), (5, 7), (3, 8))
    assert all(torch.equal(raw(p), e) for p, e in zip(k + v, expected))
    expected = [want(p, [1], [2], None) for p in (k[0], v[0])]
    b200.paged_copy(k[0], v[0], [1], [2])
    assert all(torch.equal(raw(p), e) for p, e in zip((k[0], v[0]), expected))
    expected = [want(p, [3], [4], [2]) for p in k + v]
    torch.ops.tensorrt.b200_paged_copy(k, v, [3], [4], [2])
    assert all(torch.equal(raw(p), e) for p, e in zip(k + v, expected))
    before = [p.clone() for p in k + v]
    b200.paged_copy(k, v, [], [])
    b200.paged_copy([], [], [1], [2])
    assert all(torch.equal(raw(p), raw(e)) for p, e in zip(k + v, before))


def test_a_captured_copy_keeps_its_numbers(b200):
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = pools(g, 3, 20, 2, 16, 64, torch.float16, "hnd")
    start = [p.clone() for p in k + v]
    src, dst = [0, 1], [10, 11]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b200.paged_copy(k, v, src, dst)
    src[:], dst[:] = [5, 6], [12, 13]                                      # the lists are the caller's again
    for p, s in zip(k + v, start):
        p.copy_(s)
    graph.replay()
    assert all(torch.equal(raw(p), want(s, [0, 1], [10, 11], None)) for p, s in zip(k + v, start))


def test_refusals(b200):
    k, v = torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    f = b200.paged_copy
    many = list(range(100))
    big = torch.zeros(300, 1, 1, 16, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: f(k, v, [0], [0]), lambda: f(k, v, [0, 1], [2, 2]), lambda: f(k, v, [0, 1], [1, 2]), lambda: f(k, v, [0], [8]), lambda: f(k, v, [-1], [1]),
                 lambda: f(k, v, [0, 1], [2]), lambda: f(k, v, [0], [1], [17]), lambda: f(k, v, [0], [1], [-1]), lambda: f(k, v, [0], [1], []),
                 lambda: f([k], [], [0], [1]), lambda: f(k.float(), v.float(), [0], [1]), lambda: f(big, big, many, [100 + i % 99 for i in many]),
                 lambda: f(big, big, many, [99 + i for i in many]), lambda: f(k, v, [0], [1 << 40])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: f(k, v[:7], [0], [1]), lambda: f(k, v.half(), [0], [1]), lambda: f(k.cpu(), v.cpu(), [0], [1]), lambda: f(k, v.cpu(), [0], [1]),
                 lambda: f(k[..., ::2], v[..., ::2], [0], [1])):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
    assert not k.any() and not v.any()
