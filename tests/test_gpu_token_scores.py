"""Log probabilities, entropy and the most likely tokens of a step's logits, against torch in 64 bits.

Bounds, from the arithmetic, in units of 2^-24: a term exp(z) is off by 4 (the hardware exponential) and by 2 for each unit of |z| log2 e (two
roundings of z); weighted by the terms themselves |z| is the entropy's second part, at most 18 for these sizes.  A thread adds up to 128 terms to
each of two sums, and 8 joins follow.  Together below 2^-16 of S, so 2^-16 of log S; z_t = (x_t - max) * scale is rounded twice.  The
entropy's sum of exp(z) z / S has the same relative bound, and is at most the entropy itself.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def reference(x, scale):
    """(log softmax, entropy, places by descending logit, equal ones the lower first), 64 bits."""
    x = x.double()
    z = (x - x.amax(1, keepdim=True)) * scale
    p = z - z.exp().sum(1, keepdim=True).log()
    return p, -(p.exp() * p.clamp_min(-1e300)).sum(1), torch.sort(x, dim=1, descending=True, stable=True).indices


def check(b200, x, tokens, top, scale=1.0):
    got = b200.token_log_probs(x, tokens, top=top, scale=scale)
    p, entropy, order = reference(x, scale)
    near = lambda a, b: torch.where(a.double() == b, 0.0, (a.double() - b).abs() - 2.0 ** -16 - 2.0 ** -22 * b.abs())  # noqa: E731
    assert got.log_probs.dtype == got.entropy.dtype == got.top_log_probs.dtype == torch.float32 and got.top_tokens.dtype == torch.int32
    if tokens is not None:
        there = (tokens >= 0) & (tokens < x.shape[1])
        want = p.gather(1, tokens.clamp(0, x.shape[1] - 1).long()[:, None])[:, 0]
        assert (near(got.log_probs, want)[there] <= 0).all() and not got.log_probs[~there].any()
    else:
        assert not got.log_probs.any()
    assert ((got.entropy.double() - entropy).abs() <= 2.0 ** -15 * (1 + entropy)).all()
    assert torch.equal(got.top_tokens.long(), order[:, :top])
    assert (near(got.top_log_probs, p.gather(1, order[:, :top])) <= 0).all()
    again = b200.token_log_probs(x, tokens, top=top, scale=scale)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    return got


def logits(g, rows, size, dt, pad=0, at=0):
    """Rows of a wider matrix: `pad` elements apart, beginning at `at`."""
    x = torch.randn(rows, size + pad, device="cuda", generator=g) * (1 + 3 * torch.rand(rows, 1, device="cuda", generator=g))
    x += torch.where(torch.rand(rows, size + pad, device="cuda", generator=g) < 5 / size, 10.0, 0.0)
    return x.to(dt)[:, at:at + size]


@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("rows,size,top,pad,at", [
    (1, 1, 1, 0, 0), (3, 2, 2, 0, 0), (5, 7, 5, 0, 0), (4, 9, 3, 2, 1), (300, 31, 31, 0, 0), (2, 64, 64, 5, 3), (7, 500, 20, 1, 1), (40, 4099, 64, 0, 0),
    (3, 32000, 6, 0, 0), (64, 50001, 20, 7, 5), (1, 128000, 64, 0, 0), (700, 8191, 8, 0, 0), (650, 20011, 50, 0, 0), (2, 260003, 1, 0, 0), (9, 50001, 0, 0, 0),
    (1000, 40007, 0, 3, 2)], ids=str)
def test_scores(b200, dt, rows, size, top, pad, at):
    g = torch.Generator(device="cuda").manual_seed(size + top)
    x = logits(g, rows, size, dt, pad, at)
    tokens = torch.randint(0, size, (rows,), device="cuda", generator=g)
    check(b200, x, tokens, top)
    check(b200, x, tokens.int(), top, 1.7)
    check(b200, x, None, top, 0.3)


@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("rows", [2, 700])
def test_orders_that_crowd_a_thread(b200, dt, rows):
    """The largest logits where one thread, or one group of threads, holds them, and equal ones everywhere."""
    size = 16384
    i = torch.arange(size, device="cuda")
    group = (i // 8 % 256 if dt != torch.float32 else i // 4 % 256) // 4
    last = i >= size * 7 // 8
    crowded = torch.where(last & (i % 8 == 0), 100.0 - group / 2, 80.0 + (i % 5) / 4)
    rising = i / 256.0
    for row in (crowded, rising, rising.flip(0), torch.full((size,), 3.0, device="cuda"), torch.where(i % 1024 == 1023, 50.0, -1.0),
                torch.where(group == 17, 40.0, (i % 3).float()), (i % 7).float()):
        x = row.to(dt).expand(rows, size)
        for top in (1, 20, 64):
            check(b200, x if rows == 2 else x.contiguous(), None, top)


@pytest.mark.parametrize("dt", DTYPES, ids=str)
def test_masked_logits(b200, dt):
    g = torch.Generator(device="cuda").manual_seed(5)
    x = logits(g, 40, 30011, dt).clone()
    allowed = torch.rand(x.shape, device="cuda", generator=g) < 0.01
    allowed[1:4] = False
    allowed[1, 30010], allowed[2, :3], allowed[3, 15000:15019] = True, True, True      # fewer than are asked for
    for low in (-math.inf, torch.finfo(dt).min):
        y = x.masked_fill(~allowed, low)
        tokens = allowed.float().argmax(1)
        tokens[7], tokens[8] = -100, 30011
        check(b200, y, tokens, 20)
        tokens[9] = (~allowed[9]).float().argmax()        # a token that the mask forbids
        got = b200.token_log_probs(y, tokens, top=20)
        assert got.log_probs[9] < -1e4 and not got.log_probs[7:9].any()
    check(b200, torch.full((3, 5000), torch.finfo(dt).min, dtype=dt, device="cuda"), None, 64)        # equal ones, whatever their size
    y = x.clone()
    y[:, 100] = torch.finfo(dt).max                        # differences beyond the type
    y[:, 200:] = torch.finfo(dt).min
    check(b200, y, torch.full((40,), 100, device="cuda"), 5)


@pytest.mark.parametrize("dt", DTYPES, ids=str)
def test_rows_without_a_distribution(b200, dt):
    g = torch.Generator(device="cuda").manual_seed(6)
    x = logits(g, 8, 9001, dt).clone()
    clean = b200.token_log_probs(x, torch.zeros(8, dtype=torch.int64, device="cuda"), top=9)
    x[1] = -math.inf
    x[3, 4000] = math.inf
    x[5, 4000] = math.nan
    x[6, 10], x[6, 20], x[6, 30], x[6, 40] = math.nan, math.inf, -math.nan, math.inf
    got = b200.token_log_probs(x, torch.zeros(8, dtype=torch.int64, device="cuda"), top=9)
    for i in (1, 3, 5, 6):
        assert got.log_probs[i].isnan() and got.entropy[i].isnan() and got.top_log_probs[i].isnan().all()
    for a, b in zip(got, clean):                           # the others do not notice
        assert all(torch.equal(a[i], b[i]) for i in (0, 2, 4, 7))
    assert got.top_tokens[1].tolist() == list(range(9))
    assert got.top_tokens[3, 0] == got.top_tokens[5, 0] == 4000 and got.top_tokens[6, :4].tolist() == [10, 30, 20, 40]


def test_zeros_of_both_signs_are_equal(b200):
    x = torch.full((2, 4096), -1.0, dtype=torch.bfloat16, device="cuda")
    x[:, 5], x[:, 6], x[:, 3000] = -0.0, 0.0, -0.0
    assert b200.token_log_probs(x, None, top=3).top_tokens.tolist() == [[5, 6, 3000]] * 2


def test_shapes_streams_graphs(b200):
    g = torch.Generator(device="cuda").manual_seed(7)
    x = logits(g, 24, 5003, torch.bfloat16)
    t = torch.randint(0, 5003, (24,), device="cuda", generator=g)
    want = b200.token_log_probs(x, t, top=7)
    cube = b200.token_log_probs(x.view(2, 3, 4, 5003), t.view(2, 3, 4), top=7)
    assert cube.top_tokens.shape == (2, 3, 4, 7) and cube.entropy.shape == (2, 3, 4)
    assert all(torch.equal(a.flatten(), b.flatten()) for a, b in zip(cube, want))
    turned = b200.token_log_probs(x.t().contiguous().t(), t, top=7)           # a vocabulary that is not contiguous
    assert all(torch.equal(a, b) for a, b in zip(turned, want))
    one = b200.token_log_probs(x[0], t[0], top=2)
    assert one.log_probs.shape == () and torch.equal(one.top_tokens, want.top_tokens[0, :2]) and one.log_probs == want.log_probs[0]
    assert all(torch.equal(a, b) for a, b in zip(torch.ops.tensorrt.b200_token_log_probs(x, t, 7, 1.0), want))
    none = b200.token_log_probs(x[:0], t[:0], top=7)
    assert none.log_probs.shape == (0,) and none.top_tokens.shape == (0, 7)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        there = b200.token_log_probs(x, t, top=7)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(there, want))
    y, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = b200.token_log_probs(y, t, top=7)
    for src in (x.flip(0), x):
        y.copy_(src)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(kept, b200.token_log_probs(src.contiguous(), t, top=7)))
    needs = x.float().requires_grad_()                     # there is no gradient, and the result says so
    with pytest.warns(UserWarning, match="autograd kernel was not registered"):
        b200.token_log_probs(needs, t).entropy.sum().backward()


def test_refusals(b200):
    x, t = torch.zeros(4, 100, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    f = b200.token_log_probs
    for call in (lambda: f(x, t, top=65), lambda: f(x, t, top=-1), lambda: f(x[:, :20], t, top=21), lambda: f(x, t, scale=0.0), lambda: f(x, t, scale=-1.0),
                 lambda: f(x, t, scale=math.nan), lambda: f(x, t, scale=math.inf), lambda: f(x, t, scale=1e-60), lambda: f(x.double(), t), lambda: f(x[:, :0], t)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: f(x, t[:3]), lambda: f(x, t.float()), lambda: f(x, t.cpu()), lambda: f(x.cpu(), t.cpu()), lambda: f(x[0, 0], t[0])):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
