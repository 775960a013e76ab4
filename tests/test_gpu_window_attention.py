"""Causal attention with a sliding window and sinks against a 64-bit restatement; the bounds are those of
tests/test_gpu_paged_cache.py: one rounding of the result, one of P to 16 bits, 32-bit sums."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def reference(q, k, v, window, sinks, nq, nk, scale=None):
    """(out, sum P |V|) in 64 bits; rows that see nothing are zero."""
    b, hq, sq, d = q.shape
    g = hq // k.shape[1]
    out, mass = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for i in range(b):
        at = torch.arange(nq[i], device="cuda")[:, None] + nk[i] - nq[i]
        j = torch.arange(nk[i], device="cuda")
        seen = j <= at
        if window > 0:
            seen = seen & ((j > at - window) | (j < sinks))
        for h in range(hq):
            kk, vv = k[i, h // g, :nk[i]].double(), v[i, h // g, :nk[i]].double()
            s = (q[i, h, :nq[i]].double() @ kk.T) * (1 / math.sqrt(d) if scale is None else scale)
            p = torch.softmax(s.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0) if nk[i] else s
            out[i, h, :nq[i]], mass[i, h, :nq[i]] = p @ vv, p @ vv.abs()
    return out, mass


def check(out, ref, mass):
    u = U[out.dtype]
    tol = u * ref.abs() + (u + 2.0 ** -13) * mass + 1e-30
    off = (out.double() - ref).abs()
    assert torch.isfinite(out.float()).all()
    assert (off <= tol).all(), (off / tol).max().item()


def inputs(g, b, hq, hkv, sq, sk, d, dt, token_major):
    def make(h, s):
        if token_major:
            return torch.randn(b, s, h + 1, d, device="cuda", generator=g).to(dt)[:, :, :h].transpose(1, 2)
        return torch.randn(b, h, s, d, device="cuda", generator=g).to(dt)
    return make(hq, sq), make(hkv, sk), make(hkv, sk)


SHAPES = [
    # b, hq, hkv, sq, sk, d, window, sinks
    (1, 1, 1, 1, 1, 64, 0, 0),
    (1, 2, 1, 1, 300, 128, 0, 0),
    (2, 4, 2, 17, 17, 16, 0, 0),
    (1, 4, 4, 127, 127, 128, 0, 0),
    (1, 4, 2, 128, 128, 128, 0, 0),
    (1, 4, 2, 129, 129, 64, 0, 0),
    (2, 6, 2, 257, 400, 80, 0, 0),
    (2, 6, 2, 300, 200, 96, 0, 0),          # more queries than keys: the first rows see nothing
    (1, 2, 2, 5, 0, 64, 0, 0),
    (1, 8, 1, 700, 1200, 128, 0, 0),
    (1, 2, 1, 513, 513, 128, 1, 0),
    (1, 2, 1, 513, 513, 128, 64, 0),
    (2, 2, 1, 513, 900, 112, 128, 4),
    (1, 2, 1, 1025, 1025, 128, 200, 130),
    (1, 2, 1, 1025, 1025, 48, 300, 5000),   # sinks cover everything
    (1, 2, 1, 100, 100, 32, 5000, 3),       # window covers everything
    (1, 2, 2, 2048, 2048, 128, 100, 1),
    (3, 2, 1, 61, 1999, 128, 1024, 4),
    (1, 40, 8, 333, 333, 64, 77, 2),
    (1, 2, 1, 4097, 4097, 128, 0, 0),
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_window_attention(b200, shape, token_major, dt):
    b, hq, hkv, sq, sk, d, window, sinks = shape
    g = torch.Generator(device="cuda").manual_seed(sq + sk + d)
    q, k, v = inputs(g, b, hq, hkv, sq, sk, d, dt, token_major)
    out = b200.window_attention(q, k, v, window=window, sinks=sinks)
    assert out.shape == q.shape and out.dtype == dt
    if token_major and sq > 1 and hq > 1:
        assert out.transpose(1, 2).is_contiguous()
    ref, mass = reference(q, k, v, window, sinks, [sq] * b, [sk] * b)
    check(out, ref, mass)
    assert torch.equal(out, b200.window_attention(q, k, v, window=window, sinks=sinks))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 3)])
def test_ragged_lengths_with_anything_beyond_them(b200, dt, window, sinks):
    b, hq, hkv, s, d = 7, 4, 2, 400, 80
    g = torch.Generator(device="cuda").manual_seed(11)
    q, k, v = inputs(g, b, hq, hkv, s, s + 50, d, dt, True)
    nq, nk = [400, 1, 0, 129, 128, 300, 40], [450, 51, 30, 129, 400, 100, 0]
    for i in range(b):
        for t, n in ((q, nq), (k, nk), (v, nk)):
            t[i, :, n[i]:] = float("nan")
        v[i, :, nk[i]::3] = float("inf")
    lens = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (nq, nk)]
    out = b200.window_attention(q, k, v, window=window, sinks=sinks, q_lens=lens[0], k_lens=lens[1])
    ref, mass = reference(q, k, v, window, sinks, nq, nk)
    check(out, ref, mass)
    wild = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([9999] * b, [-5] * b)]
    assert not b200.window_attention(q, k, v, q_lens=wild[0], k_lens=wild[1]).any()      # cut to the tensors; no keys


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 2)])
def test_masked_keys_do_not_matter(b200, bad, window, sinks):
    """A key or value that is not finite shows in the rows that see it, and in no other."""
    g = torch.Generator(device="cuda").manual_seed(12)
    q, k, v = inputs(g, 1, 4, 2, 500, 500, 64, torch.bfloat16, False)
    at = 201
    seen = torch.arange(500, device="cuda") >= at
    if window > 0:
        seen &= torch.arange(500, device="cuda") < at + window
    clean = b200.window_attention(q, k, v, window=window, sinks=sinks)
    v2 = v.clone()
    v2[0, 0, at] = bad
    out = b200.window_attention(q, k, v2, window=window, sinks=sinks)
    ref, mass = reference(q, k, v, window, sinks, [500], [500])
    check(out[:, :2, ~seen], ref[:, :2, ~seen], mass[:, :2, ~seen])
    assert not torch.isfinite(out[:, :2, seen].float()).any() and torch.equal(out[:, 2:], clean[:, 2:])
    k2 = k.clone()
    k2[0, 0, at] = bad
    out = b200.window_attention(q, k2, v, window=window, sinks=sinks)
    check(out[:, :2, ~seen], ref[:, :2, ~seen], mass[:, :2, ~seen])
    assert torch.equal(out[:, 2:], clean[:, 2:])


def test_logits_of_every_size(b200):
    """A maximum that keeps rising along the keys, and logits of some hundreds: the running maximum is followed."""
    g = torch.Generator(device="cuda").manual_seed(13)
    q, k, v = inputs(g, 1, 2, 1, 700, 700, 128, torch.bfloat16, False)
    ramp = torch.linspace(0.01, 8.0, 700, device="cuda")[:, None]
    for f in (ramp, ramp.flip(0), 20.0, 1e-4):
        kk = (k.float() * f).bfloat16()
        qq = (q.float().abs() + 0.25).bfloat16()
        kk = torch.where(kk < 0, kk * 0.5, kk)
        scale = 0.25
        out = b200.window_attention(qq, kk, v, scale=scale)
        ref, mass = reference(qq, kk, v, 0, 0, [700], [700], scale=scale)
        size = (qq.float().abs() @ kk.float().abs().transpose(2, 3)).amax() * scale
        u = 2.0 ** -8
        tol = u * ref.abs() + (u + 2.0 ** -13 + 2.0 ** -22 * size.item()) * mass + 1e-30   # a logit of size s is off by 2^-24 s and a sum's rounding
        assert ((out.double() - ref).abs() <= tol).all()


def test_streams_and_graphs(b200):
    g = torch.Generator(device="cuda").manual_seed(14)
    q, k, v = inputs(g, 2, 4, 2, 300, 300, 128, torch.bfloat16, True)
    here = b200.window_attention(q, k, v, window=64, sinks=2)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        there = b200.window_attention(q, k, v, window=64, sinks=2)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(here, there)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b200.window_attention(q, k, v, window=64, sinks=2)
    q.normal_(generator=g)
    graph.replay()
    ref, mass = reference(q, k, v, 64, 2, [300] * 2, [300] * 2)
    check(out, ref, mass)


def test_one_token_agrees_with_the_paged_form(b200):
    """The last row of a window over contiguous keys is the single-token form over pages of the same keys."""
    g = torch.Generator(device="cuda").manual_seed(15)
    n, rows, d = 700, 16, 128
    q, k, v = inputs(g, 1, 8, 2, n, n, d, torch.bfloat16, False)
    pages = -(-n // rows)
    kp, vp = (torch.zeros(pages, 2, rows, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)[None]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    b200.paged_append(k[0].transpose(0, 1), v[0].transpose(0, 1), kp, vp, table, lens, cu)
    for window, sinks in ((0, 0), (256, 4)):
        one = b200.paged_attention(q[:, :, -1], kp, vp, table, lens, window=window, sinks=sinks)
        all_ = b200.window_attention(q, k, v, window=window, sinks=sinks)
        ref, mass = reference(q[:, :, -1:], k, v, window, sinks, [1], [n])
        check(one[:, :, None], ref, mass)
        check(all_[:, :, -1:], ref, mass)


def test_inputs_that_cannot_be_read_in_place(b200):
    """K and V expanded over batches and heads, rows that start between 16-byte boundaries, a head dimension with a stride."""
    g = torch.Generator(device="cuda").manual_seed(16)
    q, k, v = inputs(g, 3, 4, 4, 130, 130, 64, torch.bfloat16, False)
    one = k[:1, :1].expand(3, 4, 130, 64)
    ref, mass = reference(q, one, v, 0, 0, [130] * 3, [130] * 3)
    check(b200.window_attention(q, one, v), ref, mass)
    odd = torch.randn(3 * 4 * 130 * 64 + 1, device="cuda", generator=g).bfloat16()[1:].view(3, 4, 130, 64)
    ref, mass = reference(odd, k, odd, 0, 0, [130] * 3, [130] * 3)
    check(b200.window_attention(odd, k, odd), ref, mass)
    across = torch.randn(3, 4, 64, 130, device="cuda", generator=g).bfloat16().transpose(2, 3)
    ref, mass = reference(across, k, across, 0, 0, [130] * 3, [130] * 3)
    check(b200.window_attention(across, k, across), ref, mass)


# Sizes at which a call takes each form: two query tiles a CTA (two heads of a group, two blocks of rows), one, and one with its keys
# split over clusters of 2, 4 and 8.
FORMS = [
    (2, 8, 2, 1500, 1500, 128, 0, 0),
    (1, 16, 16, 2000, 2000, 112, 700, 3),
    (1, 6, 2, 900, 1100, 64, 0, 0),
    (1, 32, 8, 300, 4000, 128, 0, 0),
    (1, 8, 1, 1000, 8000, 128, 0, 0),
    (1, 8, 1, 61, 4000, 80, 0, 0),
    (2, 4, 1, 33, 9000, 64, 5000, 200),
]


@pytest.mark.parametrize("bad", [None, float("nan"), float("inf")])
@pytest.mark.parametrize("shape", FORMS, ids=str)
def test_every_form_of_the_kernel(b200, shape, bad):
    """The form depends on the sizes alone; in each, a key or value that is not finite shows in the rows that see it, and in no other."""
    b, hq, hkv, sq, sk, d, window, sinks = shape
    g = torch.Generator(device="cuda").manual_seed(sq + sk)
    q, k, v = inputs(g, b, hq, hkv, sq, sk, d, torch.bfloat16, True)
    ref, mass = reference(q, k, v, window, sinks, [sq] * b, [sk] * b)
    if bad is None:
        out = b200.window_attention(q, k, v, window=window, sinks=sinks)
        check(out, ref, mass)
        assert torch.equal(out, b200.window_attention(q, k, v, window=window, sinks=sinks))
        return
    at = sk - sq + (2 * sq) // 3                          # seen by the later rows only
    pos = torch.arange(sq, device="cuda") + sk - sq
    seen = pos >= at
    if window > 0:
        seen &= pos < at + window
    k, v = k.clone(), v.clone()
    v[0, 0, at] = bad
    k[0, 0, at, 0] = bad
    out = b200.window_attention(q, k, v, window=window, sinks=sinks)
    check(out[0, :, ~seen], ref[0, :, ~seen], mass[0, :, ~seen])
    check(out[1:], ref[1:], mass[1:])
    check(out[:, hq // hkv:], ref[:, hq // hkv:], mass[:, hq // hkv:])
    assert not torch.isfinite(out[0, :hq // hkv][:, seen].float()).all(-1).any() if bad != bad else True


def test_ragged_lengths_in_a_large_call(b200):
    g = torch.Generator(device="cuda").manual_seed(17)
    nq, nk = [1000, 3, 700, 0, 129], [1000, 300, 900, 10, 129]
    q, k, v = inputs(g, 5, 16, 4, 1000, 1000, 128, torch.float16, True)
    lens = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (nq, nk)]
    for window, sinks in ((0, 0), (300, 130)):
        out = b200.window_attention(q, k, v, window=window, sinks=sinks, q_lens=lens[0], k_lens=lens[1])
        ref, mass = reference(q, k, v, window, sinks, nq, nk)
        check(out, ref, mass)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nats", [8.0, 12.0, 16.0])
@pytest.mark.parametrize("shape", [(1, 2, 1, 300, 300, 128, 0, 0), (2, 4, 4, 129, 129, 64, 0, 0), (1, 32, 8, 61, 1999, 128, 1024, 4), (1, 4, 1, 40, 3000, 80, 0, 0),
                                   (4, 8, 2, 2000, 2000, 128, 600, 1), (1, 32, 8, 2500, 2500, 64, 0, 0)], ids=str)
def test_keys_far_below_the_heaviest(b200, shape, nats, dt):
    """A first key with nearly all of the weight and no value, seen by every row: the results are made of keys whose weights, down to e^-17
    of the heaviest, P holds as normal numbers of fp16; the values are large, so that the results are normal numbers too."""
    b, hq, hkv, sq, sk, d, window, sinks = shape
    g = torch.Generator(device="cuda").manual_seed(sq + d)
    q, k, v = inputs(g, b, hq, hkv, sq, sk, d, torch.float32, False)
    k, v = k * 0.02, (v.abs() + 0.5) * 4096
    q[..., 0], k[..., 0] = 4.0, 0.0
    k[:, :, 0], v[:, :, 0] = 0.0, 0.0
    k[:, :, 0, 0] = nats / 4
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    out = b200.window_attention(q, k, v, window=window, sinks=sinks, scale=1.0)
    ref, mass = reference(q, k, v, window, sinks, [sq] * b, [sk] * b, scale=1.0)
    check(out, ref, mass)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sq,sk", [(700, 700), (40, 3000), (4000, 4000)])
@pytest.mark.parametrize("size", [2.0 ** e for e in (4, 12, 20, 23, 24, 25, 26, 27, 28, 30, 60)], ids=str)
def test_logits_that_32_bits_hold_coarsely(b200, sq, sk, dt, size):
    """Logits whose neighbours in 32 bits are up to many nats apart, rising along the keys: every result is a mean of the values."""
    g = torch.Generator(device="cuda").manual_seed(32)
    q, _, v = inputs(g, 1, 4, 2, sq, sk, 64, dt, False)
    q = (q.float().abs() + 0.5).to(dt)
    k = (torch.linspace(3.0, 4.0, sk, device="cuda")[:, None] * torch.ones(64, device="cuda")).to(dt).expand(1, 2, sk, 64)
    out = b200.window_attention(q, k, v, scale=size / (4 * 64)).float().view(1, 2, 2, sq, 64)
    room = 2.0 ** -6 * v.float().abs().amax()            # roundings of P, of its sum and of the result
    top, low = (t[:, :, None, sk - sq:] for t in (v.float().cummax(2).values, v.float().cummin(2).values))
    assert torch.isfinite(out).all() and (out >= low - room).all() and (out <= top + room).all()


# ----------------------------------------------------------------------------- the forms by name
# sizes -> (query tiles a CTA, CTAs that share an item's keys, the two tiles are of two heads) on 148 SMs
NAMED = [
    ((4, 8, 2, 900, 900, 128, 200, 2), (2, 1, 1)), ((5, 16, 4, 1000, 1000, 112, 0, 0), (2, 1, 1)),
    ((4, 20, 4, 193, 977, 80, 0, 4), (2, 1, 0)), ((4, 10, 2, 404, 1013, 128, 1000, 1), (2, 1, 0)),
    ((4, 16, 4, 280, 1345, 64, 0, 130), (2, 1, 1)), ((2, 16, 8, 591, 1478, 48, 1000, 4), (2, 1, 1)), ((4, 20, 4, 149, 2454, 48, 0, 4), (2, 1, 0)),
    ((7, 4, 2, 400, 450, 80, 0, 0), (1, 1, 0)), ((1, 16, 4, 2000, 2000, 64, 0, 0), (1, 1, 0)), ((8, 12, 12, 500, 500, 128, 130, 1), (1, 1, 0)),
    ((8, 12, 4, 28, 2252, 128, 0, 130), (1, 2, 0)), ((3, 8, 8, 278, 1100, 80, 1000, 1), (1, 2, 0)), ((2, 40, 8, 53, 1155, 64, 0, 4), (1, 2, 0)),
    ((1, 20, 4, 131, 555, 80, 0, 0), (1, 4, 0)), ((3, 12, 4, 27, 577, 128, 1000, 4), (1, 4, 0)), ((2, 24, 8, 21, 793, 64, 300, 130), (1, 4, 0)),
    ((4, 1, 1, 20, 514, 80, 300, 130), (1, 8, 0)), ((3, 8, 2, 60, 3000, 128, 0, 0), (1, 8, 0)), ((3, 8, 2, 60, 3000, 64, 0, 0), (1, 8, 0)),
]


def form_of(b, hq, hkv, sq, sk, d, window, sinks):
    import ctypes

    from tensorrt_b200 import _lib

    form = (ctypes.c_int32 * 3)()
    assert _lib.load().b200q_window_attention_form(b, hq, hkv, sq, sk, d, window, sinks, ctypes.byref(form)) == 0
    return tuple(form)


needs_148 = pytest.mark.skipif("torch.cuda.is_available() and torch.cuda.get_device_properties(0).multi_processor_count != 148",
                               reason="the choice of a form goes by the SMs")


@needs_148
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,form", NAMED, ids=str)
def test_each_form_on_its_own(b200, shape, form, dt):
    """Whole and ragged sequences, some with fewer key tiles than a cluster has CTAs, some without queries or keys."""
    assert form_of(*shape) == form
    b, hq, hkv, sq, sk, d, window, sinks = shape
    g = torch.Generator(device="cuda").manual_seed(sq + sk)
    q, k, v = inputs(g, b, hq, hkv, sq, sk, d, dt, True)
    out = b200.window_attention(q, k, v, window=window, sinks=sinks)
    check(out, *reference(q, k, v, window, sinks, [sq] * b, [sk] * b))
    for turn in range(3):
        nq = [(sq, sq // 2 + 1, 1, 0, sq - 1)[(i + turn) % 5] for i in range(b)]
        nk = [(100, sk, sk // 3, 7, sk - 3, 0, 129)[(i + 2 * turn) % 7] for i in range(b)]
        lens = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (nq, nk)]
        qq, kk, vv = q.clone(), k.clone(), v.clone()
        for i in range(b):
            qq[i, :, nq[i]:], kk[i, :, nk[i]:], vv[i, :, nk[i]:] = float("nan"), float("nan"), float("inf")
        out = b200.window_attention(qq, kk, vv, window=window, sinks=sinks, q_lens=lens[0], k_lens=lens[1])
        check(out, *reference(q, k, v, window, sinks, nq, nk))


@needs_148
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,form", NAMED, ids=str)
def test_each_form_with_values_that_are_not_finite(b200, shape, form, dt):
    """A value that is not finite is the whole result of the rows that see it; a key that makes their logit infinite makes them NaN or, at
    -inf, is a key less.  Other rows and heads are as they were."""
    b, hq, hkv, sq, sk, d, window, sinks = shape
    g = torch.Generator(device="cuda").manual_seed(sq - sk)
    q, k, v = inputs(g, b, hq, hkv, sq, sk, d, dt, False)
    group = hq // hkv
    ref, mass = reference(q, k, v, window, sinks, [sq] * b, [sk] * b)
    at = sk - sq + (2 * sq) // 3                          # seen by the later rows only
    pos, j = torch.arange(sq, device="cuda") + sk - sq, torch.arange(sk, device="cuda")
    seen = j <= pos[:, None]
    if window > 0:
        seen = seen & ((j > pos[:, None] - window) | (j < sinks))
    hit = seen[:, at]
    assert hit.any() and not hit.all()

    def others(out):
        check(out[:, group:], ref[:, group:], mass[:, group:])
        check(out[1:], ref[1:], mass[1:])
        check(out[0, :group, ~hit], ref[0, :group, ~hit], mass[0, :group, ~hit])
        return out[0, :group, hit]

    for bad in (float("nan"), float("inf"), -float("inf")):
        vv = v.clone()
        vv[0, 0, at] = bad
        mine = others(b200.window_attention(q, k, vv, window=window, sinks=sinks))
        assert (mine.isnan() if bad != bad else mine == bad).all()
        vv = v.clone()
        vv[0, 0, at, 5] = bad                             # one element of it: the others are as they were
        mine = others(b200.window_attention(q, k, vv, window=window, sinks=sinks))
        assert (mine[..., 5].isnan() if bad != bad else mine[..., 5] == bad).all()
        rest = [x for x in range(d) if x != 5]
        check(mine[..., rest], ref[0, :group, hit][..., rest], mass[0, :group, hit][..., rest])
        kk = k.clone()
        kk[0, 0, at, 0] = bad
        mine = others(b200.window_attention(q, kk, v, window=window, sinks=sinks))
        sign = q[0, :group, hit, 0].float() * bad
        gone = sign == -math.inf
        assert mine[~gone].isnan().all()
        for h in range(group):
            s = (q[0, h].double() @ k[0, 0].double().T / math.sqrt(d)).masked_fill(~seen | (j == at), -math.inf)[hit]
            p = torch.softmax(s, -1)[gone[h]]
            check(mine[h][gone[h]], p @ v[0, 0].double(), p @ v[0, 0].double().abs())
