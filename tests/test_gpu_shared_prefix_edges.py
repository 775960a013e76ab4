"""Attention over shared prefixes where its arithmetic or its loads are at an edge, against the 64-bit restatement of tests/test_gpu_shared_prefix.py and by its
bounds."""
import ctypes

import pytest
import torch

from test_gpu_paged_cache import E4M3, check_out, raw
from test_gpu_shared_prefix import made, on_device, reference

pytestmark = pytest.mark.gpu


def attend(b200, case, q, kp, vp, ka, va, table, lens, members, tokens, **kw):
    return b200.shared_prefix_attention(q, kp, vp, table, on_device(lens), b200.SharedPrefix(members, tokens, len(lens)), k_amax=ka, v_amax=va, **kw)


@pytest.mark.parametrize("power", [20, 50, 58])
def test_scales_far_below_one(b200, power):
    """Products of queries and keys far beyond one under a scale that brings the logits back."""
    case = ([(700, [5, 9, 30])], [50], 2, 4, 64, 16, torch.bfloat16, torch.bfloat16, "hnd", False)
    q, kp, vp, ka, va, table, lens, members, tokens = made(case)
    big = 2.0 ** power
    q, kp, scale = q * big, kp * big, 0.125 / big / big
    ref, mass, _ = reference(q, kp, vp, table, lens, members, tokens, ka, va, scale)
    check_out(attend(b200, case, q, kp, vp, ka, va, table, lens, members, tokens, scale=scale), ref, mass)


@pytest.mark.parametrize("rows", [1, 3, 5, 7])
@pytest.mark.parametrize("dt,pt", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, E4M3), (torch.float16, E4M3)], ids=str)
def test_small_pages_under_many_rows(b200, dt, pt, rows):
    """Rows that no tensor map takes, several blocks of queries, tiles that end inside a page, holes among them."""
    case = ([(391, [3] * 19), (130, [1, 40, 2])], [21], 2, 16, 96, rows, dt, pt, "nhd", True)
    q, kp, vp, ka, va, table, lens, members, tokens = made(case)
    table[members[0][0], 17 % table.shape[1]] = -1
    table[members[1][2], 130 // rows + 1:] = 1 << 30
    ref, mass, used = reference(q, kp, vp, table, lens, members, tokens, ka, va)
    for t in (kp, vp):
        raw(t)[(~used)[:, None].expand(t.shape[:3])] = 0x7F if t.element_size() == 1 else float("nan")
    check_out(attend(b200, case, q, kp, vp, ka, va, table, lens, members, tokens), ref, mass)


@pytest.mark.parametrize("size", [2.0 ** 16, 2.0 ** 28, 2.0 ** 60])
@pytest.mark.parametrize("dt,pt", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, E4M3)], ids=str)
def test_the_largest_logit_takes_all(b200, dt, pt, size):
    """Under a large scale the result is the value of the largest logit.  32-bit sums of 64 products hold a logit to 64 x 2^-24 of the sum of their sizes at most: rows
    whose two largest are further apart than twice that, and by 64 under the scale, have one term."""
    case = ([(700, [5, 9]), (300, [1, 1, 8])], [77], 2, 4, 64, 16, dt, pt, "hnd", False)
    q, kp, vp, ka, va, table, lens, members, tokens = made(case)
    ref, mass, _ = reference(q, kp, vp, table, lens, members, tokens, ka, va, size)
    clear = torch.zeros(q.shape[:2], dtype=torch.bool)
    for b in range(len(lens)):
        at = torch.arange(lens[b], device="cuda")
        lead = next((m[0] for m in members if b in m), b)
        page = torch.where(at < next((t for m, t in zip(members, tokens) if b in m), 0), table[lead].long()[at // 16], table[b].long()[at // 16])
        for h in range(8):
            k = raw(kp)[page, h // 4, at % 16].view(kp.dtype).double() * (1.0 if ka is None else (ka.float() / 448).double()[h // 4 if ka.numel() > 1 else 0])
            x, sizes = k @ q[b, h].double(), k.abs() @ q[b, h].double().abs()
            two = x.topk(2).values
            clear[b, h] = two[0] - two[1] > 2 * 64 * 2.0 ** -24 * sizes.max() + 64 / size
    assert clear.float().mean() > 0.9
    out = attend(b200, case, q, kp, vp, ka, va, table, lens, members, tokens, scale=size)
    check_out(out[clear], ref[clear], mass[clear])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at", [0, 16, 32, 240])
def test_a_workspace_at_any_multiple_of_16_bytes(b200, d, at):
    """As callers of the C entry may have it; every buffer has exactly the bytes that are asked for, and what stands around them stays."""
    from tensorrt_b200 import _lib

    lib, i64 = _lib.load(), ctypes.c_int64
    case = ([(300, [5, 9, 30])], [50], 2, 4, d, 16, torch.bfloat16, torch.bfloat16, "hnd", False)
    q, kp, vp, _, _, table, lens, members, tokens = made(case)
    q, n, prefix = q.contiguous(), on_device(lens), b200.SharedPrefix(members, tokens, 4)
    want = b200.shared_prefix_attention(q, kp, vp, table, n, prefix)
    strides = (i64 * 3)(*kp.stride()[:3])
    cache = _lib.PagedCache(kp.data_ptr(), vp.data_ptr(), 2, 16, kp.shape[0], 2, d, strides, (i64 * 3)(*vp.stride()[:3]), None, None, 0)
    size = lib.b200q_shared_prefix_workspace_bytes(4, 8, 2, d, 1, 3)
    held = torch.full((1024 + size,), 0xA5, dtype=torch.uint8, device="cuda")
    start = -held.data_ptr() % 256 + 256 + at
    head = torch.zeros(lib.b200q_paged_attention_workspace_bytes(), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    rc = lib.b200q_shared_prefix_attention(q.data_ptr(), 2, (i64 * 2)(*q.stride()[:2]), ctypes.byref(cache), table.data_ptr(), table.stride(0), table.shape[1], n.data_ptr(), 4, 8,
                                           prefix.plan(8, 2).data_ptr(), 1, 3, d ** -0.5, out.data_ptr(), head.data_ptr(), head.numel(), held.data_ptr() + start, size,
                                           torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(out, want)
    assert (held[:start] == 0xA5).all() and (held[start + size:] == 0xA5).all()
