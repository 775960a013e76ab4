"""Attention over shared prefixes where its arithmetic or its loads are at an edge, against the 64-bit restatement of tests/test_gpu_shared_prefix.py and by its
bounds."""
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
