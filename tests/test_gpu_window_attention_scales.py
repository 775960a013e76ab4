"""Attention with a window where the products of queries and keys are far beyond one and the scale brings the logits back, by the bounds of
tests/test_gpu_window_attention.py."""
import pytest
import torch

from test_gpu_window_attention import check, inputs, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [20, 50, 58])
@pytest.mark.parametrize("shape", [(2, 6, 2, 257, 400, 80, 0, 0), (1, 20, 4, 131, 555, 80, 100, 3), (1, 4, 2, 1500, 1500, 64, 0, 0)], ids=str)
def test_scales_far_below_one(b200, shape, power):
    b, hq, hkv, sq, sk, d, window, sinks = shape
    g = torch.Generator(device="cuda").manual_seed(power)
    q, k, v = inputs(g, b, hq, hkv, sq, sk, d, torch.bfloat16, False)
    q, k, scale = q * 2.0 ** power, k * 2.0 ** power, 0.125 * 4.0 ** -power
    ref, mass = reference(q, k, v, window, sinks, [sq] * b, [sk] * b, scale)
    check(b200.window_attention(q, k, v, window=window, sinks=sinks, scale=scale), ref, mass)
