"""`token_log_probs` over the whole range of scales and logits, against torch in 64 bits, by the bounds of tests/test_gpu_token_scores.py.  These count two
roundings of z; a difference that is taken before the product has two more (the difference, and the product of the scale and the base's logarithm): together 4 x 2^-24 of
|z|, whose mean over a distribution is at most 18 here, 2^-18 of S beside the 2^-17.5 of the exponentials and sums.
"""
import math

import pytest
import torch

from test_gpu_token_scores import DTYPES, check, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("by", [0.0, 100.0, -3000.0, 30000.0, -50000.0])
@pytest.mark.parametrize("size", [4, 5003])
def test_a_constant_changes_nothing(b200, by, size):
    """The entropy of logits is that of the same logits with a number added to all: those that count in 16 bytes, which one thread sums, and anywhere."""
    g = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(64, size, device="cuda", generator=g) * 2 ** torch.linspace(-3, 2, 64, device="cuda")[:, None]
    check(b200, x + by, x.argmax(1), 4)
    check(b200, x + by, None, 1, 0.75)
    x[:, 4:] -= 50
    check(b200, x + by, x.argmax(1), 4)


@pytest.mark.parametrize("scale", [1e4, 1e5, 1e6, 1e7, 1e9])
@pytest.mark.parametrize("dt", DTYPES, ids=str)
def test_scales_that_leave_the_largest_alone(b200, dt, scale):
    """A temperature next to zero: the product of a logit and the scale is far beyond what 32 bits hold to a unit, differences are not."""
    g = torch.Generator(device="cuda").manual_seed(11)
    x = logits(g, 24, 32000, dt).clone()
    x[1, 31999] = x[1].max()                                # two maxima
    x[2, :200] = x[2].max()
    x[3] = x[3] / 1024
    check(b200, x, x.float().argmax(1), 8, scale)
    check(b200, x[:, :9], x[:, :9].float().argmin(1), 3, scale)


@pytest.mark.parametrize("rows,size", [(3, 4), (2, 33000), (700, 5000)])
@pytest.mark.parametrize("dt,large", [(torch.float32, 1e6), (torch.float32, 3e8), (torch.float32, -1e9), (torch.float32, 1e25), (torch.bfloat16, 1e6), (torch.bfloat16, -3e8),
                                      (torch.float16, 6e4), (torch.float16, -6e4)], ids=str)
def test_large_logits_close_to_one_another(b200, dt, large, rows, size):
    at = torch.tensor(large, dtype=dt).float().item()
    step = 2.0 ** (math.frexp(at)[1] - {torch.float32: 24, torch.bfloat16: 8, torch.float16: 11}[dt])      # of neighbouring values
    i = torch.arange(size, device="cuda")
    for x in (torch.full((size,), at, device="cuda"), at - (i % 5) * step, at - (i % 7 != 3) * step):
        x = x.to(dt).expand(rows, size).contiguous()
        for scale in (1.0, 1 / step, 300.0):
            check(b200, x, torch.full((rows,), size - 1, device="cuda"), 3, torch.tensor(scale).item())


@pytest.mark.parametrize("scale", [1e9, 1e30])
@pytest.mark.parametrize("dt", DTYPES, ids=str)
def test_masked_logits_at_scales_that_leave_the_type(b200, dt, scale):
    """The product of the scale and what stands in for a masked logit is an infinity; its term is nothing all the same."""
    size = 9001
    x = torch.full((5, size), -math.inf, device="cuda")
    x[0, ::3] = 0.0                                         # equal ones: log of their number
    x[1, 5:8] = 0.0
    x[2, ::2] = -1.0 / scale
    x[2, ::40] = 0.0
    x[3, 4] = 2.0 ** -100
    x[4] = torch.where(torch.arange(size, device="cuda") % 2 == 0, 0.0, torch.finfo(dt).min)
    check(b200, x.to(dt), torch.full((5,), 4, device="cuda"), 3, torch.tensor(scale).item())


@pytest.mark.parametrize("dt", DTYPES, ids=str)
def test_the_largest_scales(b200, dt):
    """Up to the type's largest: the scale times log2 e is beyond it, the products are not."""
    size, scale = 3001, 1.75 * 2.0 ** 127
    x = torch.zeros(4, size, device="cuda")
    x[1, 1::2] = -math.inf
    x[2, 1::2] = -2.0 ** -127
    x[3, 7] = 1.0
    check(b200, x.to(dt), torch.full((4,), 7, device="cuda"), 3, scale)
