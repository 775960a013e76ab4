"""`token_log_probs` over the whole range of scales and logits, against torch in 64 bits, by the bounds of tests/test_gpu_token_scores.py.
"""
import pytest
import torch

from test_gpu_token_scores import check

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
