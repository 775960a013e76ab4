"""Continuations of a prompt on several streams: nothing that a call makes on the side is read by another before it is there, nor given away before it has been read."""
import pytest
import torch

from test_gpu_shared_prefix import made, on_device

pytestmark = pytest.mark.gpu

CASE = ([(320, [3, 4, 5]), (48, [1, 2])], [40], 2, 4, 64, 16, torch.bfloat16, torch.bfloat16, "hnd", False)
SLEEP = 200_000_000                                         # clocks: a tenth of a second


@pytest.fixture
def call(b200):
    q, kp, vp, _, _, table, lens, members, tokens = made(CASE)
    n = on_device(lens)
    f = lambda prefix: b200.shared_prefix_attention(q, kp, vp, table, n, prefix)  # noqa: E731
    new = lambda t=tokens: b200.SharedPrefix(members, t, 6)  # noqa: E731
    want = f(new())
    torch.cuda.synchronize()
    return f, new, want


def test_a_second_call_beside_a_first_one_that_waits(call):
    """The first call makes the plan; the stream that it is on has other work to do."""
    f, new, want = call
    for _ in range(3):                                      # streams may share a queue of the device, which orders them by itself: not all of these
        busy, other = torch.cuda.Stream(), torch.cuda.Stream()
        prefix = new()
        with torch.cuda.stream(busy):
            torch.cuda._sleep(SLEEP)
            first = f(prefix)
        with torch.cuda.stream(other):
            second = f(prefix)
        other.synchronize()
        assert torch.equal(second, want)
        busy.synchronize()
        assert torch.equal(first, want)


def test_groups_that_are_gone_before_their_call_has_run(call):
    """A call that waits for its stream reads the plan of groups that nobody holds any more, and that others of the same size have followed."""
    f, new, want = call
    for _ in range(3):
        busy, prefix = torch.cuda.Stream(), new()
        with torch.cuda.stream(busy):
            torch.cuda._sleep(SLEEP)
            out = f(prefix)
        del prefix
        others = [new([16, 32]) for _ in range(8)]
        for other in others:
            f(other)
        busy.synchronize()
        assert torch.equal(out, want)


def test_an_update_of_groups_that_are_gone(call):
    """The values of an update that waits for its stream do not reach a plan that has taken the place of its own."""
    f, new, want = call
    for _ in range(3):
        busy, prefix = torch.cuda.Stream(), new()
        f(prefix)
        with torch.cuda.stream(busy):
            torch.cuda._sleep(SLEEP)
            prefix.update([[0, 1]], [16])
        del prefix
        others = [new() for _ in range(8)]
        outs = [f(other) for other in others]
        busy.synchronize()
        outs += [f(other) for other in others]
        assert all(torch.equal(out, want) for out in outs)
