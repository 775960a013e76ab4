"""CPU checks of continuations at their edges: groups that hold nothing, calls that fail on the way."""
import pytest
import torch


@pytest.mark.parametrize("batch,members,tokens", [(4, [], []), (4, [[0]], [64]), (4, [[1, 2]], [0]), (1, [], []), (0, [], [])])
def test_an_update_where_nothing_is_shared(b200, batch, members, tokens):
    prefix = b200.SharedPrefix(members, tokens, batch, device="cpu")
    plan = prefix.plan(8, 2)
    assert prefix.groups == 0 and plan.numel() == 0
    for now in ((members, tokens), ([], []), ([[0]] * min(batch, 1), [9] * min(batch, 1))):
        prefix.update(*now)
        assert prefix.tokens == 0 and prefix.plan(8, 2) is plan
    if batch > 1:
        with pytest.raises(ValueError):
            prefix.update([[0, 1]], [8])
        assert prefix.tokens == 0


@pytest.mark.parametrize("largest", [None, 0, 1])
def test_room_for_groups_of_nobody(b200, largest):
    """Groups of up to one sequence hold nothing that is shared: a call has to be possible all the same."""
    prefix = b200.SharedPrefix([], [], 4, device="cpu", groups=2, largest=largest)
    assert prefix.groups == 0 and prefix.plan(8, 2).numel() == 0
    prefix.update([[1]], [50])
    with pytest.raises(ValueError):
        prefix.update([[0, 1]], [50])
