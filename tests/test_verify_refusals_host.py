"""What a verification step refuses before its forward, and what a refused layer
leaves behind; on the CPU, with stand-ins for the device side."""
import pytest
import torch

from specfit_amd.runtime import Eagle3DraftTree, LogitRules, verify_draft_tree


class _Cache:
    def get_seq_length(self, layer=0):
        return 5


def _no_forward(**kwargs):
    raise AssertionError("the forward was reached")


@pytest.mark.parametrize("more", ({}, dict(commit=False), dict(rules=LogitRules()),
                                  dict(allowed=torch.zeros((1, 4), dtype=torch.int32))))
def test_a_seed_that_is_no_token(more):
    """-1 is the pending seed where nothing was allowed: also a call without rules
    refuses it, before it can index the embedding."""
    tree = Eagle3DraftTree((), (), (), (), ())
    with pytest.raises(ValueError, match="seed"):
        verify_draft_tree(_no_forward, tree, torch.tensor([[-1]]), _Cache(), **more)
    with pytest.raises(ValueError, match="shape"):
        verify_draft_tree(_no_forward, tree, torch.tensor([-1, 3]), _Cache(), **more)
    with pytest.raises(AssertionError, match="forward"):
        verify_draft_tree(_no_forward, tree, torch.tensor([[0]]), _Cache(), **more)
