"""StreamingController's drafts on the host: which call's drafts an acceptance takes."""
import pytest
import torch

from flash_evict.streaming_adapter import StreamingController
from test_streaming_cpu import tiny_model


def test_a_new_tree_drops_the_drafts_of_the_last_one():
    ctl = StreamingController(tiny_model(), decode_budget=8)
    try:
        ctl.finish_prefill()
        ctl.states = {0: {}, 1: {}}
        ctl.draft(torch.eye(2, dtype=torch.bool))
        for state in ctl.states.values():
            state["drafts"] = ("of the first tree",)
        # another tree, whose call has not come: the first tree's drafts are not its drafts
        ctl.draft(torch.eye(4, dtype=torch.bool))
        for path in ([3], []):
            with pytest.raises(ValueError, match="No drafts"):
                ctl.accept(path)
        assert ctl.states == {0: {}, 1: {}} and ctl.tree.shape == (4, 4)
    finally:
        ctl.restore()
