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


def test_a_call_of_more_tokens_than_drafts_goes_in_parts(monkeypatch):
    from flash_evict import streaming_adapter as A
    seen = []

    def attend(q, k, v, cache, *, tree, scale):
        assert tree is None and scale == 0.5
        seen.append(("attend", q.shape[2]))
        return q + 1, q[..., 0].float()

    def commit(cache, q, k, v, lse, accepted, positions, *, tree, scale, recency_decay):
        seen.append(("commit", accepted.tolist(), positions.tolist()))
        assert torch.equal(lse, q[..., 0].float()) and q.shape[2] == k.shape[2] == v.shape[2] == accepted.shape[1]

    monkeypatch.setattr(A, "tree_attention", attend)
    monkeypatch.setattr(A, "commit_tokens", commit)
    monkeypatch.setattr(A, "evict_tokens", lambda cache, budget, *, recent: seen.append(("evict", budget)))
    ctl = StreamingController(tiny_model(), decode_budget=8)
    try:
        for n, parts in ((1, [1]), (128, [128]), (129, [128, 1]), (300, [128, 128, 44])):
            seen.clear()
            state = {"cache": None, "next": torch.full((1, 1), 40, dtype=torch.int32)}
            q, kv = torch.randn(1, 4, n, 8), torch.randn(1, 2, n, 8)
            out = A._budgeted_attention(ctl, state, q, kv, kv, 0.5)
            assert torch.equal(out, q + 1) and int(state["next"]) == 40 + n
            assert seen[0::3] == [("attend", m) for m in parts] and seen[2::3] == [("evict", 8)] * len(parts)
            at = 40
            for m, (what, accepted, positions) in zip(parts, seen[1::3]):
                assert what == "commit" and accepted == [list(range(m))] and positions == [list(range(at, at + m))]
                at += m
    finally:
        ctl.restore()
