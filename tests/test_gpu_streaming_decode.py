"""StreamingController decoding under a budget, on the small random-init Qwen2 of test_gpu_streaming_model.

With room for everything the budgeted decode agrees with the dense model; a
tree of drafts gives each draft the logits of its own path and accepting a path
leaves the caches as decoding it token by token would; under a small budget
every layer keeps exactly its budget, the newest tokens among it.
"""
import pytest
import torch

from flash_evict.streaming_adapter import StreamingController
from test_gpu_streaming_model import HEAD_DIM, KV_HEADS, N, model, prompt  # noqa: F401

pytestmark = pytest.mark.gpu


def call(m, tokens, first, depth=None):
    pos = first + (torch.arange(len(tokens)) if depth is None else torch.tensor(depth))
    ids = torch.tensor([tokens], device="cuda")
    with torch.no_grad():
        return m(ids, position_ids=pos[None].cuda(), use_cache=False).logits[0].float()


def start(m, prompt, **kw):
    ctl = StreamingController(m, **kw)
    with torch.no_grad():
        logits = m(prompt, use_cache=False).logits[0, -1].float()
    ctl.finish_prefill()
    return ctl, logits


def test_budgeted_decode_matches_the_growing_cache(model, prompt):
    toks = [3, 77, 500, 12]
    ctl, first = start(model, prompt, backend="full", budget=4 * N)
    dense = [call(model, [t], N + i)[0] for i, t in enumerate(toks)]
    ctl.restore()
    scale = first.abs().max().item()
    for chunk in (1, 2, 4):
        for backend, budget in (("full", 4 * N), ("fused", N)):
            ctl, again = start(model, prompt, backend=backend, budget=budget, decode_budget=2 * N)
            assert torch.equal(again, first)
            got = torch.cat([call(model, toks[i:i + chunk], N + i) for i in range(0, 4, chunk)])
            lengths = [s["cache"].lengths.tolist() for s in ctl.states.values()]
            positions = [s["cache"].positions[0, 0, N:N + 4].tolist() for s in ctl.states.values()]
            ctl.restore()
            torch.testing.assert_close(got, torch.stack(dense), atol=0.03 * scale, rtol=0.03)
            assert all(n == [[N + 4] * KV_HEADS] for n in lengths) and all(p == [N, N + 1, N + 2, N + 3] for p in positions)


def test_a_tree_of_drafts(model, prompt):
    # root 5 with children 9 and 40; 40 has child 2
    tokens, parents, depth = [5, 9, 40, 2], [-1, 0, 0, 2], [0, 1, 1, 2]
    tree = torch.zeros(4, 4, dtype=torch.bool)
    for j, p in enumerate(parents):
        if p >= 0:
            tree[j] = tree[p]
        tree[j, j] = True
    kw = dict(backend="fused", budget=512, decode_budget=600, scoring={"recency_decay": 0.1})
    ctl, first = start(model, prompt, **kw)
    with pytest.raises(ValueError, match="No drafts"):
        ctl.accept([0])
    ctl.draft(tree.cuda())
    drafts = call(model, tokens, N, depth)
    ctl.accept([0, 2])
    after = call(model, [33], N + 2)[0]
    cache = {i: s["cache"] for i, s in ctl.states.items()}
    ctl.restore()
    scale = first.abs().max().item()
    ctl, _ = start(model, prompt, **kw)
    chain = torch.cat([call(model, [5], N), call(model, [40], N + 1), call(model, [33], N + 2)])
    for i, s in ctl.states.items():
        assert s["cache"].lengths.tolist() == cache[i].lengths.tolist() == [[515] * KV_HEADS]
        assert torch.equal(s["cache"].positions[..., :515], cache[i].positions[..., :515])
        torch.testing.assert_close(s["cache"].mass[..., :515], cache[i].mass[..., :515], rtol=0.05, atol=0.05)
    ctl.restore()
    # bf16 activations: rounding differs between a call of 1 and of 4 tokens
    torch.testing.assert_close(torch.stack([drafts[0], drafts[2], after]), chain, atol=0.03 * scale, rtol=0.03)


@pytest.mark.parametrize("backend", ["fused", "snap", "full"])
def test_the_budget_holds(model, prompt, backend):
    ctl, _ = start(model, prompt, backend=backend, budget=300, decode_budget=256, reserved_recent=16)
    for s in ctl.states.values():
        assert s["cache"].lengths.tolist() == [[256] * KV_HEADS]
        newest = s["cache"].positions[..., :256].sort(-1).values[..., -16:]
        assert torch.equal(newest, torch.arange(N - 16, N, dtype=torch.int32, device="cuda").expand_as(newest))
    for i in range(20):
        assert torch.isfinite(call(model, [i, 7], N + 2 * i)).all()
    for s in ctl.states.values():
        cache = s["cache"]
        assert cache.lengths.tolist() == [[256] * KV_HEADS] and cache.k.shape[-1] == HEAD_DIM
        pos = cache.positions[..., :256].sort(-1).values
        assert (pos[..., 1:] > pos[..., :-1]).all()
        assert torch.equal(pos[..., -16:], torch.arange(N + 24, N + 40, dtype=torch.int32, device="cuda").expand_as(pos[..., -16:]))
        assert torch.isfinite(cache.mass[..., :256]).all() and (cache.mass[..., :256] >= 0).all()
    ctl.restore()
