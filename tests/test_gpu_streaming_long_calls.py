"""StreamingController decoding under a budget, with calls of more tokens than the operators take at once."""
import pytest
import torch

from test_gpu_streaming_decode import call, start
from test_gpu_streaming_model import KV_HEADS, N, model, prompt  # noqa: F401

pytestmark = pytest.mark.gpu


def test_long_calls_match_the_growing_cache(model, prompt):  # noqa: F811
    toks = [(7 * i + 3) % 500 for i in range(300)]
    ctl, first = start(model, prompt, backend="full", budget=4 * N)
    dense = torch.cat([call(model, toks[:290], N), call(model, toks[290:], N + 290)])
    ctl.restore()
    ctl, _ = start(model, prompt, backend="full", budget=4 * N, decode_budget=N + 400)
    got = torch.cat([call(model, toks[:290], N), call(model, toks[290:], N + 290)])
    states = list(ctl.states.values())
    ctl.restore()
    # bf16 activations, as in test_gpu_streaming_decode
    torch.testing.assert_close(got, dense, atol=0.03 * first.abs().max().item(), rtol=0.03)
    for s in states:
        assert s["cache"].lengths.tolist() == [[N + 300] * KV_HEADS]
        assert s["cache"].positions[0, 0, :N + 300].tolist() == list(range(N + 300))


def test_the_budget_holds_after_a_long_call(model, prompt):  # noqa: F811
    ctl, _ = start(model, prompt, backend="fused", budget=300, decode_budget=200, reserved_recent=16)
    assert torch.isfinite(call(model, [i % 400 for i in range(333)], N)).all()
    for s in ctl.states.values():
        assert s["cache"].lengths.tolist() == [[200] * KV_HEADS]
        newest = s["cache"].positions[..., :200].sort(-1).values[..., -16:]
        assert torch.equal(newest, torch.arange(N + 317, N + 333, dtype=torch.int32, device="cuda").expand_as(newest))
    ctl.restore()
