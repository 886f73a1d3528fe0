"""Decode operators at the ends of the number formats' range.

Tolerance of the light tokens' test: test_gpu_decode's for the output, u * (sum
p|v| + |out|) + 2 * (eps + 2^-20) * sum p|v| with eps the logits' error, but with
fp16's absolute spacing of the weights at 2^-32 of the row's largest, once a token.
"""
import math

import pytest
import torch

from flash_evict.decode import KVCache, commit_tokens, tree_attention
from test_gpu_decode import U, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,hq,hk,d,t,below", [(131072, 4, 1, 128, 1, 17.5), (2000, 28, 4, 128, 1, 19.0), (3000, 8, 2, 64, 100, 18.0),
                                               (1500, 4, 2, 256, 2, 17.5)])
def test_many_light_tokens_beside_a_heavy_one(dtype, n, hq, hk, d, t, below):
    # One key `below` nats above all others, whose values are 1 and its own 0: the
    # output is the light tokens' share of the weight.
    q, kn, vn, cache, gen = make(61, 1, hq, hk, d, n + 8, t, dtype, n)
    q.zero_(), kn.zero_(), vn.fill_(1.0)
    q[..., 0] = 1.0
    cache.k[:, :, :n], cache.v[:, :, :n] = 0.0, 1.0
    cache.k[:, :, :n, 1:] = (0.25 * torch.randn(1, hk, n, d - 1, generator=gen)).to(dtype).cuda()  # (not seen by the queries)
    cache.k[:, :, 7, 0], cache.v[:, :, 7] = below, 0.0
    out, lse = tree_attention(q, kn, vn, cache, scale=1.0)
    top = float(torch.tensor(below, dtype=dtype))
    others = n - 1 + torch.arange(1, t + 1, dtype=torch.float64, device="cuda")[:, None]
    share = others * math.exp(-top) / (1 + others * math.exp(-top))
    tol = 2 * U[dtype] * 1.01 * share + 2 * (2.0 ** -22 * top + 2.0 ** -20) * share + (2.0 ** -32 * others if dtype == torch.float16 else 0.0)
    err = (out.double() - share).abs()
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,d,t,took", [(4, 2, 128, 1, 1), (28, 4, 64, 5, 3), (3, 1, 80, 2, 2), (8, 1, 256, 3, 3)])
def test_keys_of_minus_infinite_score_add_nothing(dtype, hq, hk, d, t, took):
    # A key that overflowed: its score is -inf for every query, its probability 0.
    n = 300
    q, kn, vn, cache, gen = make(62, 1, hq, hk, d, n + 8, t, dtype, n)
    q[..., 0] = q[..., 0].abs() + 1
    cache.k[:, :, [5, 127, 128, 299], 0] = -torch.inf
    mass = torch.rand(1, hk, n + 8, generator=gen).cuda()
    pos = torch.arange(n + 8, dtype=torch.int32, device="cuda").expand(1, hk, n + 8).contiguous()
    cache = KVCache(cache.k, cache.v, cache.lengths, mass.clone(), pos)
    out, lse = tree_attention(q, kn, vn, cache)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    accepted = torch.arange(took, dtype=torch.int32, device="cuda")[None]
    commit_tokens(cache, q, kn, vn, lse, accepted, torch.full((1, t), n, dtype=torch.int32, device="cuda"))
    assert torch.equal(cache.mass[:, :, [5, 127, 128, 299]], mass[:, :, [5, 127, 128, 299]])
    live = cache.mass[:, :, :n + took]
    assert torch.isfinite(live).all()
    # the accepted queries' weights add up to one each (2^-18: as for the mass in test_gpu_decode_cache)
    # but for what goes to drafts that were not accepted, which none of these sees
    assert ((live.sum(-1) - mass[:, :, :n].sum(-1) - took * (hq // hk)).abs() <= 2.0 ** -18 * live.sum(-1)).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,hq,t,parts", [(256, 1, 1, 4), (256, 40, 2, 2), (128, 4, 1, 4)])
def test_committed_weights_do_not_lean(dtype, d, hq, t, parts):
    """The mean error of equally heavy keys' weights, whose random part averages out.

    A sum of 16 channels cut off to FP32 loses half a last place on average, at most
    2^-24 of the sum so far; over a part's d / 16 / parts steps, with terms of one sign
    and size, that is (steps + 1) / 2 * 2^-24 of the score.  Half a unit more covers
    the rounding of scale * log2(e) and ex2.  (parts: the fewest that a score may be
    summed in.)
    """
    n, scale = 4096, 1 / 16
    gen = torch.Generator().manual_seed(63)
    spread = lambda *shape: (1 + 0.3 * (2 * torch.rand(*shape, generator=gen) - 1)) * (40 / (scale * d)) ** 0.5  # noqa: E731
    q, k, kn = (spread(1, h, m, d).to(dtype).cuda() for h, m in ((hq, t), (1, n + 2), (1, t)))
    vn = torch.zeros_like(kn)
    s = scale * (q[0].double() @ k[0, 0, :n].double().T)  # [hq, t, n]
    # row sums whose product with log2(e) FP32 holds exactly, or nearly
    near = (s.mean() + math.log(n)).float() * (1 + torch.arange(4096, device="cuda") * 2.0 ** -23).float()
    bias = near.double() * math.log2(math.e)
    lse = near[(bias - bias.float().double()).abs().argmin()].expand(1, hq, t).contiguous()
    book = (torch.full((1, 1), n, dtype=torch.int32, device="cuda"), torch.zeros(1, 1, n + 2, device="cuda"),
            torch.zeros(1, 1, n + 2, dtype=torch.int32, device="cuda"))
    cache = KVCache(k, torch.zeros_like(k), *book)
    accepted = torch.arange(t, dtype=torch.int32, device="cuda")[None]
    commit_tokens(cache, q, kn, vn, lse, accepted, torch.full((1, t), n, dtype=torch.int32, device="cuda"), scale=scale)
    want = torch.exp(s - lse[0, 0, 0].double()).sum((0, 1))
    lean = (cache.mass[0, 0, :n].double() / want - 1).mean().item()
    steps = d // 16 // parts
    assert abs(lean) <= ((steps + 1) / 2 + 0.5) * 2.0 ** -24 * s.mean().item(), lean / (2.0 ** -24 * s.mean().item())
