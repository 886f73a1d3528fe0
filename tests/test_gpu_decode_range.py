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
