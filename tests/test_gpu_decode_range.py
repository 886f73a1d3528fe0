"""Decode operators at the ends of the number formats' range.

Tolerance of the light tokens' test: test_gpu_decode's for the output, u * (sum
p|v| + |out|) + 2 * (eps + 2^-20) * sum p|v| with eps the logits' error, but with
fp16's absolute spacing of the weights at 2^-32 of the row's largest, once a token.
"""
import math

import pytest
import torch

from flash_evict.decode import tree_attention
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
