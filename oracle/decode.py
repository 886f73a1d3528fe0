"""Plain 64-bit restatement of the decode operators, row by row (torch on the CPU).

tree_attention: softmax over the cached tokens of a row and the drafts its tree
mask names, and the log of the row's sum; commit: the accepted drafts' weight on
every cached token and on each other, and the appended rows; evict: the kept
tokens by reserved suffix, weight and slot, each hole below the budget filled by
the next kept token above it.
"""
import math

import torch


def visible(t, tree, b):
    """[T, T] bool: draft t sees draft j."""
    if tree is None:
        return torch.ones(t, t, dtype=torch.bool).tril()
    return (tree if tree.ndim == 2 else tree[b]).cpu()


def tree_attention(q, k_new, v_new, k, v, lengths, tree=None, scale=None):
    """(out, lse, spread): spread = sum p |v|, the scale of out's rounding errors."""
    q, k_new, v_new, k, v = (x.detach().cpu().double() for x in (q, k_new, v_new, k, v))
    b, hq, t, d = q.shape
    hk = k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out, spread = torch.zeros(b, hq, t, d, dtype=torch.float64), torch.zeros(b, hq, t, d, dtype=torch.float64)
    lse = torch.full((b, hq, t), -math.inf, dtype=torch.float64)
    for i in range(b):
        sees = visible(t, tree, i)
        for j in range(hq):
            h = j // (hq // hk)
            n = min(max(int(lengths[i, h]), 0), k.shape[2])
            for r in range(t):
                who = sees[r].nonzero()[:, 0]
                keys = torch.cat([k[i, h, :n], k_new[i, h, who]])
                if not len(keys):
                    continue
                values = torch.cat([v[i, h, :n], v_new[i, h, who]])
                x = scale * (keys @ q[i, j, r])
                lse[i, j, r] = torch.logsumexp(x, 0)
                p = torch.exp(x - lse[i, j, r])
                out[i, j, r] = (p[:, None] * values).sum(0)
                spread[i, j, r] = (p[:, None] * values.abs()).sum(0)
    return out, lse, spread
