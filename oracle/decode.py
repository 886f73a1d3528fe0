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


def commit(k, v, lengths, mass, norms, positions, q, k_new, v_new, lse, accepted, new_positions, tree=None, scale=None, decay=0.0):
    """The cache after the accepted drafts, per row: dict (b, h) -> (k, v, mass, norms, positions); norms None: weights unscaled.

    Floating inputs are taken as they are and computed with in 64 bits; an accepted
    entry outside [0, T) is none, and rows past the capacity are dropped.
    """
    cpu = lambda x: None if x is None else x.detach().cpu()  # noqa: E731
    k, v, mass, norms, positions, q, k_new, v_new, lse = map(cpu, (k, v, mass, norms, positions, q, k_new, v_new, lse))
    b, hq, t, d = q.shape
    hk, cap = k.shape[1:3]
    g = hq // hk
    scale = d ** -0.5 if scale is None else scale
    rows = {}
    for i in range(b):
        sees = visible(t, tree, i)
        path = [j for j in accepted[i].tolist() if 0 <= j < t]
        m = len(path)
        for h in range(hk):
            n = min(max(int(lengths[i, h]), 0), cap)
            new_norm = v_new[i, h, path].double().abs().sum(-1)
            size = torch.ones(n + m, dtype=torch.float64) if norms is None else torch.cat([norms[i, h, :n].double(), new_norm])
            got = torch.cat([mass[i, h, :n].double() * math.exp(-decay * m), torch.zeros(m, dtype=torch.float64)])
            keys = torch.cat([k[i, h, :n], k_new[i, h, path]]).double()
            for r, j in enumerate(path):
                may = torch.cat([torch.ones(n, dtype=torch.bool), sees[j, path]])
                for head in range(h * g, h * g + g):
                    if lse[i, head, j] == -math.inf:
                        continue
                    x = scale * (keys @ q[i, head, j].double()) - lse[i, head, j].double()
                    p = torch.where(may, torch.exp(x), torch.zeros((), dtype=torch.float64))
                    got = got + size * math.exp(-decay * (m - 1 - r)) * p
            keep = min(n + m, cap)
            rows[i, h] = (torch.cat([k[i, h, :n], k_new[i, h, path]])[:keep], torch.cat([v[i, h, :n], v_new[i, h, path]])[:keep],
                          got[:keep], None if norms is None else size[:keep],
                          torch.cat([positions[i, h, :n], new_positions[i, path].cpu()])[:keep])
    return rows


def evict_slots(mass, positions, budget, recent):
    """For one row's live mass and positions: the source slot of every slot after the eviction."""
    n = len(mass)
    if n <= budget:
        return list(range(n))
    newest = max(positions)

    def order(i):
        if positions[i] > newest - recent:
            return (0, 0.0, i)
        return (1, 0.0, i) if math.isnan(mass[i]) else (2, -mass[i], i)

    kept = set(sorted(range(n), key=order)[:budget])
    movers = iter(sorted(i for i in kept if i >= budget))
    return [i if i in kept else next(movers) for i in range(budget)]
