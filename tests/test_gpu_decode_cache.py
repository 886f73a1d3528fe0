"""commit_tokens and evict_tokens against the 64-bit oracle, and the decode step they form.

mass tolerance, relative (all terms are positive): the logits' FP32 error
2^-22 * scale * |q||k| (as in test_gpu_decode), the rounding of the FP32
exponents 2^-22 * (|lse| + |s|), and 2^-18 for ex2 and FP32 sums of up to 2000
terms in 8 interleaved parts.  Everything else is exact.
"""
import math

import pytest
import torch

from flash_evict import _lib, check_status
from flash_evict.decode import KVCache, commit_tokens, evict_tokens, tree_attention
from oracle import decode as O
from test_gpu_decode import make, random_tree

pytestmark = pytest.mark.gpu


def with_book(cache, gen, norms=True, shuffle=True):
    """The cache with random bookkeeping; slots past the lengths hold junk."""
    b, h, c, _ = cache.k.shape
    live = (torch.arange(c) < cache.lengths.cpu()[..., None])
    mass = torch.where(live, torch.exp(2 * torch.randn(b, h, c, generator=gen)), torch.tensor(math.nan))
    pos = torch.stack([torch.randperm(c, generator=gen) if shuffle else torch.arange(c) for _ in range(b * h)]).view(b, h, c)
    size = torch.where(live, cache.v.cpu().double().abs().sum(-1).float(), torch.tensor(math.nan))
    return KVCache(cache.k, cache.v, cache.lengths, mass.cuda(), pos.to(torch.int32).cuda(), size.cuda() if norms else None)


def beside(cache, fill=-7):
    """A cache of the same k and v with bookkeeping of its own, prefilled with a mark."""
    return KVCache(cache.k, cache.v, torch.full_like(cache.lengths, fill), torch.full_like(cache.mass, fill),
                   torch.full_like(cache.positions, fill), None if cache.norms is None else torch.full_like(cache.norms, fill))


def clone(cache):
    c = lambda t: None if t is None else t.clone()  # noqa: E731
    k, v = torch.empty_strided(cache.k.shape, cache.k.stride(), dtype=cache.k.dtype, device="cuda"), torch.empty_strided(
        cache.v.shape, cache.v.stride(), dtype=cache.v.dtype, device="cuda")
    return KVCache(k.copy_(cache.k), v.copy_(cache.v), c(cache.lengths), c(cache.mass), c(cache.positions), c(cache.norms))


def bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


def path_of(tree, n):
    """A chain of n accepted drafts, each seen by the next ones: the ancestors of the draft that sees most."""
    best = int(tree.sum(1).argmax())
    return tree[best].nonzero()[:n, 0].tolist()


def check_commit(cache, q, kn, vn, lse, accepted, positions, tree=None, scale=None, decay=0.0):
    d = q.shape[-1]
    ref = O.commit(cache.k, cache.v, cache.lengths, cache.mass, cache.norms, cache.positions, q, kn, vn, lse, accepted, positions,
                   tree, scale, decay)
    s = abs(d ** -0.5 if scale is None else scale)
    live = (torch.arange(cache.k.shape[2]) < cache.lengths.cpu()[..., None])[..., None]
    size = lambda x: x.cpu().double().pow(2).sum(-1).sqrt().amax().item() if x.numel() else 0.0  # noqa: E731
    top = s * size(q) * max(size(torch.where(live, cache.k.cpu(), torch.zeros((), dtype=q.dtype))), size(kn))
    seen = lse[torch.isfinite(lse)]
    rel = 2.0 ** -22 * (2 * top + (seen.abs().max().item() if seen.numel() else 0.0)) + 2.0 ** -18
    inplace, other = clone(cache), beside(cache)
    before = clone(cache)
    got = commit_tokens(cache, q, kn, vn, lse, accepted, positions, tree=tree, scale=scale, recency_decay=decay, out=other)
    assert got is other
    for a, b in ((cache.lengths, before.lengths), (cache.mass, before.mass), (cache.positions, before.positions)):
        assert torch.equal(bits(a), bits(b))
    same = commit_tokens(inplace, q, kn, vn, lse, accepted, positions, tree=tree, scale=scale, recency_decay=decay)
    assert same is inplace
    for (i, h), (rk, rv, rm, rn, rp) in ref.items():
        n = len(rk)
        for c in (other, inplace):
            assert int(c.lengths[i, h]) == n
            assert torch.equal(bits(c.k[i, h, :n].cpu()), bits(rk)) and torch.equal(bits(c.v[i, h, :n].cpu()), bits(rv))
            assert torch.equal(c.positions[i, h, :n].cpu(), rp)
            m = c.mass[i, h, :n].cpu().double()
            assert ((m - rm).abs() <= rel * rm.abs() + 1e-37).all(), ((m - rm).abs() / rm.abs().clamp(min=1e-37)).max() / rel
            if rn is not None:
                torch.testing.assert_close(c.norms[i, h, :n].cpu().double(), rn, rtol=2.0 ** -20, atol=0)
        # nothing past the new length is touched
        assert (other.mass[i, h, n:] == -7).all() and (other.positions[i, h, n:] == -7).all()
        assert torch.equal(bits(other.k[i, h, n:]), bits(before.k[i, h, n:]))
        assert torch.equal(bits(inplace.mass[i, h, n:]), bits(before.mass[i, h, n:]))
        assert torch.equal(bits(inplace.mass[i, h, :n]), bits(other.mass[i, h, :n]))
    return other


SHAPES = [
    # b, hq, hk, d, capacity, t, lengths, accepted per sequence
    (1, 4, 2, 128, 300, 1, 0, [1]),
    (1, 28, 4, 128, 2304, 1, 2048, [1]),
    (2, 4, 4, 64, 530, 5, 513, [3, 0]),
    (3, 6, 2, 80, 700, 7, 640, [1, 4, 2]),
    (2, 8, 1, 256, 400, 9, 257, [2, 3]),
    (1, 3, 1, 200, 260, 9, 128, [4]),
    (2, 4, 2, 20, 200, 4, 77, [2, 1]),
    (1, 2, 2, 16, 40, 2, 33, [1]),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("decay,norms", [(0.0, True), (0.1, True), (0.05, False)])
def test_commit(shape, dtype, decay, norms):
    b, hq, hk, d, cap, t, n, took = shape
    q, kn, vn, cache, gen = make(sum(shape[:7]), b, hq, hk, d, cap, t, dtype, n)
    cache = with_book(cache, gen, norms)
    tree = random_tree(gen, b, t) if t > 1 else None
    accepted = torch.full((b, max(took)), -1, dtype=torch.int32)
    for i, m in enumerate(took):
        path = [0] if t == 1 else path_of(tree[i], m)
        accepted[i, :len(path[:m])] = torch.tensor(path[:m], dtype=torch.int32)
    positions = torch.randint(0, 10000, (b, t), generator=gen, dtype=torch.int32).cuda()
    tree = tree.cuda() if tree is not None else None
    _, lse = tree_attention(q, kn, vn, cache, tree=tree)
    check_commit(cache, q, kn, vn, lse, accepted.cuda(), positions, tree=tree, decay=decay)


@pytest.mark.parametrize("b,hq,hk,d,t", [(1, 28, 4, 128, 64), (1, 8, 8, 64, 128), (2, 5, 1, 256, 33), (1, 150, 1, 200, 3)])
def test_commit_every_draft_of_a_chain(b, hq, hk, d, t):
    # more query rows than one launch holds
    q, kn, vn, cache, gen = make(21, b, hq, hk, d, 700, t, torch.bfloat16, 500)
    cache = with_book(cache, gen)
    _, lse = tree_attention(q, kn, vn, cache)
    accepted = torch.arange(t, dtype=torch.int32).expand(b, t).contiguous().cuda()
    positions = torch.arange(500, 500 + t, dtype=torch.int32).expand(b, t).contiguous().cuda()
    check_commit(cache, q, kn, vn, lse, accepted, positions, decay=0.01)


def test_commit_ragged_rows_and_long_ones():
    lengths = [[0, 1, 700], [255, 0, 256], [0, 0, 0], [257, 1000, 31], [1000, 999, 5]]
    q, kn, vn, cache, gen = make(22, 5, 12, 3, 128, 1024, 9, torch.bfloat16, lengths)
    cache = with_book(cache, gen)
    tree = random_tree(gen, 5, 9)
    accepted = torch.full((5, 4), -1, dtype=torch.int32)
    for i, m in enumerate((4, 0, 2, 1, 3)):
        path = path_of(tree[i], m)
        accepted[i, :len(path)] = torch.tensor(path, dtype=torch.int32)
    accepted[4] = torch.tensor([-1, accepted[4, 0], -5, accepted[4, 1]])  # gaps are skipped
    positions = torch.arange(45, dtype=torch.int32).view(5, 9).cuda()
    _, lse = tree_attention(q, kn, vn, cache, tree=tree.cuda())
    check_commit(cache, q, kn, vn, lse, accepted.cuda(), positions, tree=tree.cuda(), decay=0.3)
    q, kn, vn, cache, gen = make(23, 1, 2, 1, 128, 40000, 2, torch.float16, 39990)
    cache = with_book(cache, gen)
    _, lse = tree_attention(q, kn, vn, cache)
    check_commit(cache, q, kn, vn, lse, torch.tensor([[0, 1]], dtype=torch.int32).cuda(), positions[:1, :2].contiguous())


def test_commit_a_row_that_saw_nothing_adds_nothing():
    q, kn, vn, cache, gen = make(24, 1, 4, 2, 64, 128, 3, torch.float16, [[0, 5]])
    cache = with_book(cache, gen)
    tree = torch.zeros(3, 3, dtype=torch.bool, device="cuda")
    _, lse = tree_attention(q, kn, vn, cache, tree=tree)
    positions = torch.arange(3, dtype=torch.int32).view(1, 3).cuda()
    got = check_commit(cache, q, kn, vn, lse, torch.tensor([[0, 2]], dtype=torch.int32).cuda(), positions, tree=tree)
    assert (got.mass[0, 0, :2] == 0).all()


def test_commit_past_the_capacity_and_bad_indices_are_reported():
    q, kn, vn, cache, gen = make(25, 1, 4, 2, 64, 130, 4, torch.float16, [[128, 130]], junk=0.0)
    cache = with_book(cache, gen)
    _, lse = tree_attention(q, kn, vn, cache)
    positions = torch.arange(4, dtype=torch.int32).view(1, 4).cuda()
    out = beside(cache)
    commit_tokens(cache, q, kn, vn, lse, torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda(), positions, out=out)
    assert out.lengths.tolist() == [[130, 130]]
    with pytest.raises(RuntimeError, match="cache full"):
        check_status()
    out = beside(cache)
    commit_tokens(cache, q, kn, vn, lse, torch.tensor([[0, 4]], dtype=torch.int32).cuda(), positions, out=out)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError):  # the next call reports it and launches nothing
        tree_attention(q, kn, vn, cache)
    assert _lib.device_status(torch.cuda.current_device(), clear=True) == _lib.STATUS_CACHE_FULL


# ------------------------------------------------------------------------------ eviction


def check_evict(cache, budget, recent):
    before = clone(cache)
    inplace, other = clone(cache), beside(cache)
    keep_k, keep_v = clone(cache).k, clone(cache).v
    assert evict_tokens(inplace, budget, recent=recent) is inplace
    got = evict_tokens(cache, budget, recent=recent, out=other)
    assert torch.equal(bits(cache.mass), bits(before.mass)) and torch.equal(cache.lengths, before.lengths)
    cap = cache.k.shape[2]
    for i in range(cache.k.shape[0]):
        for h in range(cache.k.shape[1]):
            n = min(max(int(before.lengths[i, h]), 0), cap)
            src = O.evict_slots(before.mass[i, h, :n].tolist(), before.positions[i, h, :n].tolist(), budget, recent)
            m = len(src)
            at = torch.tensor(src, dtype=torch.long, device="cuda")
            for c in (got, inplace):
                assert int(c.lengths[i, h]) == m
                assert torch.equal(bits(c.k[i, h, :m]), bits(keep_k[i, h][at])) and torch.equal(bits(c.v[i, h, :m]), bits(keep_v[i, h][at]))
                assert torch.equal(bits(c.k[i, h, m:]), bits(keep_k[i, h, m:])), "slots past the budget change"
                assert torch.equal(bits(c.mass[i, h, :m]), bits(before.mass[i, h][at]))
                assert torch.equal(c.positions[i, h, :m], before.positions[i, h][at])
                if c.norms is not None:
                    assert torch.equal(bits(c.norms[i, h, :m]), bits(before.norms[i, h][at]))
            assert (got.mass[i, h, m:] == -7).all() and (got.positions[i, h, m:] == -7).all()
    return got


def cache_for_eviction(seed, b, h, d, cap, lengths, dtype=torch.bfloat16, norms=True, layout="bhnd"):
    _, _, _, cache, gen = make(seed, b, h, h, d, cap, 1, dtype, lengths, layout=layout)
    return with_book(cache, gen, norms), gen


@pytest.mark.parametrize("n", [0, 1, 99, 100, 101, 102, 163, 199, 200, 201, 255, 256, 500])
@pytest.mark.parametrize("recent", [0, 1, 37, 100])
def test_evict_lengths(n, recent):
    cache, _ = cache_for_eviction(n + recent, 1, 2, 64, 500, n)
    check_evict(cache, 100, recent)


@pytest.mark.parametrize("d,dtype,layout", [(128, torch.float16, "bhnd"), (80, torch.bfloat16, "bnhd"), (20, torch.float16, "bhnd"),
                                            (256, torch.bfloat16, "bnhd"), (1, torch.float16, "bhnd")])
def test_evict_channels_and_layouts(d, dtype, layout):
    cache, _ = cache_for_eviction(31, 2, 3, d, 700, [[700, 0, 650], [300, 301, 10]], dtype, norms=d != 80, layout=layout)
    check_evict(cache, 300, 40)


@pytest.mark.parametrize("budget", [1, 64, 9000, 19999, 30000])
def test_evict_long_rows(budget):
    cache, _ = cache_for_eviction(32, 1, 2, 16, 20000, [[20000, 13001]])
    check_evict(cache, budget, min(budget, 64))


def test_evict_many_rows():
    gen = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 600, (40, 8), generator=gen).tolist()
    cache, _ = cache_for_eviction(33, 40, 8, 32, 600, lengths)
    check_evict(cache, 256, 20)


def test_evict_many_rows_with_much_to_move():
    # enough rows and bytes that the moves are a launch of their own
    gen = torch.Generator().manual_seed(7)
    lengths = torch.randint(0, 2301, (5, 8), generator=gen)
    lengths[0, 0], lengths[4, 7], lengths[2, 3] = 0, 2300, 1101
    cache, _ = cache_for_eviction(37, 5, 8, 128, 2300, lengths.tolist(), dtype=torch.float16)
    check_evict(clone(cache), 1100, 64)
    cache, _ = cache_for_eviction(38, 5, 8, 100, 2900, 2900, norms=False)
    check_evict(cache, 1449, 0)


@pytest.mark.parametrize("rows, cap, budget, recent", [
    (3, 2300, 1100, 64),     # one CTA a row, moves in a launch of their own
    (3, 8300, 4000, 0),      # small clusters, and the same
    (2, 33000, 9000, 100),   # large ones
    (20, 17000, 260, 0),     # clusters of four, which move the rows themselves
    (70, 8300, 300, 20),     # of two
    (80, 8300, 200, 0),      # too many rows for clusters
])
def test_evict_launch_shapes(rows, cap, budget, recent):
    gen = torch.Generator().manual_seed(rows + cap)
    lengths = torch.randint(budget - 50, cap + 1, (1, rows), generator=gen)
    lengths[0, 0], lengths[0, -1] = cap, budget + 1
    cache, _ = cache_for_eviction(39, 1, rows, 96, cap, lengths.tolist())
    check_evict(cache, budget, recent)


def test_evict_ties_zeros_infinities_and_nan():
    cache, gen = cache_for_eviction(34, 1, 4, 32, 3000, 3000)
    m = cache.mass
    m[0, 0] = 1.0                                             # one tie over the whole row
    m[0, 1] = torch.where(torch.rand(3000, device="cuda") < 0.5, 0.0, -0.0)
    m[0, 2] = torch.randint(0, 4, (3000,), device="cuda").float() - 1.5
    m[0, 3, ::7], m[0, 3, 1::7], m[0, 3, 2::7] = float("nan"), float("inf"), float("-inf")
    for budget, recent in ((1, 0), (428, 0), (429, 100), (1200, 7), (2999, 2999)):
        check_evict(clone(cache), budget, recent)


def test_evict_rows_longer_than_shared_memory():
    # 500k slots a row: the keys are read again on every pass instead of kept
    cap = 500_000
    cache, _ = cache_for_eviction(35, 1, 1, 8, cap, cap)
    check_evict(cache, 3000, 64)


def test_positions_at_the_ends_of_their_range():
    cache, _ = cache_for_eviction(36, 1, 1, 16, 300, 300)
    cache.positions[0, 0, :] = torch.arange(300, device="cuda", dtype=torch.int32) - 2 ** 31
    check_evict(clone(cache), 200, 50)
    check_evict(clone(cache), 299, 299)


def test_offsets_past_32_bits():
    """A [B, C, H, D] cache of 2.5 G elements a tensor: head 0's last slots and head 8's first lie past 2^31 elements."""
    cap, h, d, t = 1_100_000, 9, 256, 2
    gen = torch.Generator().manual_seed(8)
    g = torch.Generator(device="cuda").manual_seed(8)
    k, v = (torch.empty(1, cap, h, d, dtype=torch.bfloat16, device="cuda").normal_(generator=g).transpose(1, 2) for _ in range(2))
    n = cap - 100
    lengths = torch.tensor([[n, 0, 1, 2, 3, 130, 0, 0, n - 5]], dtype=torch.int32, device="cuda")
    mass = torch.rand(1, h, cap, generator=g, device="cuda")
    pos = torch.arange(cap, dtype=torch.int32, device="cuda").expand(1, h, cap).contiguous()
    cache = KVCache(k, v, lengths, mass, pos)
    q, kn, vn = (torch.randn(1, t, h, d, generator=gen).to(torch.bfloat16).cuda().transpose(1, 2) for _ in range(3))
    out, lse = tree_attention(q, kn, vn, cache)
    want = mass.clone()
    for head in (0, 5, 8):
        m = int(lengths[0, head])
        keys, values = torch.cat([k[0, head, :m], kn[0, head]]).double(), torch.cat([v[0, head, :m], vn[0, head]]).double()
        x = q[0, head].double() @ keys.T * d ** -0.5
        x[0, -1] = -math.inf  # a chain: the first draft does not see the second
        ref_lse = torch.logsumexp(x, -1)
        p = torch.exp(x - ref_lse[:, None])
        spread = p @ values.abs()
        assert ((lse[0, head] - ref_lse).abs() <= 1e-5 * ref_lse.abs()).all()
        assert ((out[0, head].double() - p @ values).abs() <= 2.0 ** -8 * 1.01 * (spread + (p @ values).abs()) + 1e-5 * spread).all()
        want[0, head, :m] += p[:, :m].sum(0).float()
        want[0, head, m:m + t] = p[:, m:].sum(0).float()
    steps = torch.arange(t, dtype=torch.int32, device="cuda")[None]
    commit_tokens(cache, q, kn, vn, lse, steps, cap + steps)
    for head in (0, 5, 8):
        m = int(lengths[0, head])  # the new length
        torch.testing.assert_close(cache.mass[0, head, :m], want[0, head, :m], rtol=1e-5, atol=1e-9)
        assert torch.equal(k[0, head, m - t:m], kn[0, head]) and torch.equal(v[0, head, m - t:m], vn[0, head])
    budget = n - 50
    old = {head: (cache.mass[0, head].clone(), k[0, head, budget:].clone(), v[0, head, budget:].clone()) for head in (0, 8)}
    untouched = k[0, 0, :1000].clone(), v[0, 8, 500_000:501_000].clone()
    evict_tokens(cache, budget, recent=20)
    for head, (m, k_old, v_old) in old.items():
        before = n if head == 0 else n - 5
        places = list(range(before)) + [cap, cap + 1]
        src = torch.tensor(O.evict_slots(m[:before + t].tolist(), places, budget, 20), device="cuda")
        moved = (src >= budget).nonzero()[:, 0]
        assert len(moved) > 0 and int(cache.lengths[0, head]) == budget
        assert torch.equal(cache.mass[0, head, :budget], m[src])
        assert torch.equal(k[0, head, moved], k_old[src[moved] - budget]) and torch.equal(v[0, head, moved], v_old[src[moved] - budget])
    assert (k[0, 0, :1000] != untouched[0]).any(-1).sum() < 10 and (v[0, 8, 500_000:501_000] != untouched[1]).any(-1).sum() < 10


# ------------------------------------------------------------------------------ together


def test_steps_in_a_graph_equal_steps_outside():
    """Attention, commit and eviction captured once and replayed, against the same calls one by one."""
    q, kn, vn, cache, gen = make(41, 2, 8, 2, 128, 400, 6, torch.bfloat16, [[250, 256], [0, 31]], junk=0.0)
    cache = with_book(cache, gen)
    plain = clone(cache)
    tree = random_tree(gen, 2, 6)
    accepted = torch.tensor([path_of(tree[0], 2), path_of(tree[1], 2)], dtype=torch.int32).cuda()
    tree = tree.cuda()
    positions = torch.arange(500, 506, dtype=torch.int32).expand(2, 6).contiguous().cuda()

    def step(c):
        out, lse = tree_attention(q, kn, vn, c, tree=tree)
        commit_tokens(c, q, kn, vn, lse, accepted, positions, tree=tree, recency_decay=0.1)
        evict_tokens(c, 256, recent=16)
        return out

    warm = clone(cache)
    step(warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for _ in range(3):
        positions += 2
        graph.replay()
        ref = step(plain)
        assert torch.equal(bits(out), bits(ref))
        assert torch.equal(cache.lengths, plain.lengths)
        for i in range(2):
            for h in range(2):
                n = int(cache.lengths[i, h])
                for a, b in ((cache.k, plain.k), (cache.v, plain.v), (cache.mass, plain.mass), (cache.norms, plain.norms)):
                    assert torch.equal(bits(a[i, h, :n]), bits(b[i, h, :n]))
                assert torch.equal(cache.positions[i, h, :n], plain.positions[i, h, :n])


def test_decode_weights_continue_the_prefill_importance():
    """A prompt prefilled whole gives the weights that a shorter prefill and committed steps give."""
    from flash_evict import prefill
    gen = torch.Generator().manual_seed(6)
    n, new, hq, hk, d, decay = 700, 5, 8, 2, 64, 0.02
    q, k, v = (torch.randn(1, h, n + new, d, generator=gen).to(torch.float16).cuda() for h in (hq, hk, hk))
    _, whole = prefill(q, k, v, recency_decay=decay)
    _, part = prefill(q[:, :, :n].contiguous(), k[:, :, :n].contiguous(), v[:, :, :n].contiguous(), recency_decay=decay)
    cache = KVCache.allocate(1, hk, n + new, d, torch.float16).fill(k[:, :, :n], v[:, :, :n], mass=part)
    for t0, t1 in ((0, 1), (1, 5)):
        at = slice(n + t0, n + t1)
        qq, kk, vv = q[:, :, at], k[:, :, at], v[:, :, at]
        _, lse = tree_attention(qq, kk, vv, cache)
        steps = torch.arange(t1 - t0, dtype=torch.int32, device="cuda")[None]
        commit_tokens(cache, qq, kk, vv, lse, steps, (n + t0 + steps), recency_decay=decay)
    assert cache.lengths.tolist() == [[n + new] * hk]
    # 705 query rows, FP32 sums on both sides and a rounding per step
    torch.testing.assert_close(cache.mass, whole, rtol=5e-5, atol=1e-6)
    torch.testing.assert_close(cache.norms, v.float().abs().sum(-1), rtol=1e-6, atol=0)
    assert torch.equal(cache.positions[0, 0], torch.arange(n + new, dtype=torch.int32, device="cuda"))
