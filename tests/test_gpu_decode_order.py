"""Decode operators back to back, as a captured step runs them, against the same calls one at a time.

Every kernel may start while the ones before it end, so whatever a call reads of
the cache has to be what the call before it wrote.  The results are compared bit
by bit: the operators are reproducible, and only the timing differs.
"""
import pytest
import torch

from flash_evict.decode import commit_tokens, evict_tokens, tree_attention
from test_gpu_decode import make, random_tree
from test_gpu_decode_cache import bits, clone, path_of, with_book

pytestmark = pytest.mark.gpu


def same(a, b):
    """The live tokens and lengths of two caches."""
    assert torch.equal(a.lengths, b.lengths)
    live = torch.arange(a.k.shape[2], device="cuda") < a.lengths[..., None]
    for x, y in ((a.k, b.k), (a.v, b.v), (a.mass, b.mass), (a.norms, b.norms), (a.positions, b.positions)):
        assert torch.equal(bits(x)[live], bits(y)[live])


# Attentions whose runs leave SMs free (so that the join of the runs can be
# resident early), with lengths that change the number of key tiles at every step.
SHAPES = [
    # b, hq, hk, d, budget, spare, t, accepted
    (1, 32, 8, 128, 1024, 128, 64, 5),
    (1, 28, 4, 128, 1024, 128, 64, 5),
    (1, 8, 1, 128, 8192, 128, 1, 1),
    (1, 4, 4, 128, 4352, 128, 1, 1),
    (4, 8, 8, 64, 256, 128, 1, 1),
    (2, 8, 4, 256, 1024, 100, 3, 2),  # (a cluster a row)
]


@pytest.mark.parametrize("shape", SHAPES)
def test_attention_right_after_a_change_of_the_lengths(shape):
    b, hq, hk, d, budget, spare, t, took = shape
    q, kn, vn, cache, gen = make(sum(shape), b, hq, hk, d, budget + spare, t, torch.bfloat16, budget + took, junk=0.0)
    cache = with_book(cache, gen)
    tree = random_tree(gen, 1, t)[0]
    path = path_of(tree, took)
    path = path + [j for j in range(t) if j not in path][:took - len(path)]
    accepted = torch.tensor([path], dtype=torch.int32).expand(b, took).contiguous().cuda()
    positions = torch.full((b, t), 10 ** 6, dtype=torch.int32, device="cuda")
    tree = tree.cuda() if t > 1 else None
    plain = clone(cache)

    def steps(c, between):
        got = []
        for _ in range(4):
            evict_tokens(c, budget, recent=8)
            between()
            got.append(tree_attention(q, kn, vn, c, tree=tree))
            between()
            commit_tokens(c, q, kn, vn, got[-1][1], accepted, positions, tree=tree)
            between()
            got.append(tree_attention(q, kn, vn, c, tree=tree))
            between()
        return got

    want = steps(plain, torch.cuda.synchronize)
    steps(clone(cache), torch.cuda.synchronize)
    graph = torch.cuda.CUDAGraph()
    start = clone(cache)
    with torch.cuda.graph(graph):
        got = steps(cache, lambda: None)
    for _ in range(5):
        for name in ("k", "v", "mass", "norms", "positions", "lengths"):
            getattr(cache, name).copy_(getattr(start, name))
        graph.replay()
        for (out, lse), (ref, ref_lse) in zip(got, want):
            assert torch.equal(bits(lse), bits(ref_lse)) and torch.equal(bits(out), bits(ref))
        same(cache, plain)


@pytest.mark.parametrize("b,hq,hk,d,n,dtype", [(1, 28, 4, 128, 2048, torch.float16), (1, 28, 4, 128, 20000, torch.bfloat16),
                                               (16, 14, 2, 64, 3000, torch.bfloat16), (1, 6, 2, 256, 3000, torch.float16)])
def test_what_ran_before_leaves_no_trace(b, hq, hk, d, n, dtype):
    # Queries fill a part of their tile; the rest holds what an earlier kernel left
    # in shared memory, here the queries of a call with full tiles.
    q, kn, vn, cache, _ = make(51, b, hq, hk, d, n + 64, 1, dtype, n, sharp=2.0)
    full, fk, fv, _, _ = make(52, b, 8 * hk, hk, d, 64, 16, dtype, 0)
    seen = []
    for loud in (0.0, 30.0, 1000.0, 0.0):
        tree_attention(full * loud, fk, fv, cache)
        seen.append(tree_attention(q, kn, vn, cache))
    for out, lse in seen[1:]:
        assert torch.equal(bits(out), bits(seen[0][0])) and torch.equal(bits(lse), bits(seen[0][1]))


@pytest.mark.parametrize("t,group,d", [(100, 2, 64), (37, 7, 128), (128, 3, 128)])
def test_drafts_without_a_mask_over_many_rows_two_query_tiles_each(t, group, d):
    # Empty rows are single tiles, through which the two warpgroups of a run pass
    # at their own pace; which drafts' values are not finite is noted per row.
    b, hk, cap = 48, 8, 400
    gen = torch.Generator().manual_seed(t)
    lengths = (torch.randint(0, 4, (b, hk), generator=gen) == 0) * torch.randint(0, cap, (b, hk), generator=gen)
    q, kn, vn, cache, _ = make(53, b, group * hk, hk, d, cap, t, torch.bfloat16, lengths.tolist())
    bad = torch.rand(b, hk, t, d, generator=gen) < 2e-4
    vn = torch.where(bad.cuda(), torch.inf, vn.float()).to(vn.dtype)
    # a chain: a draft sees the ones before it and itself
    want = bad.cumsum(2).bool().repeat_interleave(group, 1).cuda()
    for _ in range(5):
        out, lse = tree_attention(q, kn, vn, cache)
        assert torch.equal(torch.isposinf(out), want) and torch.equal(torch.isfinite(out), ~want) and torch.isfinite(lse).all()


def test_a_captured_first_commit_leaves_the_cache_ready_for_others():
    """The first commit of a cache captured and not yet replayed: eager commits and other graphs count their CTAs all the same."""
    q, kn, vn, cache, gen = make(54, 1, 4, 2, 64, 300, 2, torch.bfloat16, [[250, 0]], junk=0.0)
    cache = with_book(cache, gen)
    _, lse = tree_attention(q, kn, vn, cache)
    accepted = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    positions = torch.tensor([[1000, 1001]], dtype=torch.int32, device="cuda")
    pool = torch.cuda.graph_pool_handle()
    before = torch.cuda.CUDAGraph()
    with torch.cuda.graph(before, pool=pool):
        junk = [torch.full((128,), 7, dtype=torch.int32, device="cuda") for _ in range(8)]
    before.replay()  # memory of the pool that holds no zeros
    del junk
    plain = clone(cache)

    def commit(c):
        commit_tokens(c, q, kn, vn, lse, accepted, positions)

    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph in graphs:
        with torch.cuda.graph(graph, pool=pool):
            commit(cache)
    n = 0
    for step in (lambda: commit(cache), graphs[1].replay, lambda: commit(cache), graphs[0].replay, graphs[1].replay):
        step()
        commit(plain)
        n += 2
        assert cache.lengths.tolist() == [[250 + n, n]]
        same(cache, plain)
