"""Decode operators over a budgeted cache against the 64-bit oracle.

Tolerances, from the arithmetic (u = unit roundoff of the 16-bit type, 2^-8 for
bf16 and 2^-11 for fp16):
  out: P is rounded to 16 bits before the value product and out at the end, so
    |error| <= u * (sum p|v| + |out|), plus for fp16 the absolute spacing 2^-25 of
    P below 2^-14, once per token;
  logits: FP32 sums of exact 16-bit products, |error| <= 2^-22 * scale * sum|q||k|
    (FP32 accumulation over <= 256 channels in blocks), which moves p relatively;
  lse: the logit error and 2^-20 for ex2/lg2 and the FP32 sum.
"""
import pytest
import torch

from flash_evict.decode import KVCache, tree_attention
from oracle import decode as O

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def random_tree(gen, batch, t, padded=0):
    """Ancestor masks of random trees; the last `padded` drafts see nothing and are seen by nobody."""
    m = torch.zeros(batch, t, t, dtype=torch.bool)
    for b in range(batch):
        for j in range(t - padded):
            if j:
                m[b, j] = m[b, int(torch.randint(0, j, (1,), generator=gen))]
            m[b, j, j] = True
    return m


def make(seed, b, hq, hk, d, cap, t, dtype, lengths, sharp=1.0, junk=float("nan"), layout="bhnd"):
    gen = torch.Generator().manual_seed(seed)
    lengths = torch.tensor(lengths, dtype=torch.int32).expand(b, hk).contiguous()
    q = (torch.randn(b, t, hq, d, generator=gen) * sharp).to(dtype).transpose(1, 2)
    kn, vn = (torch.randn(b, t, hk, d, generator=gen).to(dtype).transpose(1, 2) for _ in range(2))
    k, v = (torch.randn(b, hk, cap, d, generator=gen).to(dtype) for _ in range(2))
    dead = torch.arange(cap) >= lengths[..., None]
    k[dead], v[dead] = junk, junk
    pitch = (d + 7) // 8 * 8

    def place(x):
        shape = (b, hk, cap, pitch) if layout == "bhnd" else (b, cap, hk, pitch)
        y = torch.full(shape, junk, dtype=dtype, device="cuda")[..., :d]
        y = y if layout == "bhnd" else y.transpose(1, 2)
        y.copy_(x)
        return y

    cache = KVCache(place(k), place(v), lengths.cuda())
    return q.cuda(), kn.cuda(), vn.cuda(), cache, gen


def check_attention(q, kn, vn, cache, tree=None, scale=None):
    out, lse = tree_attention(q, kn, vn, cache, tree=tree, scale=scale)
    ref, ref_lse, spread = O.tree_attention(q, kn, vn, cache.k, cache.v, cache.lengths, tree, scale)
    d, dtype = q.shape[-1], q.dtype
    scale = d ** -0.5 if scale is None else scale
    n = int(cache.lengths.max()) + q.shape[2]
    fin = lambda x: torch.nan_to_num(x.float().cpu(), 0, 0, 0).abs()  # noqa: E731
    live = (torch.arange(cache.k.shape[2]) < cache.lengths.cpu()[..., None])[..., None]
    size = lambda x: fin(x).pow(2).sum(-1).sqrt().amax().item() if x.numel() else 0.0  # noqa: E731
    kmax = max(size(torch.where(live, cache.k.cpu(), torch.zeros((), dtype=dtype))), size(kn))
    eps = 2.0 ** -22 * abs(scale) * size(q) * kmax
    vmax = max(fin(torch.where(live, cache.v.cpu(), torch.zeros((), dtype=dtype))).max().item(), fin(vn).max().item())
    got, got_lse = out.double().cpu(), lse.double().cpu()
    seen = torch.isfinite(ref_lse)
    assert torch.equal(torch.isneginf(got_lse), torch.isneginf(ref_lse))
    assert ((got_lse - ref_lse).abs()[seen] <= eps + 2.0 ** -20 * (1 + ref_lse.abs()[seen])).all()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isposinf(got), torch.isposinf(ref))
    ok = torch.isfinite(ref)
    tol = U[dtype] * 1.01 * (spread + ref.abs()) + 2 * (eps + 2.0 ** -20) * spread
    tol = tol + (n * 2.0 ** -25 * vmax if dtype == torch.float16 else 1e-30)
    assert ((got - ref).abs()[ok] <= tol[ok]).all(), ((got - ref).abs()[ok] / tol[ok]).max()
    return out, lse


SHAPES = [
    # b, hq, hk, d, capacity, t, lengths
    (1, 4, 2, 128, 300, 1, 0),
    (1, 4, 2, 128, 300, 1, 1),
    (1, 4, 2, 128, 300, 1, 127),
    (1, 4, 2, 128, 300, 1, 128),
    (1, 4, 2, 128, 300, 1, 129),
    (1, 28, 4, 128, 2304, 1, 2048),
    (2, 4, 4, 64, 513, 5, 513),
    (1, 6, 2, 80, 700, 7, 611),
    (3, 8, 1, 256, 400, 3, 333),
    (1, 3, 1, 200, 260, 9, 201),
    (2, 4, 2, 20, 200, 4, 77),
    (1, 2, 2, 16, 40, 2, 33),
    (1, 5, 1, 1, 40, 3, 33),
    (1, 28, 4, 128, 1100, 64, 1000),   # 448 rows: two query tiles of 256
    (1, 8, 8, 128, 700, 128, 600),     # 128 rows, all drafts of a call
    (1, 7, 1, 64, 700, 37, 650),       # 259 rows: the last query tile holds 3
    (1, 40, 1, 256, 300, 11, 290),     # 440 rows, one query tile at a time
    (1, 256, 1, 64, 300, 1, 200),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_tree_attention(shape, dtype):
    b, hq, hk, d, cap, t, n = shape
    q, kn, vn, cache, gen = make(sum(shape), b, hq, hk, d, cap, t, dtype, n)
    check_attention(q, kn, vn, cache)
    if t > 1:
        check_attention(q, kn, vn, cache, tree=random_tree(gen, b, t, padded=t // 3).cuda())


def test_tree_attention_ragged_rows():
    # every row its own length, some empty, some one token short of or past a tile
    lengths = [[0, 1, 700], [255, 0, 256], [0, 0, 0], [257, 1024, 31], [1024, 1023, 5]]
    q, kn, vn, cache, gen = make(7, 5, 12, 3, 128, 1024, 9, torch.bfloat16, lengths)
    tree = random_tree(gen, 5, 9, padded=2)
    check_attention(q, kn, vn, cache, tree=tree.cuda())
    # one mask for all sequences
    check_attention(q, kn, vn, cache, tree=tree[1].cuda())


@pytest.mark.parametrize("d", [64, 20, 81, 200])
def test_tree_attention_many_short_rows(d):
    # far more rows than SMs: each run covers several rows and writes most of them itself
    gen = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 400, (40, 8), generator=gen).tolist()
    q, kn, vn, cache, _ = make(8, 40, 16, 8, d, 400, 2, torch.float16, lengths)
    check_attention(q, kn, vn, cache)


@pytest.mark.parametrize("b,hq,hk,d,t", [(3, 16, 8, 128, 6), (3, 16, 8, 72, 5), (2, 30, 10, 256, 4), (1, 5, 1, 200, 3), (2, 24, 2, 64, 20)])
def test_masked_drafts_in_every_kernel_shape(b, hq, hk, d, t):
    # one row a run and several, one warpgroup and two, one query tile and two
    for lengths in (0, 3, 260):
        q, kn, vn, cache, gen = make(17 + lengths, b, hq, hk, d, 300, t, torch.bfloat16, lengths)
        tree = random_tree(gen, 1, t)[0]
        tree[:, t - 1] = False
        kn[:, :, t - 1], vn[:, :, t - 1] = float("nan"), float("-inf")
        vn[:, :, 1, 3] = float("inf")
        check_attention(q, kn, vn, cache, tree=tree.cuda())


def test_tree_attention_long_row_is_shared():
    q, kn, vn, cache, gen = make(9, 1, 4, 1, 128, 40000, 4, torch.bfloat16, 39990)
    check_attention(q, kn, vn, cache, tree=random_tree(gen, 1, 4).cuda())


def test_tree_attention_rows_that_see_nothing():
    q, kn, vn, cache, _ = make(10, 2, 4, 2, 64, 128, 6, torch.float16, [[0, 3], [0, 0]])
    tree = torch.eye(6, dtype=torch.bool, device="cuda")
    tree[2, 2] = tree[5, 5] = False
    out, lse = check_attention(q, kn, vn, cache, tree=tree)
    assert torch.isneginf(lse[1, :, 2]).all() and (out[1, :, 2] == 0).all()
    out, lse = check_attention(q, kn, vn, cache, tree=torch.zeros_like(tree))
    assert torch.isneginf(lse[1]).all() and (out[1] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("t", [6, 70])
def test_masked_drafts_may_hold_anything(bad, t):
    q, kn, vn, cache, gen = make(11, 1, 8, 2, 128, 300, t, torch.bfloat16, 200)
    tree = random_tree(gen, 1, t)[0]
    tree[:, 3] = False
    kn[:, :, 3], vn[:, :, 3] = bad, bad
    check_attention(q, kn, vn, cache, tree=tree.cuda())
    # a draft with a non-finite value row reaches exactly the rows that see it
    vn[:, :, 1, 5] = bad
    out, _ = check_attention(q, kn, vn, cache, tree=tree.cuda())
    assert torch.equal(~torch.isfinite(out[0, 0, :, 5]).cpu(), tree[:, 1])


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_scales_and_sharp_logits(scale):
    q, kn, vn, cache, gen = make(12, 1, 4, 2, 64, 900, 5, torch.float16, 850)
    check_attention(q, kn, vn, cache, scale=scale)
    q, kn, vn, cache, gen = make(13, 1, 4, 2, 128, 900, 3, torch.bfloat16, 850, sharp=30.0)
    check_attention(q, kn, vn, cache)


def test_layouts_and_streams():
    q, kn, vn, cache, gen = make(14, 2, 6, 2, 80, 500, 5, torch.bfloat16, [[499, 130], [0, 256]], layout="bnhd")
    ref = check_attention(q, kn, vn, cache)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tree_attention(q, kn, vn, cache)
    side.synchronize()
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    # q whose rows are neither aligned nor contiguous
    wide = torch.zeros(2, 6, 5, 83, dtype=q.dtype, device="cuda")
    wide[..., 3:] = q
    got = tree_attention(wide[..., 3:], kn, vn, cache)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_expanded_inputs():
    # one K/V head, one query and one mask for all: dimensions of stride 0
    q, kn, vn, cache, gen = make(16, 2, 8, 4, 64, 300, 5, torch.float16, 200)
    tree = random_tree(gen, 1, 5).cuda()
    q, kn, vn = q[:, :1].expand_as(q), kn[:, :1].expand_as(kn), vn[:1].expand_as(vn)
    got = check_attention(q, kn, vn, cache, tree=tree.expand(2, 5, 5))
    ref = tree_attention(q.contiguous(), kn.contiguous(), vn.contiguous(), cache, tree=tree[0])
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_attention_in_a_graph_follows_the_lengths():
    q, kn, vn, cache, gen = make(15, 1, 8, 2, 128, 800, 1, torch.bfloat16, 300, junk=0.5)
    tree_attention(q, kn, vn, cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = tree_attention(q, kn, vn, cache)
    for n in (0, 17, 799):
        cache.lengths.fill_(n)
        graph.replay()
        want = check_attention(q, kn, vn, cache)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
