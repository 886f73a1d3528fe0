"""Host-side contract of flash_evict.decode (no GPU): arguments, refusals, and the oracle's own arithmetic."""
import ctypes
import math

import pytest
import torch

from flash_evict import _lib
from flash_evict.decode import KVCache, _check_drafts, evict_tokens
from flash_evict.streaming_adapter import StreamingController
from oracle import decode as O
from test_streaming_cpu import tiny_model


def c_cache(**kw):
    fields = dict(k=256, v=256, k_strides=(512, 256, 8, 1), v_strides=(512, 256, 8, 1), mass=256, norms=256, positions=256,
                  lengths=256, sync=256, batch=1, kv_heads=2, capacity=32, channels=8, dtype=_lib.DTYPE_F16)
    fields.update(kw)
    c = _lib.Cache()
    for name, value in fields.items():
        setattr(c, name, (ctypes.c_int64 * 4)(*value) if name.endswith("strides") else value)
    return c


def test_c_abi_refusals_without_a_gpu():
    lib = _lib.load()
    st = (ctypes.c_int64 * 4)(64, 32, 8, 1)
    fake = 256  # never dereferenced: the argument checks fail first

    def attend(cache, q_heads=4, drafts=2, scale=0.1, q=fake, lse=fake, stride=0):
        return lib.fe_tree_attention(ctypes.byref(cache), q, st, fake, st, fake, st, None, stride, fake, lse, fake, 1 << 30,
                                     q_heads, drafts, scale, None)

    assert lib.fe_tree_attention(None, fake, st, fake, st, fake, st, None, 0, fake, fake, fake, 0, 4, 2, 0.1, None) == _lib.STATUS_INVALID
    for kw, text in (({"batch": 0}, b"empty cache"), ({"channels": 257}, b"channels"), ({"dtype": 7}, b"dtype"), ({"k": None}, b"null")):
        assert attend(c_cache(**kw)) == _lib.STATUS_INVALID and text in lib.fe_last_error(), kw
    assert attend(c_cache(capacity=1 << 31)) == _lib.STATUS_UNSUPPORTED
    assert attend(c_cache(), q_heads=3) == _lib.STATUS_INVALID and b"divisible" in lib.fe_last_error()
    assert attend(c_cache(), drafts=0) == _lib.STATUS_INVALID
    assert attend(c_cache(), drafts=129) == _lib.STATUS_UNSUPPORTED and b"128" in lib.fe_last_error()
    assert attend(c_cache(), q_heads=1024) == _lib.STATUS_UNSUPPORTED
    assert attend(c_cache(), scale=math.inf) == _lib.STATUS_INVALID and b"scale" in lib.fe_last_error()
    assert attend(c_cache(), lse=None) == _lib.STATUS_INVALID and b"null" in lib.fe_last_error()
    assert attend(c_cache(), stride=-1) == _lib.STATUS_INVALID
    assert lib.fe_tree_workspace_bytes(ctypes.byref(c_cache()), 4, 129) == -1

    def commit(cache, out, accepted=1, decay=0.0, size=1 << 20):
        # (in place: needs a workspace for the new lengths)
        return lib.fe_commit_tokens(ctypes.byref(cache), ctypes.byref(out), fake, st, fake, st, fake, st, None, 0, fake, fake, accepted,
                                    fake, fake, size, 4, 2, 0.1, decay, None)

    other = dict(mass=512, norms=512, positions=512, lengths=512)
    assert commit(c_cache(), c_cache(k=512)) == _lib.STATUS_INVALID and b"same cache" in lib.fe_last_error()
    assert commit(c_cache(), c_cache(**{**other, "mass": 256})) == _lib.STATUS_INVALID and b"share all" in lib.fe_last_error()
    assert commit(c_cache(norms=None), c_cache(**other)) == _lib.STATUS_INVALID and b"norms" in lib.fe_last_error()
    assert commit(c_cache(mass=None), c_cache()) == _lib.STATUS_INVALID and b"mass" in lib.fe_last_error()
    assert commit(c_cache(sync=None), c_cache()) == _lib.STATUS_INVALID and b"sync" in lib.fe_last_error()
    assert commit(c_cache(), c_cache(), accepted=0) == _lib.STATUS_INVALID
    assert commit(c_cache(), c_cache(), accepted=129) == _lib.STATUS_INVALID
    assert commit(c_cache(), c_cache(), decay=-1.0) == _lib.STATUS_INVALID and b"recency_decay" in lib.fe_last_error()
    assert commit(c_cache(), c_cache(), size=4) == _lib.STATUS_INVALID and b"workspace" in lib.fe_last_error()

    def evict(cache, out, budget=4, recent=0, size=1 << 20):
        return lib.fe_evict_tokens(ctypes.byref(cache), ctypes.byref(out), budget, recent, fake, size, None)

    assert evict(c_cache(), c_cache(), budget=0) == _lib.STATUS_INVALID
    assert evict(c_cache(), c_cache(), recent=5) == _lib.STATUS_INVALID and b"recent" in lib.fe_last_error()
    assert evict(c_cache(), c_cache(), size=3) == _lib.STATUS_INVALID
    bad = (512, 256, 9, 1)
    assert evict(c_cache(k_strides=bad), c_cache(k_strides=bad)) == _lib.STATUS_UNSUPPORTED
    assert lib.fe_evict_workspace_bytes(ctypes.byref(c_cache()), 0) == -1
    assert lib.fe_evict_workspace_bytes(ctypes.byref(c_cache()), 10) == 2 * (10 * 8 + 4)
    assert lib.fe_evict_workspace_bytes(ctypes.byref(c_cache()), 100) == 2 * 12


def test_cache_refuses_tensors_it_cannot_hold():
    k = torch.zeros(1, 2, 16, 8, dtype=torch.float16)
    n = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="one shape"):
        KVCache(k, k[:, :, :8], n)
    with pytest.raises(ValueError, match="CUDA"):
        KVCache(k, k, n)
    with pytest.raises(ValueError, match="CUDA"):
        KVCache(k.float(), k.float(), n)
    with pytest.raises(ValueError, match="channels"):
        KVCache(torch.zeros(1, 2, 16, 264), torch.zeros(1, 2, 16, 264), n)
    with pytest.raises(ValueError, match="positive"):
        KVCache.allocate(1, 0, 4, 8)


class Stub:
    """What the draft checks read of a cache, on the CPU."""

    def __init__(self):
        self.k = torch.zeros(2, 2, 16, 8, dtype=torch.float16)
        self.dtype, self.device = self.k.dtype, self.k.device
        self.mass = None


def test_draft_checks():
    c = Stub()
    q, kv = torch.zeros(2, 4, 3, 8, dtype=torch.float16), torch.zeros(2, 2, 3, 8, dtype=torch.float16)
    tree, stride, scale = _check_drafts(q, kv, kv, c, None, None)
    assert tree is None and stride == 0 and scale == 8 ** -0.5
    assert _check_drafts(q, kv, kv, c, torch.ones(3, 3, dtype=torch.bool), 0.5)[1:] == (0, 0.5)
    assert _check_drafts(q, kv, kv, c, torch.ones(2, 3, 3, dtype=torch.bool), 0.5)[1] == 9
    for bad, match in (((q[0], kv, kv, c, None, None), "q must have shape"), ((q[:, :3], kv, kv, c, None, None), "multiple"),
                       ((q[:, :, :0], kv, kv, c, None, None), "drafted tokens"),
                       ((torch.zeros(2, 4, 129, 8), kv, kv, c, None, None), "drafted tokens"),
                       ((q, kv[:, :1], kv, c, None, None), "k_new and v_new"), ((q, kv, kv.float(), c, None, None), "dtype"),
                       ((q, kv, kv, c, torch.ones(3, 3), None), "tree"), ((q, kv, kv, c, torch.ones(2, 2, dtype=torch.bool), None), "tree"),
                       ((q, kv, kv, c, None, math.nan), "scale")):
        with pytest.raises(ValueError, match=match):
            _check_drafts(*bad)
    with pytest.raises(ValueError, match="Inference only"):
        _check_drafts(q.clone().requires_grad_(), kv, kv, c, None, None)
    with pytest.raises(ValueError, match="no mass"):
        evict_tokens(c, 4)


def test_evict_argument_checks():
    c = Stub()
    c.mass = torch.zeros(2, 2, 16)
    for bad in (0, -1, True, 2.5):
        with pytest.raises(ValueError, match="budget"):
            evict_tokens(c, bad)
    for bad in (-1, 5, True, 1.0):
        with pytest.raises(ValueError, match="recent"):
            evict_tokens(c, 4, recent=bad)


def test_streaming_decode_budget_checks():
    m = tiny_model()
    for bad in (0, -1, True, 2.0):
        with pytest.raises(ValueError, match="decode_budget"):
            StreamingController(m, decode_budget=bad)
    ctl = StreamingController(m, decode_budget=8)
    try:
        with pytest.raises(ValueError, match="decode mode"):
            ctl.draft(torch.eye(2, dtype=torch.bool))
        ctl.finish_prefill()
        with pytest.raises(ValueError, match="bool matrix"):
            ctl.draft(torch.eye(2))
        with pytest.raises(ValueError, match="No drafts"):
            ctl.accept([0])
    finally:
        ctl.restore()


def test_oracle_attention_is_softmax():
    g = torch.Generator().manual_seed(1)
    q, kn, vn = torch.randn(1, 4, 3, 8, generator=g), torch.randn(1, 2, 3, 8, generator=g), torch.randn(1, 2, 3, 8, generator=g)
    k, v = torch.randn(1, 2, 9, 8, generator=g), torch.randn(1, 2, 9, 8, generator=g)
    lengths = torch.tensor([[9, 4]])
    out, lse, _ = O.tree_attention(q, kn, vn, k, v, lengths)
    for h in range(4):
        n = int(lengths[0, h // 2])
        keys, values = torch.cat([k[0, h // 2, :n], kn[0, h // 2]]).double(), torch.cat([v[0, h // 2, :n], vn[0, h // 2]]).double()
        x = q[0, h].double() @ keys.T * 8 ** -0.5
        x = x.masked_fill(torch.arange(n + 3)[None] > torch.arange(n, n + 3)[:, None], -math.inf)
        torch.testing.assert_close(out[0, h], torch.softmax(x, -1) @ values)
        torch.testing.assert_close(lse[0, h], torch.logsumexp(x, -1))


def test_oracle_commit_continues_the_importance():
    # weights of a causal prompt, recomputed whole and continued one token at a time
    from oracle import restate
    g = torch.Generator().manual_seed(2)
    q, k, v = torch.randn(1, 4, 12, 8, generator=g), torch.randn(1, 2, 12, 8, generator=g), torch.randn(1, 2, 12, 8, generator=g)
    n, decay = 9, 0.2
    _, whole = restate.materialized(q, k, v, recency_decay=decay)
    _, mass = restate.materialized(q[:, :, :n], k[:, :, :n], v[:, :, :n], recency_decay=decay)
    mass, norms, pos = torch.tensor(mass), v[:, :, :n].abs().sum(-1), torch.arange(n).expand(1, 2, n)
    at = slice(n, 12)
    _, lse, _ = O.tree_attention(q[:, :, at], k[:, :, at], v[:, :, at], k[:, :, :n], v[:, :, :n], torch.tensor([[n, n]]))
    cap = torch.cat([k[:, :, :n], torch.zeros(1, 2, 5, 8)], 2), torch.cat([v[:, :, :n], torch.zeros(1, 2, 5, 8)], 2)
    rows = O.commit(*cap, torch.tensor([[n, n]]), mass, norms, pos, q[:, :, at], k[:, :, at], v[:, :, at], lse,
                    torch.tensor([[0, 1, 2]]), torch.arange(n, 12)[None], decay=decay)
    for h in range(2):
        torch.testing.assert_close(rows[0, h][2], torch.as_tensor(whole)[0, h].double(), rtol=1e-5, atol=1e-6)
        assert rows[0, h][4].tolist() == list(range(12))


def test_oracle_evict_fills_holes_in_order():
    assert O.evict_slots([1.0, 2.0], [0, 1], 2, 0) == [0, 1]
    # slots 0 and 2 go; 3 and 4 (of weight 5, 4) take their places in order
    assert O.evict_slots([0.0, 3.0, 1.0, 5.0, 4.0], [0, 1, 2, 3, 4], 3, 0) == [3, 1, 4]
    # the newest position is kept whatever its weight; NaN counts as the largest; ties to the lower slot
    assert O.evict_slots([0.0, math.nan, 1.0, 1.0], [9, 1, 2, 3], 3, 1) == [0, 1, 2]
