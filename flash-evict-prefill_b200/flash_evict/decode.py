"""Decoding over a budgeted KV cache.

After `evict()` (or the streaming adapter) has cut a prompt's K/V down to a
budget, decoding adds tokens to the kept ones.  Three operators make up a step,
all on the current CUDA stream, with no host synchronisation (the lengths stay
on the device, so a step can be captured in a CUDA graph):

  tree_attention(q, k_new, v_new, cache, tree=...)  -> fe_tree_attention
      drafted tokens (one: an ordinary step) attend to the cache and to each other
  commit_tokens(cache, q, k_new, v_new, lse, accepted, positions)
                                                    -> fe_commit_tokens
      the accepted drafts' attention weight is added to every cached token's, and
      their K/V rows to the cache
  evict_tokens(cache, budget, recent=...)           -> fe_evict_tokens
      rows over their budget lose the tokens of least weight, in place
"""
import ctypes
import functools
import math
import weakref

import torch

from . import _lib
from .prefill import _tma_view

__all__ = ["KVCache", "tree_attention", "commit_tokens", "evict_tokens", "MAX_DRAFTS"]

MAX_DRAFTS = 128

_raw_stream = torch._C._cuda_getCurrentRawStream
_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


class KVCache:
    """K/V of the kept tokens of one layer, and what is known about each.

    k, v: [B, Hkv, C, D] fp16 or bf16; row (b, h) uses its first lengths[b, h]
    slots, in any order (a cached key carries its rotary position).  Any strides
    with channel stride 1, the others multiples of 8 elements, on a 16-byte base.
    lengths: int32 [B, Hkv].  Optional, contiguous [B, Hkv, C]: mass (FP32, the
    accumulated attention weight), positions (int32, the token's place in its
    sequence; required with mass) and norms (FP32, ||v||_1; when given, weights
    are scaled by it as `prefill(value_weighted=True)` scales its importance).
    Slots past a row's length may hold anything.  The tensors are kept, not
    copied, and cannot be replaced: update them in place.
    """

    __slots__ = ("k", "v", "lengths", "mass", "positions", "norms", "device", "dtype", "_sync", "_sizes", "_over", "_c", "_ref",
                 "_device_index", "__weakref__")

    def __init__(self, k, v, lengths, mass=None, positions=None, norms=None):
        if k.ndim != 4 or k.shape != v.shape or k.numel() == 0 or k.shape[-1] > 256:
            raise ValueError("K/V must be nonempty, of one shape [batch, kv_heads, capacity, channels <= 256]")
        if k.dtype not in _DTYPES or v.dtype != k.dtype or not k.is_cuda or v.device != k.device:
            raise ValueError("K/V must be CUDA fp16 or bf16 tensors of one dtype and device")
        for t in (k, v):
            if t.stride(3) != 1 or t.data_ptr() % 16 or any(s % 8 or s <= 0 for s, n in zip(t.stride()[:3], t.shape) if n > 1):
                raise ValueError("cache K/V need channel stride 1, other strides positive multiples of 8, a 16-byte base")
        if (mass is None) != (positions is None) or (norms is not None and mass is None):
            raise ValueError("mass and positions go together, and norms need them")
        for name, t, shape, dtype in (("lengths", lengths, k.shape[:2], torch.int32), ("mass", mass, k.shape[:3], torch.float32),
                                      ("positions", positions, k.shape[:3], torch.int32), ("norms", norms, k.shape[:3], torch.float32)):
            if t is not None and (t.shape != shape or t.dtype != dtype or t.device != k.device or not t.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on the cache's device")
        init = object.__setattr__
        for name, t in (("k", k), ("v", v), ("lengths", lengths), ("mass", mass), ("positions", positions), ("norms", norms)):
            init(self, name, t)
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        b, h, c, d = k.shape
        init(self, "_sync", None)  # made by the first commit in place outside a capture
        init(self, "_c", _lib.Cache(k.data_ptr(), v.data_ptr(), k.stride(), v.stride(), ptr(mass), ptr(norms), ptr(positions),
                                    lengths.data_ptr(), None, b, h, c, d, _DTYPES[k.dtype]))
        init(self, "_ref", ctypes.byref(self._c))
        init(self, "_sizes", {})  # workspace bytes by the calls' shapes
        init(self, "_over", lambda: None)  # gives the cache that this one was last checked to be another bookkeeping of
        _lib.check(_lib.load().fe_cache_prepare(self._ref))
        init(self, "device", k.device)
        init(self, "dtype", k.dtype)
        init(self, "_device_index", k.device.index)

    def __setattr__(self, name, value):
        raise AttributeError("a KVCache's tensors cannot be replaced; update them in place")

    def _make_sync(self):
        # The word that counts a commit's CTAs: zero before and after.  Under capture it
        # is zeroed by the graph only, so the graph has one of its own and the cache none.
        word = torch.zeros(1, dtype=torch.int32, device=self.device)
        with torch.cuda.device(self.device):
            if not torch.cuda.is_current_stream_capturing():
                object.__setattr__(self, "_sync", word)
        self._c.sync = word.data_ptr()
        return word

    @classmethod
    def allocate(cls, batch, kv_heads, capacity, channels, dtype=torch.bfloat16, device="cuda", *, value_weighted=True):
        """An empty cache of `capacity` slots a row, with all its bookkeeping."""
        if min(batch, kv_heads, capacity, channels) < 1:
            raise ValueError("batch, kv_heads, capacity and channels must be positive")
        pitch = (channels + 7) // 8 * 8
        k, v = (torch.zeros(batch, kv_heads, capacity, pitch, dtype=dtype, device=device)[..., :channels] for _ in range(2))
        row = (batch, kv_heads, capacity)
        return cls(k, v, torch.zeros(row[:2], dtype=torch.int32, device=device), torch.zeros(row, device=device),
                   torch.zeros(row, dtype=torch.int32, device=device), torch.zeros(row, device=device) if value_weighted else None)

    def fill(self, k, v, positions=None, mass=None):
        """Replace the cache's contents by k, v [B, Hkv, n, D] (kept rows of a prefill).

        positions: the tokens' places ([B, Hkv, n] or broadcastable; default
        0..n-1), as `select_tokens`' indices; mass: their weights (default 0), as
        the gathered importance.  Returns the cache.
        """
        b, h, c, d = self.k.shape
        n = k.shape[2] if k.ndim == 4 else -1
        if k.shape != v.shape or tuple(k.shape) != (b, h, n, d) or n > c:
            raise ValueError("rows to fill in must have shape [batch, kv_heads, n <= capacity, channels]")
        self.k[:, :, :n].copy_(k)
        self.v[:, :, :n].copy_(v)
        self.lengths.fill_(n)
        if self.mass is not None:
            self.positions[:, :, :n].copy_(torch.arange(n, device=k.device) if positions is None else positions)
            if mass is None:
                self.mass[:, :, :n].zero_()
            else:
                self.mass[:, :, :n].copy_(mass)
            if self.norms is not None:
                torch.sum(self.v[:, :, :n].abs(), -1, dtype=torch.float32, out=self.norms[:, :, :n])
        return self


@functools.lru_cache(maxsize=1024)
def _stride_array(strides):
    return (ctypes.c_int64 * 4)(*strides)


def _readable(t):
    """(tensor, its stride array): t if the kernels can read it in place, else a copy that they can."""
    st = t.stride()
    if st[3] != 1 or (st[0] | st[1] | st[2]) & 7 or t.data_ptr() & 15 or 0 in st:
        t = _tma_view(t.contiguous() if 0 in st else t)  # expanded dimensions are laid out
        st = t.stride()
    return t, _stride_array(st)


def _workspace(cache, key, bytes_of, *args):
    # (size, tensor, pointer) of a call's workspace; its size depends on the shapes alone.
    size = cache._sizes.get(key)
    if size is None:
        size = bytes_of(*args)
        if size < 0:
            _lib.check(_lib.STATUS_UNSUPPORTED)
        cache._sizes[key] = size
    if size == 0:
        return 0, None, None
    tensor = torch.empty(size, dtype=torch.uint8, device=cache.device)
    return size, tensor, tensor.data_ptr()


def _call(fn, device_index, *args):
    # One launch sequence on the cache's device and its current stream.
    if torch._C._cuda_getDevice() == device_index:
        rc = fn(*args, _raw_stream(device_index))
    else:
        with torch.cuda.device(device_index):
            rc = fn(*args, _raw_stream(device_index))
    if rc:
        _lib.check(rc)


def _check_drafts(q, k_new, v_new, cache, tree, scale):
    """Checks shared by the operators that take drafted tokens; returns (tree, its batch stride, scale)."""
    b, hk, _, d = cache.k.shape
    shape = q.shape
    if len(shape) != 4 or shape[0] != b or shape[3] != d or shape[1] % hk or not shape[1]:
        raise ValueError("q must have shape [batch, q_heads, drafts, channels], q_heads a multiple of the cache's kv_heads")
    t = shape[2]
    if not 1 <= t <= MAX_DRAFTS:
        raise ValueError(f"between 1 and {MAX_DRAFTS} drafted tokens per call")
    shape = (b, hk, t, d)
    if k_new.shape != shape or v_new.shape != shape:
        raise ValueError("k_new and v_new must have shape [batch, kv_heads, drafts, channels]")
    device = cache.device
    if not (q.dtype == k_new.dtype == v_new.dtype == cache.dtype) or not (q.device == k_new.device == v_new.device == device):
        raise ValueError("q, k_new, v_new and the cache must have the same device and dtype")
    if (q.requires_grad or k_new.requires_grad or v_new.requires_grad) and torch.is_grad_enabled():
        raise ValueError("Inference only: no backward implementation")
    stride = 0
    if tree is not None:
        if tree.dtype != torch.bool or tree.device != device or tree.shape not in ((t, t), (b, t, t)):
            raise ValueError("tree must be a bool tensor of shape [drafts, drafts] or [batch, drafts, drafts] on the cache's device")
        if not tree.is_contiguous():
            tree = tree.contiguous()
        stride = t * t if tree.ndim == 3 else 0
    scale = d ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    return tree, stride, scale


def tree_attention(q, k_new, v_new, cache, *, tree=None, scale=None):
    """Attention of drafted tokens over a cache and over each other: (out, lse).

    q [B, Hq, T, D], k_new/v_new [B, Hkv, T, D]: T drafted tokens (1..128) of each
    sequence; Hq a multiple of Hkv.  Draft t sees all of its row's cached tokens
    and the drafts j with tree[t, j] (bool [T, T] or [B, T, T]; None: j <= t, so a
    single token or a chain).  The cache is not changed: `commit_tokens` adds the
    drafts that were accepted.

    out [B, Hq, T, D] in q's dtype; lse FP32 [B, Hq, T], the natural log of the
    sum of exp(scale * q.k).  A row that sees nothing gives out 0 and lse -inf.
    """
    tree, tree_stride, scale = _check_drafts(q, k_new, v_new, cache, tree, scale)
    b, hq, t, d = q.shape
    lib = _lib.load()
    size, workspace, pointer = _workspace(cache, (hq, t), lib.fe_tree_workspace_bytes, cache._ref, hq, t)
    out = q.new_empty((b, hq, t, d))
    lse = torch.empty((b, hq, t), dtype=torch.float32, device=q.device)
    q, qs = _readable(q)
    k_new, ks = _readable(k_new)
    v_new, vs = _readable(v_new)
    _call(lib.fe_tree_attention, cache._device_index, cache._ref, q.data_ptr(), qs, k_new.data_ptr(), ks, v_new.data_ptr(), vs,
          None if tree is None else tree.data_ptr(), tree_stride, out.data_ptr(), lse.data_ptr(), pointer, size, hq, t, scale)
    return out, lse


def _check_out(cache, out):
    if cache.mass is None:
        raise ValueError("the cache has no mass and positions")
    if out is None or out is cache:
        return cache
    if out._over() is cache:  # neither's tensors can have been replaced since
        return out
    if out.mass is None or (out.norms is None) != (cache.norms is None) or out.mass.data_ptr() == cache.mass.data_ptr() \
            or out.positions.data_ptr() == cache.positions.data_ptr() or out.lengths.data_ptr() == cache.lengths.data_ptr() \
            or (out.norms is not None and out.norms.data_ptr() == cache.norms.data_ptr()):
        raise ValueError("out needs bookkeeping tensors of its own, the same ones that the cache has")
    if cache.k.data_ptr() != out.k.data_ptr() or cache.v.data_ptr() != out.v.data_ptr() or cache.k.shape != out.k.shape \
            or cache.k.dtype != out.k.dtype or cache.k.stride() != out.k.stride() or cache.v.stride() != out.v.stride():
        raise ValueError("out must hold the cache's own k and v")
    object.__setattr__(out, "_over", weakref.ref(cache))
    return out


def commit_tokens(cache, q, k_new, v_new, lse, accepted, positions, *, tree=None, scale=None, recency_decay=0., out=None):
    """Add accepted drafts to the cache; returns the cache with the updated bookkeeping.

    q, k_new, v_new, tree, scale as for `tree_attention`, lse as it returned it.
    accepted: int32 [B, A], the accepted drafts of each sequence in their order
    (the path from the tree's root), negative entries none, A at most 128.
    positions: int32 [B, T], the drafts' places in their sequences.

    With n accepted drafts, every token's weight becomes
      mass = exp(-recency_decay * n) * mass + norm * sum_{i,heads} w_i * p_i,
      w_i = exp(-recency_decay * (n - 1 - i)),
    p_i the attention probability that accepted draft i gives it (norm 1 if the
    cache has no norms): `prefill`'s importance, continued over the new tokens.
    The appended tokens' weights are those that the accepted drafts give them.
    Rows that do not fit are dropped and reported as `check_status` describes.

    out: a KVCache of the same k and v with bookkeeping of its own, which then
    receives the new mass, norms, positions and lengths (slots below the new
    lengths only) while `cache` keeps the old ones.  Default: in place.
    """
    out = _check_out(cache, out)
    tree, tree_stride, scale = _check_drafts(q, k_new, v_new, cache, tree, scale)
    b, hq, t, _ = q.shape
    device = cache.device
    if lse.shape != (b, hq, t) or lse.dtype != torch.float32 or lse.device != device:
        raise ValueError("lse must be FP32 [batch, q_heads, drafts] on the cache's device")
    if accepted.ndim != 2 or accepted.shape[0] != b or not 1 <= accepted.shape[1] <= MAX_DRAFTS or accepted.dtype != torch.int32 \
            or accepted.device != device:
        raise ValueError(f"accepted must be int32 [batch, 1..{MAX_DRAFTS}] on the cache's device")
    if positions.shape != (b, t) or positions.dtype != torch.int32 or positions.device != device:
        raise ValueError("positions must be int32 [batch, drafts] on the cache's device")
    recency_decay = float(recency_decay)
    if not math.isfinite(recency_decay) or recency_decay < 0:
        raise ValueError("recency_decay must be finite and nonnegative")
    sync = cache._make_sync() if out is cache and cache._sync is None else None  # (kept until the launch)
    lib = _lib.load()
    a = accepted.shape[1]
    size, workspace, pointer = _workspace(cache, (hq, t, a, out is cache), lib.fe_commit_workspace_bytes, cache._ref, out._ref, hq, t, a)
    q, qs = _readable(q)
    k_new, ks = _readable(k_new)
    v_new, vs = _readable(v_new)
    if not (lse.is_contiguous() and accepted.is_contiguous() and positions.is_contiguous()):
        lse, accepted, positions = lse.contiguous(), accepted.contiguous(), positions.contiguous()
    _call(lib.fe_commit_tokens, cache._device_index, cache._ref, out._ref, q.data_ptr(), qs, k_new.data_ptr(), ks,
          v_new.data_ptr(), vs, None if tree is None else tree.data_ptr(), tree_stride,
          lse.data_ptr(), accepted.data_ptr(), a, positions.data_ptr(), pointer, size, hq, t,
          scale, recency_decay)
    return out


def evict_tokens(cache, budget, *, recent=0, out=None):
    """Cut every row of more than `budget` tokens back to `budget`; returns the cache with the updated bookkeeping.

    Kept are the tokens whose position lies within `recent` of the row's newest,
    then those of the largest mass (NaN above every number, ties by lower slot).
    K/V rows move in place: kept tokens below slot `budget` stay, the i-th evicted
    slot there takes the i-th kept token from above, so a step that is one token
    over moves one row and the slots' order is not the tokens'.  `out` as for
    `commit_tokens`, but k and v change all the same.
    """
    out = _check_out(cache, out)
    if isinstance(budget, bool) or not isinstance(budget, int) or budget < 1:
        raise ValueError("budget must be a positive integer")
    if isinstance(recent, bool) or not isinstance(recent, int) or not 0 <= recent <= budget:
        raise ValueError("recent must be an integer in [0, budget]")
    budget = min(budget, cache.k.shape[2])  # a row holds no more
    recent = min(recent, budget)
    lib = _lib.load()
    size, workspace, pointer = _workspace(cache, budget, lib.fe_evict_workspace_bytes, cache._ref, budget)
    _call(lib.fe_evict_tokens, cache._device_index, cache._ref, out._ref, budget, recent, pointer, size)
    return out
