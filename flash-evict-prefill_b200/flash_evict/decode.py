"""Decoding over a budgeted KV cache.

After `evict()` (or the streaming adapter) has cut a prompt's K/V down to a
budget, decoding adds tokens to the kept ones.  Three operators make up a step,
all on the current CUDA stream, with no host synchronisation (the lengths stay
on the device, so a step can be captured in a CUDA graph):

  tree_attention(q, k_new, v_new, cache, tree=...)  -> fe_tree_attention
      drafted tokens (one: an ordinary step) attend to the cache and to each other
"""
import ctypes
import math

import torch

from . import _lib
from .prefill import _tma_view

__all__ = ["KVCache", "tree_attention", "MAX_DRAFTS"]

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

    __slots__ = ("k", "v", "lengths", "mass", "positions", "norms", "_c", "_ref", "_device_index")

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
        init(self, "_c", _lib.Cache(k.data_ptr(), v.data_ptr(), k.stride(), v.stride(), ptr(mass), ptr(norms), ptr(positions),
                                    lengths.data_ptr(), b, h, c, d, _DTYPES[k.dtype]))
        init(self, "_ref", ctypes.byref(self._c))
        init(self, "_device_index", k.device.index)

    def __setattr__(self, name, value):
        raise AttributeError("a KVCache's tensors cannot be replaced; update them in place")

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


def _strides(t):
    return (ctypes.c_int64 * 4)(*t.stride())


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
    ck = cache.k
    b, hk, _, d = ck.shape
    if q.ndim != 4 or q.shape[0] != b or q.shape[3] != d or q.shape[1] % hk or not q.shape[1]:
        raise ValueError("q must have shape [batch, q_heads, drafts, channels], q_heads a multiple of the cache's kv_heads")
    t = q.shape[2]
    if not 1 <= t <= MAX_DRAFTS:
        raise ValueError(f"between 1 and {MAX_DRAFTS} drafted tokens per call")
    shape = (b, hk, t, d)
    if k_new.shape != shape or v_new.shape != shape:
        raise ValueError("k_new and v_new must have shape [batch, kv_heads, drafts, channels]")
    if not (q.dtype == k_new.dtype == v_new.dtype == ck.dtype) or not (q.device == k_new.device == v_new.device == ck.device):
        raise ValueError("q, k_new, v_new and the cache must have the same device and dtype")
    if torch.is_grad_enabled() and (q.requires_grad or k_new.requires_grad or v_new.requires_grad):
        raise ValueError("Inference only: no backward implementation")
    stride = 0
    if tree is not None:
        if tree.dtype != torch.bool or tree.device != ck.device or tree.shape not in ((t, t), (b, t, t)):
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
    size = lib.fe_tree_workspace_bytes(cache._ref, hq, t)
    if size < 0:
        _lib.check(_lib.STATUS_UNSUPPORTED)
    device = q.device
    out = torch.empty((b, hq, t, d), dtype=q.dtype, device=device)
    lse = torch.empty((b, hq, t), dtype=torch.float32, device=device)
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    if q.stride(3) != 1:
        q = q.contiguous()
    k_new, v_new = _tma_view(k_new), _tma_view(v_new)
    _call(lib.fe_tree_attention, cache._device_index, cache._ref, q.data_ptr(), _strides(q), k_new.data_ptr(), _strides(k_new),
          v_new.data_ptr(), _strides(v_new), None if tree is None else tree.data_ptr(), tree_stride, out.data_ptr(),
          lse.data_ptr(), workspace.data_ptr(), size, hq, t, scale)
    return out, lse
