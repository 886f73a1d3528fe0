"""Per-layer prefill-and-compact on a transformers Qwen2 model.

Mirrors the reference's streaming adapter (flash_evict/streaming_adapter.py:
`StreamingController` :17-31, `chunk_mlp` :34-54, the patched attention
forward :57-87) for the Qwen2 attention modules of the installed transformers
(5.x, where the decoder layer hands each attention module its rotary
`position_embeddings`).  The reference builds on the external kv_distill
Controller (its prefill/decode modes, per-layer `states`, and decoding over
the compacted cache); that package is not available, so this controller keeps
those pieces itself:

* prefill (``mode == 'prefill'``), one unpadded prompt, no external cache:
  each layer projects q/k/v, views them ``[B,N,H,D]`` and transposes them
  (no copy; the kernels read the strided views), applies RoPE, and then
    - ``'fused'``: ``prefill(q, k, v, **scoring)`` for the dense output and the
      importance, then one launch that selects ``min(N, budget)`` tokens with
      ``reserved_recent`` pinned and ``pool_kernel`` pooling and gathers the
      kept K/V rows (streaming_adapter.py:61-66,86);
    - ``'snap'``: dense attention, SnapKV window-32 scores and selection, gather
      (streaming_adapter.py:78-83,86);
    - ``'full'``: dense attention, the whole K/V kept.
  The dense attention output always feeds ``o_proj``: only the stored K/V are
  compacted, so the next layer sees exactly the uncompressed model's input.
* decode (after ``finish_prefill()``): every new token's K/V is appended to its
  layer's stored K/V and its query attends to all of them (plus the new tokens
  before it); positions continue from the caller's ``position_ids``.  Decode
  attention is torch's ``scaled_dot_product_attention`` over a growing cache;
* decode under a budget (``decode_budget=``): each layer's kept K/V go into a
  ``flash_evict.decode.KVCache`` together with their importance.  A call's new
  tokens attend with ``tree_attention``, add their attention weight to the kept
  tokens and are appended (``commit_tokens``), and the cache is cut back to
  ``decode_budget`` by weight, the newest ``reserved_recent`` tokens excepted
  (``evict_tokens``); calls of more than 128 tokens go in parts of 128.  For speculative decoding, ``draft(tree)`` makes the next
  call's tokens a tree of drafts that are not appended until
  ``accept(path)`` names the ones to keep.

The model is called with ``use_cache=False``; the controller owns the cache
(``states[layer_idx] = {'k', 'v', 'indices'}``, with a decode budget
``{'cache', 'indices', ...}``).
"""
import types

import torch
import torch.nn.functional as F

from .baselines import flash_attention, snap_scores, snap_select
from .compact import gather_tokens, select_and_gather
from .decode import MAX_DRAFTS, KVCache, commit_tokens, evict_tokens, tree_attention
from .prefill import prefill

__all__ = ["StreamingController", "chunk_mlp"]


def _attention_modules(model):
    return [layer.self_attn for layer in model.model.layers]


class StreamingController:
    """Compact every layer's K/V cache during prefill (streaming_adapter.py:17-31).

    Same keyword arguments, defaults and ValueErrors as the reference's
    ``StreamingController``.  ``scoring`` is passed to ``prefill`` as keyword
    arguments (e.g. ``{'recency_decay': 0.1}``).  ``restore()`` puts the
    model's original attention forwards back.

    ``decode_budget`` (default None: the caches grow) bounds every layer's cache
    while decoding.  Tokens then compete by importance: the prefill's (``'fused'``
    with ``scoring``, ``'snap'``'s scores; 0 with ``'full'``) plus the attention
    weight that decoded tokens give them.
    """

    def __init__(self, model, *, backend="fused", budget=1024, scoring=None, reserved_recent=64, pool_kernel=1,
                 decode_budget=None):
        if backend not in ("fused", "snap", "full"):
            raise ValueError("Unsupported backend")
        if isinstance(budget, bool) or not isinstance(budget, int) or budget < 1:
            raise ValueError("Positive integer budget required")
        if decode_budget is not None and (isinstance(decode_budget, bool) or not isinstance(decode_budget, int)
                                          or decode_budget < 1):
            raise ValueError("decode_budget must be a positive integer or None")
        self.model = model
        self.decode_budget = decode_budget
        self.tree = None
        self.prefill_backend = backend
        self.cache_budget = budget
        self.scoring = {} if scoring is None else dict(scoring)
        self.reserved_recent = reserved_recent
        self.pool_kernel = pool_kernel
        self.mode = "prefill"
        self.states = {}
        self.originals = [(attn, attn.forward) for attn in _attention_modules(model)]
        for attn, _ in self.originals:
            attn._kv_controller = self
            attn.forward = types.MethodType(_forward, attn)

    def finish_prefill(self):
        """Switch to decoding over the compacted caches (streaming_adapter.py:29-30)."""
        self.mode = "decode"

    def reset(self):
        """Drop every cache and return to prefill mode for the next prompt."""
        self.mode = "prefill"
        self.states = {}
        self.tree = None

    def draft(self, tree):
        """Make the next call's tokens drafts: token t sees the cache and the drafts j with ``tree[t, j]`` (bool [T, T]).

        Nothing is appended until ``accept``; drafts of an earlier tree that were not accepted are dropped.  Give the call
        ``position_ids`` by depth in the tree.
        """
        if self.decode_budget is None or self.mode != "decode":
            raise ValueError("Drafts need decode_budget and decode mode")
        if tree.ndim != 2 or tree.shape[0] != tree.shape[1] or not 1 <= tree.shape[0] <= MAX_DRAFTS or tree.dtype != torch.bool:
            raise ValueError(f"tree must be a bool matrix of 1 to {MAX_DRAFTS} drafts")
        for state in self.states.values():
            state.pop("drafts", None)
        self.tree = tree

    def accept(self, path):
        """Append the drafts of the last call named by ``path`` (indices from the tree's root on; may be empty) and drop the rest."""
        if self.tree is None or any("drafts" not in s for s in self.states.values()):
            raise ValueError("No drafts to accept")
        path = [int(j) for j in path]
        if len(path) > MAX_DRAFTS or any(not 0 <= j < self.tree.shape[0] for j in path):
            raise ValueError("path must name drafts of the tree")
        for state in self.states.values():
            drafts = state.pop("drafts")
            if path:
                accepted = torch.tensor([path], dtype=torch.int32, device=state["cache"].device)
                _commit(self, state, *drafts, accepted, self.tree)
        self.tree = None

    def restore(self):
        """Give the attention modules their original forward back."""
        for attn, original in self.originals:
            attn.forward = original
            if hasattr(attn, "_kv_controller"):
                del attn._kv_controller
        self.originals = []


def chunk_mlp(model, chunk_size):
    """Run every layer's feed-forward block on at most ``chunk_size`` tokens at a time.

    Bounds the activation memory of inference on long prompts; returns a
    function that restores the original MLP forwards (streaming_adapter.py:34-54).
    The GEMM shapes change, so results may differ in the last bits.
    """
    if isinstance(chunk_size, bool) or not isinstance(chunk_size, int) or chunk_size < 1:
        raise ValueError("chunk_size must be a positive integer")
    saved = []

    def chunked_forward(original):
        def run(hidden):
            if torch.is_grad_enabled():
                raise RuntimeError("Chunked MLP is inference-only")
            n = hidden.shape[1]
            if n <= chunk_size:
                return original(hidden)
            out = torch.empty_like(hidden)
            for start in range(0, n, chunk_size):
                out[:, start:start + chunk_size] = original(hidden[:, start:start + chunk_size])
            return out
        return run

    for layer in model.model.layers:
        saved.append((layer.mlp, layer.mlp.forward))
        layer.mlp.forward = chunked_forward(layer.mlp.forward)

    def restore():
        for mlp, original in saved:
            mlp.forward = original

    return restore


def _decode_attention(q, k, v, scale):
    # q [B,Hq,n,D] are the newest n positions of the Hkv-headed k/v [B,Hkv,L,D].
    n, total = q.shape[2], k.shape[2]
    mask = None
    if n > 1:
        qpos = torch.arange(total - n, total, device=q.device)[:, None]
        mask = torch.arange(total, device=q.device)[None, :] <= qpos
    return F.scaled_dot_product_attention(q, k, v, attn_mask=mask, scale=scale, enable_gqa=True)


def _fill_cache(ctl, state, n, idx, weights, k, v):
    # The kept rows of an n-token prompt, their positions and importance, with
    # room for one call's drafts past the budget.
    kept = k.shape[2]
    cache = KVCache.allocate(1, k.shape[1], max(kept, ctl.decode_budget) + MAX_DRAFTS, k.shape[3], k.dtype, k.device,
                             value_weighted=ctl.prefill_backend == "fused" and ctl.scoring.get("value_weighted", True))
    mass = None if weights is None else weights if idx is None else weights.gather(2, idx)
    state["cache"] = evict_tokens(cache.fill(k, v, idx, mass), ctl.decode_budget, recent=min(ctl.decode_budget, ctl.reserved_recent))
    state["next"] = torch.full((1, 1), n, dtype=torch.int32, device=k.device)


def _commit(ctl, state, q, k, v, lse, accepted, tree=None):
    t = q.shape[2]
    depth = torch.arange(t, device=q.device)[None] if tree is None else tree.sum(1)[None] - 1
    positions = (state["next"] + depth).to(torch.int32)
    commit_tokens(state["cache"], q, k, v, lse, accepted, positions, tree=tree, scale=state["scale"],
                  recency_decay=ctl.scoring.get("recency_decay", 0.))
    evict_tokens(state["cache"], ctl.decode_budget, recent=min(ctl.decode_budget, ctl.reserved_recent))
    state["next"] += accepted.shape[1]


def _budgeted_attention(ctl, state, q, k, v, scale):
    state["scale"] = scale
    t = q.shape[2]
    if ctl.tree is not None:
        if ctl.tree.shape[0] != t:
            raise ValueError("The call's tokens are not the tree's drafts")
        out, lse = tree_attention(q, k, v, state["cache"], tree=ctl.tree, scale=scale)
        state["drafts"] = (q, k, v, lse)
        return out
    parts = []
    for at in range(0, t, MAX_DRAFTS):  # each part attends to the cache that the one before left
        part = [x[:, :, at:at + MAX_DRAFTS] for x in (q, k, v)]
        out, lse = tree_attention(*part, state["cache"], tree=None, scale=scale)
        _commit(ctl, state, *part, lse, torch.arange(part[0].shape[2], dtype=torch.int32, device=q.device)[None])
        parts.append(out)
    return parts[0] if len(parts) == 1 else torch.cat(parts, 2)


def _forward(self, hidden_states, position_embeddings=None, attention_mask=None, past_key_values=None, **kwargs):
    """Attention forward installed by StreamingController (streaming_adapter.py:57-87)."""
    ctl = self._kv_controller
    b, n, _ = hidden_states.shape
    if b != 1 or past_key_values is not None or kwargs.get("output_attentions"):
        raise ValueError("Streaming adapter expects one unpadded prompt and an empty external cache")
    if position_embeddings is None:
        raise ValueError("Streaming adapter needs the rotary position_embeddings of the decoder layer")
    from transformers.models.qwen2.modeling_qwen2 import apply_rotary_pos_emb

    hq, hk, d = self.config.num_attention_heads, self.config.num_key_value_heads, self.head_dim
    q = self.q_proj(hidden_states).view(b, n, hq, d).transpose(1, 2)
    k = self.k_proj(hidden_states).view(b, n, hk, d).transpose(1, 2)
    v = self.v_proj(hidden_states).view(b, n, hk, d).transpose(1, 2)
    cos, sin = position_embeddings
    q, k = apply_rotary_pos_emb(q, k, cos, sin)

    if ctl.mode == "prefill":
        budget = min(n, ctl.cache_budget)
        weights = None
        if ctl.prefill_backend == "fused":
            out, importance = prefill(q, k, v, **ctl.scoring)
            idx, _, k_kept, v_kept = select_and_gather(importance, budget, k, v,
                                                       reserved_recent=min(budget, ctl.reserved_recent),
                                                       pool_kernel=ctl.pool_kernel)
            weights = importance
        elif ctl.prefill_backend == "snap":
            out = flash_attention(q, k, v)
            weights = snap_scores(q, k, 32)
            idx, _ = snap_select(weights, budget, 32)
            k_kept, v_kept = gather_tokens(k, idx), gather_tokens(v, idx)
        else:
            out = flash_attention(q, k, v)
            idx, k_kept, v_kept = None, k, v
        state = ctl.states[self.layer_idx] = {"indices": idx}
        if ctl.decode_budget is None:
            state["k"], state["v"] = k_kept, v_kept
        else:
            _fill_cache(ctl, state, n, idx, weights, k_kept, v_kept)
    elif ctl.decode_budget is not None:
        out = _budgeted_attention(ctl, ctl.states[self.layer_idx], q, k, v, self.scaling)
    else:
        state = ctl.states[self.layer_idx]
        state["k"] = torch.cat([state["k"], k], dim=2)
        state["v"] = torch.cat([state["v"], v], dim=2)
        out = _decode_attention(q, state["k"], state["v"], self.scaling)
    out = out.transpose(1, 2).reshape(b, n, hq * d)
    return self.o_proj(out), None
