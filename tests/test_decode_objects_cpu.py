"""KVCache objects on the host: what they keep alive, and what the operators hand to the library."""
import gc
import weakref

import pytest
import torch

from flash_evict.decode import KVCache, _check_out


def host_cache(k, v):
    """A KVCache of CPU tensors (the constructor wants a GPU's), with bookkeeping of its own."""
    cache = KVCache.__new__(KVCache)
    row = k.shape[:3]
    for name, value in (("k", k), ("v", v), ("lengths", torch.zeros(row[:2], dtype=torch.int32)), ("mass", torch.zeros(row)),
                        ("positions", torch.zeros(row, dtype=torch.int32)), ("norms", None), ("device", k.device), ("dtype", k.dtype),
                        ("_sync", None), ("_sizes", {}), ("_over", lambda: None), ("_c", None), ("_ref", None), ("_device_index", 0)):
        object.__setattr__(cache, name, value)
    return cache


def test_caches_that_take_turns_do_not_keep_each_other():
    k, v = torch.zeros(2, 1, 2, 8, 8)
    a, b = host_cache(k, v), host_cache(k, v)
    assert _check_out(a, b) is b and _check_out(b, a) is a and _check_out(a, b) is b
    books = [weakref.ref(c.mass) for c in (a, b)]
    gc.disable()
    try:
        del a
        assert books[0]() is None and books[1]() is not None
        # whoever comes in its place is checked anew
        with pytest.raises(ValueError, match="own k and v"):
            _check_out(host_cache(k.clone(), v), b)
        del b
        assert books[1]() is None
    finally:
        gc.enable()


def test_a_budget_past_64_bits_reaches_the_library_as_one_that_holds_everything(monkeypatch):
    from flash_evict import decode
    k = torch.zeros(1, 2, 8, 8)
    cache, sent = host_cache(k, k), []
    monkeypatch.setattr(decode, "_workspace", lambda cache, key, bytes_of, *args: (0, None, None))
    monkeypatch.setattr(decode, "_call", lambda fn, device, ref, out, budget, recent, *rest: sent.append((budget, recent)))
    for budget, recent in ((3, 2), (8, 8), (9, 9), (1 << 40, 7), (2 ** 64 + 1, 0), (2 ** 64 + 2, 2 ** 64 + 1)):
        assert decode.evict_tokens(cache, budget, recent=recent) is cache
    assert sent == [(3, 2), (8, 8), (8, 8), (8, 7), (8, 0), (8, 8)]
