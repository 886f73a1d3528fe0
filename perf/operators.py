"""The decode operators over a budgeted KV cache: their cases, inputs, plain forms and exact results.

A decode step over a cache of kept tokens is three operators of `flash_evict.decode`:

  attend   attention of a tree of drafted tokens (one token: an ordinary decode step) over the cache
  commit   the accepted drafts' attention weight added to every cached token, their K/V rows appended
  evict    the cache cut back to its budget by accumulated weight, in place

With `own` false, `run` computes them in elementary torch operations in 32 bits; with `own` true it
makes the calls a user makes.  `exact` gives the results from the definitions in 64 bits.

A cache is k, v [B, Hkv, C, D] of which row (b, h) uses the first lengths[b, h] slots, and per slot a
weight (mass), the L1 norm of its value row (norms) and the token's position.  The bookkeeping of a
pass is written beside the old one (`out=`), so a pass can be repeated.
"""
import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _case(name, kind, **kw):
    c = dict(kind=kind, batch=1, q_heads=28, kv_heads=4, channels=128, dtype="float16", length=2048, spare=256, ragged=False,
             drafts=1, accept=1, decay=0.0, budget=0, recent=0)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one token over one layer's cache kept at a 2048-token budget (the smallest call of a decode loop)
        _case("attend-one-kept2048", "attend"),
        # a tree of 64 drafts over a whole 32768-token prompt
        _case("attend-tree64-32k", "attend", length=32768, drafts=64, accept=5),
        # a serving batch: one token per sequence, lengths spread from nothing to 8192, heads kept to different lengths
        _case("attend-batch16-ragged", "attend", batch=16, q_heads=32, kv_heads=8, dtype="bfloat16", length=8192, ragged=True),
        # the longest: 64 drafts over a 131072-token prompt
        _case("attend-tree64-131k", "attend", q_heads=32, kv_heads=8, dtype="bfloat16", length=131072, drafts=64, accept=8),
        # odd everything: 80 channels, 5 drafts, an odd ragged length, 3 sequences
        _case("attend-odd-d80", "attend", batch=3, q_heads=6, kv_heads=2, channels=80, length=1237, spare=64, ragged=True, drafts=5, accept=3),
        # the weight of one decoded token over the 2048-token budget
        _case("commit-one-kept2048", "commit", decay=0.1),
        # 5 of 64 drafts accepted over a 32768-token prompt
        _case("commit-tree64-32k", "commit", length=32768, drafts=64, accept=5),
        # the serving batch's step
        _case("commit-batch16-ragged", "commit", batch=16, q_heads=32, kv_heads=8, dtype="bfloat16", length=8192, ragged=True, decay=0.1),
        # a long accepted run over the 131072-token prompt
        _case("commit-run64-131k", "commit", q_heads=32, kv_heads=8, dtype="bfloat16", length=131072, drafts=64, accept=64),
        # one token over budget, as after every step of a decode loop
        _case("evict-one-kept2048", "evict", length=2049, budget=2048, recent=64),
        # a batch whose rows reach the budget at different times
        _case("evict-batch16-ragged", "evict", batch=16, q_heads=32, kv_heads=8, dtype="bfloat16", length=8192, ragged=True, budget=4096, recent=128),
        # a whole 131072-token prompt cut to 1024 tokens a head
        _case("evict-131k-to-1024", "evict", q_heads=32, kv_heads=8, dtype="bfloat16", length=131072, budget=1024, recent=64),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "commit", "commit", "evict"])
    hq, hk = rng.choice([(28, 4), (32, 8), (32, 32), (6, 2), (4, 2), (8, 1)])
    channels = rng.choice([128, 128, 64, 80, 256])
    batch = _log_uniform(rng, 1, 16)
    drafts = 1 if rng.random() < 0.35 else _log_uniform(rng, 2, 64)
    # at most the largest listed case's K/V bytes and products
    most = min((8 * 131072 * 128) // (batch * hk * channels), (2048 * 131072 * 128) // (batch * hq * drafts * channels), 131072)
    length = _log_uniform(rng, 1, max(1, most))
    budget = max(1, min(length, _log_uniform(rng, max(1, length // 64), length)))
    return _case(None, kind, batch=batch, q_heads=hq, kv_heads=hk, channels=channels, dtype=rng.choice(["float16", "bfloat16"]), length=length,
                 spare=rng.choice([64, 77, 256]), ragged=rng.random() < 0.5, drafts=drafts, accept=_log_uniform(rng, 1, drafts),
                 decay=rng.choice([0.0, 0.1]), budget=budget, recent=rng.choice([0, min(budget, 64), budget // 3]))


def _lengths(case):
    """The rows' lengths, batch and heads flat: all `length`, or spread evenly up to it, one of four rows or more empty."""
    n = case["batch"] * case["kv_heads"]
    if not case["ragged"]:
        return [case["length"]] * n
    return [case["length"] * (i + 1) // n if i or n < 4 else 0 for i in range(n)]


def _accepts(case):
    return [max(0, case["accept"] - b % 3) for b in range(case["batch"])]


def _trees(case, gen):
    """([B, T, T] mask of the drafts each draft sees, or None for one draft; [B, A] accepted drafts, -1 past their number)."""
    b, t, a = case["batch"], case["drafts"], case["accept"]
    mask = torch.zeros(b, t, t, dtype=torch.bool)
    path = torch.full((b, a), -1, dtype=torch.int32)
    for i, n in enumerate(_accepts(case)):
        live = t - (i % 3 if t >= 8 and t - 2 > a else 0)  # the last drafts of some sequences are padding and see no draft
        spine = [0] + sorted((torch.randperm(live - 1, generator=gen)[:a - 1] + 1).tolist())
        before = dict(zip(spine[1:], spine))
        for j in range(live):
            if j:
                mask[i, j] = mask[i, before[j] if j in before else int(torch.randint(0, j, (1,), generator=gen))]
            mask[i, j, j] = True
        path[i, :n] = torch.tensor(spine[:n], dtype=torch.int32)
    return (mask.cuda() if t > 1 else None), path.cuda()


def _book(case):
    b, h, c, dev = case["batch"], case["kv_heads"], case["length"] + case["spare"], "cuda"
    return dict(mass=torch.zeros(b, h, c, device=dev), norms=torch.zeros(b, h, c, device=dev),
                positions=torch.zeros(b, h, c, dtype=torch.int32, device=dev), lengths=torch.zeros(b, h, dtype=torch.int32, device=dev))


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, hq, hk, d, t = (case[n] for n in ("batch", "q_heads", "kv_heads", "channels", "drafts"))
    dtype, cap = DTYPES[case["dtype"]], case["length"] + case["spare"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    rows = torch.tensor(_lengths(case), dtype=torch.int32)
    lengths = rows[torch.randperm(b * hk, generator=gen)].view(b, hk).cuda()
    slots = torch.arange(cap, device="cuda")
    live = slots < lengths[..., None]
    # slots never written hold whatever was there: here large values
    # one key in a hundred draws much attention, as the first tokens of a prompt do
    sink = torch.where(torch.rand(b, hk, cap, 1, generator=g, device="cuda") < 0.01, 8.0, 1.0).to(dtype)
    k = torch.where(live[..., None], randn(b, hk, cap, d) * sink, 1000.0).to(dtype)
    v = torch.where(live[..., None], randn(b, hk, cap, d), 1000.0).to(dtype)
    # accumulated weights are heavy-tailed: a few tokens hold most of them
    mass = torch.where(live, torch.exp(2 * torch.randn(b, hk, cap, generator=g, device="cuda")), 0.0)
    norms = torch.where(live, v.float().abs().sum(-1), 0.0)
    # slots are not in order of age once holes have been filled; the newest `spare` tokens are
    old = (lengths - case["spare"]).clamp(min=0)[..., None]
    shuffled = torch.where(slots < old, torch.rand(b, hk, cap, generator=g, device="cuda"), 2.0).argsort(-1).argsort(-1)
    positions = torch.where(live, torch.where(slots < old, shuffled, slots), 0).to(torch.int32)
    book = dict(mass=mass, norms=norms, positions=positions, lengths=lengths)
    s = dict(case=case, k=k, v=v, book=book, out=_book(case))
    if case["kind"] != "evict":
        # as a model's projections hand them over: [B, T, H, D] buffers seen as [B, H, T, D]
        q, k_new, v_new = (randn(b, t, h, d).transpose(1, 2) for h in (hq, hk, hk))
        tree, accepted = _trees(case, gen)
        s.update(q=q, k_new=k_new, v_new=v_new, tree=tree, accepted=accepted, scale=d ** -0.5)
        depth = tree.sum(-1).clamp(min=1) - 1 if tree is not None else torch.zeros(b, 1, device="cuda")
        s["new_positions"] = (case["length"] + depth).to(torch.int32)
        if case["kind"] == "commit":
            s["lse"] = _plain_attend(s)[1]
    if own:
        from flash_evict.decode import KVCache
        s["cache"] = KVCache(k, v, **book)
        s["out_cache"] = KVCache(k, v, **s["out"])
    return s


# --------------------------------------------------------------------------- plain forms


def _plain_logits(s):
    """[B, Hkv, G*T, C] and [B, Hkv, G*T, T] scaled logits, -inf where a query does not look."""
    b, hk, c, d = s["k"].shape
    t = s["q"].shape[2]
    q = s["q"].float().reshape(b, hk, -1, d)
    old = (q @ s["k"].float().transpose(-1, -2)).mul_(s["scale"])
    old.masked_fill_((torch.arange(c, device="cuda") >= s["book"]["lengths"][..., None])[:, :, None], -math.inf)
    new = (q @ s["k_new"].float().transpose(-1, -2)) * s["scale"]
    if s["tree"] is not None:
        sees = s["tree"][:, None, None].expand(b, hk, new.shape[2] // t, t, s["k_new"].shape[2]).reshape(new.shape)
        new = new.masked_fill(~sees, -math.inf)
    return old, new


def _plain_attend(s):
    b, hq, t, d = s["q"].shape
    old, new = _plain_logits(s)
    top = torch.maximum(old.amax(-1), new.amax(-1))
    m = torch.where(torch.isinf(top), 0.0, top)[..., None]
    old, new = old.sub_(m).exp_(), (new - m).exp()
    total = old.sum(-1, keepdim=True) + new.sum(-1, keepdim=True)
    live = torch.arange(s["v"].shape[2], device="cuda") < s["book"]["lengths"][..., None]
    acc = old @ torch.where(live[..., None], s["v"].float(), 0.0) + new @ s["v_new"].float()
    out = torch.where(total > 0, acc / total, 0.0).view(b, hq, t, d).to(s["q"].dtype)
    return out, (m + total.log()).view(b, hq, t)


def _plain_commit(s):
    case, book, out = s["case"], s["book"], s["out"]
    b, hk, c, d = s["k"].shape
    hq, t = s["q"].shape[1:3]
    acc = s["accepted"].long()
    a = acc.shape[1]
    valid = acc >= 0
    count = valid.sum(-1)
    rank = torch.arange(a, device="cuda")
    weight = torch.where(valid, torch.exp(-case["decay"] * (count[:, None] - 1 - rank).float()), 0.0)
    at = acc.clamp(min=0)
    old, new = _plain_logits(dict(s, q=s["q"].gather(2, at[:, None, :, None].expand(b, hq, a, d)),
                                  tree=None if s["tree"] is None else s["tree"].gather(1, at[..., None].expand(b, a, t))) if t > 1 else s)
    lse = s["lse"].gather(2, at[:, None].expand(b, hq, a)).reshape(b, hk, -1, 1)
    w = weight[:, None].expand(b, hq, a).reshape(b, hk, -1, 1)
    old, new = old.sub_(lse).exp_().mul_(w).sum(2), ((new - lse).exp() * w).sum(2)
    lengths = book["lengths"].long()
    live = torch.arange(c, device="cuda") < lengths[..., None]
    faded = book["mass"] * torch.exp(-case["decay"] * count.float())[:, None, None]
    for name, value in (("mass", faded + book["norms"] * old), ("norms", book["norms"]), ("positions", book["positions"])):
        out[name].copy_(torch.where(live, value, out[name]))
    # the accepted rows go to the first free slots
    slot = lengths[..., None] + rank
    fits = valid[:, None] & (slot < c)
    slot = slot.clamp(max=c - 1)

    def put(into, rows):
        i = slot.view(slot.shape + (1,) * (into.dim() - 3)).expand(slot.shape + into.shape[3:])
        here = fits.view(fits.shape + (1,) * (into.dim() - 3))
        into.scatter_(2, i, torch.where(here, rows, into.gather(2, i)))

    rows = at[:, None].expand(b, hk, a)
    wide = rows[..., None].expand(b, hk, a, d)
    v_rows = s["v_new"].gather(2, wide)
    norm = v_rows.float().abs().sum(-1)
    put(s["k"], s["k_new"].gather(2, wide))
    put(s["v"], v_rows)
    put(out["norms"], norm)
    put(out["mass"], norm * new.gather(2, rows))
    put(out["positions"], s["new_positions"].gather(1, at)[:, None].expand(b, hk, a))
    out["lengths"].copy_((lengths + count[:, None]).clamp(max=c))
    return s["k"], s["v"], out["mass"], out["norms"], out["positions"], out["lengths"]


def _plain_evict(s):
    case, book, out = s["case"], s["book"], s["out"]
    budget, c = min(case["budget"], s["k"].shape[2]), s["k"].shape[2]
    slot = torch.arange(c, device="cuda").expand_as(book["mass"])
    lengths = book["lengths"][..., None]
    live = slot < lengths
    newest = torch.where(live, book["positions"], -1).amax(-1, keepdim=True)
    key = torch.where(book["positions"] > newest - case["recent"], math.inf, book["mass"])
    key = torch.where(live, key, -math.inf)
    rank = key.sort(dim=-1, descending=True, stable=True).indices.argsort(-1)
    keep = live & (rank < budget)
    # the i-th free slot below the budget takes the i-th kept token above it
    hole, mover = ~keep & (slot < budget) & (slot < lengths), keep & (slot >= budget)
    source = slot.clone()
    holes = torch.full((*slot.shape[:2], c + 1), c, device="cuda")
    holes.scatter_(2, torch.where(hole, hole.cumsum(-1) - 1, c), torch.where(hole, slot, c))
    target = torch.where(mover, holes.gather(2, (mover.cumsum(-1) - 1).clamp(min=0)), c)
    source = torch.cat([source, torch.zeros_like(source[..., :1])], -1).scatter_(2, target, slot)[..., :budget]
    wide = source[..., None].expand(*source.shape, s["k"].shape[3])
    for into in (s["k"], s["v"]):
        into[:, :, :budget] = into.gather(2, wide)
    left = live[..., :budget]
    for name in ("mass", "norms", "positions"):
        out[name][:, :, :budget] = torch.where(left, book[name].gather(2, source), out[name][:, :, :budget])
    out["lengths"].copy_(book["lengths"].clamp(max=budget))
    return s["k"], s["v"], out["mass"], out["norms"], out["positions"], out["lengths"]


# --------------------------------------------------------------------------- a pass


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        return {"attend": _plain_attend, "commit": _plain_commit, "evict": _plain_evict}[kind](s)
    from flash_evict import decode
    if kind == "attend":
        return decode.tree_attention(s["q"], s["k_new"], s["v_new"], s["cache"], tree=s["tree"], scale=s["scale"])
    if kind == "commit":
        o = decode.commit_tokens(s["cache"], s["q"], s["k_new"], s["v_new"], s["lse"], s["accepted"], s["new_positions"], tree=s["tree"],
                                 scale=s["scale"], recency_decay=s["case"]["decay"], out=s["out_cache"])
    else:
        o = decode.evict_tokens(s["cache"], s["case"]["budget"], recent=s["case"]["recent"], out=s["out_cache"])
    return o.k, o.v, o.mass, o.norms, o.positions, o.lengths


def work(case):
    b, hq, hk, d, t = (case[n] for n in ("batch", "q_heads", "kv_heads", "channels", "drafts"))
    g = hq // hk
    rows = _lengths(case)
    tokens = sum(rows)
    if case["kind"] == "attend":
        # K and V once, the drafts' q, k, v, the mask, out and the row sums; QK^T and PV
        extra = 2 * b * t * d * (2 * hq + 2 * hk) + 4 * b * hq * t + (b * t * t if t > 1 else 0) + 4 * b * hk
        return {"bytes": 4 * tokens * d + extra, "flops": 4 * g * t * d * tokens + 4 * b * hq * t * t * d}
    if case["kind"] == "commit":
        # K once, the bookkeeping read and written; QK^T of the accepted rows
        took = _accepts(case)
        per = sum(rows) / b  # tokens of a sequence over its heads, on average
        moved = sum(took)
        extra = 2 * moved * d * (hq + 4 * hk) + 4 * moved * (hq + 4 * hk) + 24 * tokens + 8 * b * hk
        return {"bytes": 2 * tokens * d + extra, "flops": 2 * g * d * per * moved + 2 * hq * d * sum(n * n for n in took)}
    # the weights and positions of every token, the kept bookkeeping written; at most budget tokens of a row move
    budget = case["budget"]
    kept = sum(min(n, budget) for n in rows)
    # rows that move: a kept token above the budget takes a free slot below it; of n tokens, budget kept at random places
    moves = sum(budget * (n - budget) / n for n in rows if n > budget)
    return {"bytes": 8 * tokens + 4 * kept + 12 * kept + 8 * moves * d + 8 * b * hk, "flops": 8 * tokens}


# --------------------------------------------------------------------------- exact results


def exact(case, seed):
    s = prepare(case, seed)
    kind, dev = case["kind"], "cuda"
    b, hk, c, d = s["k"].shape
    lengths = s["book"]["lengths"].tolist()
    if kind == "evict":
        return _exact_evict(s, lengths)
    hq, t = s["q"].shape[1:3]
    g = hq // hk
    sees = s["tree"] if s["tree"] is not None else torch.ones(b, t, t, dtype=torch.bool, device=dev)
    if kind == "attend":
        out = torch.zeros(b, hq, t, d, dtype=torch.float64, device=dev)
        lse = torch.full((b, hq, t), -math.inf, dtype=torch.float64, device=dev)
        for i in range(b):
            for h in range(hk):
                n = lengths[i][h]
                keys = torch.cat([s["k"][i, h, :n], s["k_new"][i, h]]).double()
                values = torch.cat([s["v"][i, h, :n], s["v_new"][i, h]]).double()
                may = torch.cat([torch.ones(t, n, dtype=torch.bool, device=dev), sees[i]], 1)
                for j in range(h * g, h * g + g):
                    x = torch.where(may, s["scale"] * (s["q"][i, j].double() @ keys.T), -math.inf)
                    lse[i, j] = torch.logsumexp(x, 1)
                    p = torch.exp(x - torch.where(lse[i, j] == -math.inf, 0.0, lse[i, j])[:, None])
                    out[i, j] = p @ values
        return out, lse
    mass, norms = s["out"]["mass"].double(), s["out"]["norms"].double()
    for i in range(b):
        path = [j for j in s["accepted"][i].tolist() if j >= 0]
        fade = [math.exp(-case["decay"] * (len(path) - 1 - r)) for r in range(len(path))]
        w = torch.tensor(fade, dtype=torch.float64, device=dev)[:, None]
        for h in range(hk):
            n = lengths[i][h]
            keys = torch.cat([s["k"][i, h, :n], s["k_new"][i, h, path]]).double()
            size = torch.cat([s["book"]["norms"][i, h, :n].double(), s["v_new"][i, h, path].double().abs().sum(-1)])
            may = torch.cat([torch.ones(len(path), n, dtype=torch.bool, device=dev), sees[i][path][:, path]], 1)
            got = torch.zeros(n + len(path), dtype=torch.float64, device=dev)
            for j in range(h * g, h * g + g):
                x = s["scale"] * (s["q"][i, j, path].double() @ keys.T) - s["lse"][i, j, path].double()[:, None]
                got += (torch.where(may, torch.exp(x), 0.0) * w).sum(0)
            got *= size
            got[:n] += s["book"]["mass"][i, h, :n].double() * math.exp(-case["decay"] * len(path))
            mass[i, h, :n + len(path)] = got
            norms[i, h, :n + len(path)] = size
    return None, None, mass, norms, None, None


def _exact_evict(s, lengths):
    """The kept tokens one by one: a host-side walk over each row's sorted weights."""
    case, book, out = s["case"], s["book"], s["out"]
    b, hk, c, _ = s["k"].shape
    budget = case["budget"]
    mass, norms = out["mass"].double().cpu(), out["norms"].double().cpu()
    all_mass, all_norms, all_pos = book["mass"].double().cpu(), book["norms"].double().cpu(), book["positions"].cpu()
    for i in range(b):
        for h in range(hk):
            n = lengths[i][h]
            if n == 0:
                continue
            m, z, pos = all_mass[i, h, :n], all_norms[i, h, :n], all_pos[i, h, :n]
            place = list(range(min(n, budget)))
            if n > budget:
                bar = int(pos.max()) - case["recent"]
                weights, ages = m.tolist(), pos.tolist()
                order = sorted(range(n), key=lambda j: (ages[j] <= bar, 0.0 if ages[j] > bar else -weights[j], j))
                kept = set(order[:budget])
                late = iter(sorted(j for j in kept if j >= budget))
                place = [j if j in kept else next(late) for j in range(budget)]
            mass[i, h, :len(place)] = m[place]
            norms[i, h, :len(place)] = z[place]
    return None, None, mass, norms, None, None
