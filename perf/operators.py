"""Serving a long context from the int8 cache: attention over a window with pinned first tokens, attention of a batch
that shares a prefix, attention that records what every slot received, and eviction by that record.

Each case is a dict of plain values. Kinds:

- ``window``   `KVCache.attention_window`: `count` new tokens per sequence are stored in the sequence's ring of slots
               and attend the first `sinks` positions and the last `window` ones (a decode step, a draft to verify, a
               prompt piece);
- ``shared``   `KVCache.attention_shared`: one decode step of sequences that share a prefix kept once;
- ``weights``  `KVCache.attention_weights`: one decode step that adds every slot's attention weight to a record;
- ``evict``    `KVCache.evict`: the cache cut to `keep` slots per sequence and kv head by that record.

The cache holds int8 codes with one fp32 scale per row (row x: top = max|x|, scale = top / 127, code = round(x * (127 /
top)), both quotients rounded to 32 bits). Where `own` is true a state holds the framework's cache, else the same
codes and scales as tensors; everything else in a state is the same on both sides.
"""
import math

import torch

own = False


# ---- the cases --------------------------------------------------------------------------------------------------
def listed():
    return [
        # one conversation, one token: the smallest call, at the released geometry (8 heads, 4 kv heads of 64, window 256)
        dict(name="window_step_1", kind="window", seqs=1, kvheads=4, per_kv=2, head_dim=64, count=1, sinks=16, window=256),
        # a full serving batch, one token each, long windows, grouped queries
        dict(name="window_step_64", kind="window", seqs=64, kvheads=8, per_kv=4, head_dim=128, count=1, sinks=4,
             window=4096),
        # five drafted tokens per sequence to verify; three query heads per kv head, odd everything
        dict(name="window_draft_7x5", kind="window", seqs=7, kvheads=5, per_kv=3, head_dim=32, count=5, sinks=3,
             window=999),
        # a prompt piece of one conversation at the released geometry: longer than its window
        dict(name="window_prompt_512", kind="window", seqs=1, kvheads=4, per_kv=2, head_dim=64, count=512, sinks=16,
             window=256),
        # odd-length prompt pieces of several conversations, grouped queries of 128
        dict(name="window_prompt_6x999", kind="window", seqs=6, kvheads=8, per_kv=4, head_dim=128, count=999, sinks=4,
             window=2048),
        # four conversations behind one short system prompt
        dict(name="shared_4", kind="shared", seqs=4, kvheads=4, per_kv=2, head_dim=64, prefix=700, length=60),
        # a full serving batch behind a long common document, each a few hundred tokens into its own answer
        dict(name="shared_64", kind="shared", seqs=64, kvheads=8, per_kv=4, head_dim=128, prefix=8192, length=512),
        # an odd batch over a very long prefix, few kv heads
        dict(name="shared_33_long", kind="shared", seqs=33, kvheads=2, per_kv=8, head_dim=64, prefix=65537, length=129),
        # one conversation whose slots' weights are recorded
        dict(name="weights_1", kind="weights", seqs=1, kvheads=4, per_kv=2, head_dim=64, length=700),
        # sequences of different ages, recorded, long caches
        dict(name="weights_16", kind="weights", seqs=16, kvheads=8, per_kv=4, head_dim=128, length=8192),
        # two conversations cut to half
        dict(name="evict_2", kind="evict", seqs=2, kvheads=4, head_dim=64, length=2048, keep=1024, sinks=4, recent=128),
        # a serving batch of different ages cut to an odd budget
        dict(name="evict_32", kind="evict", seqs=32, kvheads=8, head_dim=128, length=8192, keep=4001, sinks=4, recent=512),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]; odd and even alike."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["window", "window", "shared", "weights", "evict"])
    c = dict(kind=kind, kvheads=rng.choice([1, 2, 3, 4, 8]), head_dim=rng.choice([32, 64, 128]))
    c["per_kv"] = rng.choice([1, 2, 3, 4, 6, 8]) if kind != "evict" else 1
    width = c["kvheads"] * c["head_dim"]  # bytes of a slot's K codes
    if kind == "window":
        c["count"] = 1 if rng.random() < 0.4 else _log(rng, 2, 8) if rng.random() < 0.4 else _log(rng, 9, 1024)
        c["sinks"], c["window"] = rng.choice([0, 1, 4, 17, 64]), _log(rng, 16, 8192)
        most = 64 * 8 * 128 * 4096 // (width * (c["window"] + c["count"]))
        if c["count"] > 8:  # no more queries and products than the largest listed case
            queries = c["count"] * width * c["per_kv"]
            most = min(most, 6 * 999 * 8 * 4 * 128 // queries, 6 * 999 * 8 * 4 * 128 * 2048 // (queries * (c["window"] + 64)))
        return dict(c, seqs=_log(rng, 1, max(1, min(64, most))))
    if kind == "shared":
        c["prefix"], c["length"] = _log(rng, 16, 65536), _log(rng, 1, 2048)
        most = 64 * 8 * 4 * 128 * 8192 // (width * c["per_kv"] * c["prefix"])
        return dict(c, seqs=_log(rng, 1, max(1, min(64, most))))
    if kind == "weights":
        c["length"] = _log(rng, 16, 16384)
        return dict(c, seqs=_log(rng, 1, max(1, min(64, 16 * 8 * 128 * 8192 // (width * c["length"])))))
    c["length"] = _log(rng, 64, 16384)
    c["keep"] = max(24, int(c["length"] * rng.uniform(0.2, 0.9)))
    c["sinks"], c["recent"] = rng.choice([0, 1, 4, 8]), _log(rng, 1, c["keep"] // 2)
    return dict(c, seqs=_log(rng, 1, max(1, min(64, 32 * 8 * 128 * 8192 // (width * c["length"])))))


# ---- inputs -----------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _whole(gen, lo, hi, *shape):
    """int32 values in [lo, hi]."""
    return torch.randint(lo, hi + 1, shape, generator=gen, device="cuda", dtype=torch.int32)


def _slots(c):
    """Slots per sequence of the case's cache."""
    return c["sinks"] + c["window"] + c["count"] - 1 if c["kind"] == "window" else c["length"]


def _quantised(rows):
    """(codes, scales) of fp32 rows."""
    top = rows.abs().amax(-1, keepdim=True)
    live = top > 0
    inv = torch.where(live, (127.0 / top.double()).float(), torch.zeros_like(top))
    scale = torch.where(live, (top.double() / 127.0).float(), torch.ones_like(top))
    return torch.round(rows * inv).clamp(-127, 127).to(torch.int8), scale[..., 0]


def _cache(k, v):
    """The cache of fp32 rows [seqs, slots, kvheads, head_dim]: the framework's, or a dict of tensors in its layout
    [seqs, kvheads, slots, head_dim]."""
    if own:
        from openneedle_amd.kv import KVCache
        n, slots, kvheads, hd = k.shape
        kv = KVCache(1, slots, kvheads, hd, n)
        kv.store(0, k.data_ptr(), v.data_ptr(), slots, stream=_stream())
        torch.cuda.synchronize()  # k and v are freed
        return kv
    (k8, ks), (v8, vs) = _quantised(k), _quantised(v)
    return dict(k=k8.transpose(1, 2).contiguous(), v=v8.transpose(1, 2).contiguous(),
                ks=ks.transpose(1, 2).contiguous(), vs=vs.transpose(1, 2).contiguous())


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _inputs(c, seed):
    """Everything but the cache's handle, from the seed alone; `rows`: the fp32 rows that the cache is made of."""
    g = _gen(seed)
    n, kvheads, hd = c["seqs"], c["kvheads"], c["head_dim"]
    s = dict(rows=tuple(_normal(g, n, _slots(c), kvheads, hd) for _ in "kv"))
    if c["kind"] == "evict":
        # accumulated weights: heavy-tailed, some slots never attended (exact zeros), the first tokens far ahead
        w = torch.exp(2 * _normal(g, n, kvheads, c["length"]) - 6)
        w = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.05, torch.zeros_like(w), w)
        w[..., :4] += 20.0
        low = max(1, c["length"] // 2)
        return dict(s, weights=w, lengths=_whole(g, low, c["length"], n))
    count = c.get("count", 1)
    s["q"] = _normal(g, n, count, kvheads * c["per_kv"], hd)
    s["new"] = tuple(_normal(g, n, count, kvheads, hd) for _ in "kv")
    if c["kind"] == "window":  # from sequences younger than their window to ones that went round the ring
        s["positions"] = _whole(g, c["window"] // 2, 8 * c["window"] + c["sinks"], n)
        return s
    s["lengths"] = _whole(g, max(1, c["length"] // 4), c["length"], n)
    if c["kind"] == "shared":
        s["prefix_rows"] = tuple(_normal(g, 1, c["prefix"], kvheads, hd) for _ in "kv")
    else:
        s["weights"] = torch.rand((n, kvheads, c["length"]), generator=g, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], s["kv"] = case, _cache(*s.pop("rows"))
    if case["kind"] == "shared":
        s["prefix"] = _cache(*s.pop("prefix_rows"))
    if case["kind"] == "evict":
        s["kept"] = torch.empty((case["seqs"], case["kvheads"], case["keep"]), dtype=torch.int32, device="cuda")
        s["new_weights"] = torch.empty_like(s["weights"])
        s["new_lengths"] = torch.empty_like(s["lengths"])
    else:
        s["out"] = torch.empty_like(s["q"])
    if own:
        s["rows"] = _rows_of(s["kv"])
    torch.cuda.synchronize()
    return s


class _Address:
    """Device memory as torch takes it; the tensor keeps this object, which keeps the cache."""

    def __init__(self, at, kind, shape):
        self.at = at
        self.__cuda_array_interface__ = dict(data=(at.ptr, False), typestr=kind, shape=shape, version=2)


def _rows_of(kv):
    """The framework cache's codes and scales as tensors over its own memory."""
    shape = (kv.seqs, kv.kvheads, kv.capacity)
    k, v, ks, vs = kv.device_rows(0)
    codes, scales = ((t, "|i1", shape + (kv.head_dim,)) for t in (k, v)), ((t, "<f4", shape) for t in (ks, vs))
    return dict(zip(("k", "v", "ks", "vs"), (torch.as_tensor(_Address(*a), device="cuda") for a in (*codes, *scales))))


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else PLAIN[state["case"]["kind"]](state)


def _run_own(st):
    c, kv, s = st["case"], st["kv"], _stream()
    if c["kind"] == "evict":
        kv.evict(0, st["weights"].data_ptr(), st["lengths"].data_ptr(), c["keep"], c["sinks"], c["recent"],
                 st["new_weights"].data_ptr(), st["new_lengths"].data_ptr(), st["kept"].data_ptr(), stream=s)
        return dict(weights=st["new_weights"], lengths=st["new_lengths"], kept=st["kept"], **st["rows"])
    q, out, heads = st["q"].data_ptr(), st["out"].data_ptr(), c["kvheads"] * c["per_kv"]
    new = tuple(t.data_ptr() for t in st["new"])
    if c["kind"] == "window":
        kv.attention_window(0, q, out, heads, c["count"], st["positions"].data_ptr(), c["sinks"], c["window"], stream=s,
                            new=new)
        return dict(out=st["out"], **st["rows"])
    if c["kind"] == "shared":
        kv.attention_shared(0, st["prefix"], c["prefix"], q, out, heads, c["length"], st["lengths"].data_ptr(), stream=s,
                            new=new)
        return dict(out=st["out"], **st["rows"])
    kv.attention_weights(0, q, out, st["weights"].data_ptr(), heads, c["length"], st["lengths"].data_ptr(), stream=s,
                         new=new)
    return dict(out=st["out"], weights=st["weights"], **st["rows"])


def _store(kv, new, slots):
    """New rows [seqs, count, kvheads, head_dim] into slots [seqs, count] of a cache of tensors."""
    at = torch.arange(slots.shape[0], device="cuda")[:, None]
    for name, rows in zip("kv", new):
        codes, scales = _quantised(rows)
        kv[name][at, :, slots] = codes
        kv[name + "s"][at, :, slots] = scales


def _values(codes, scales):
    return codes.float() * scales[..., None]


def _window(st):
    c, kv = st["case"], st["kv"]
    n, count, kvheads, group, hd = c["seqs"], c["count"], c["kvheads"], c["per_kv"], c["head_dim"]
    sinks, window = c["sinks"], c["window"]
    ring = _slots(c) - sinks
    first = st["positions"].long()[:, None]
    mine = first + torch.arange(count, device="cuda")  # [n, count] positions of the new tokens

    def slot(p):
        return torch.where(p < sinks, p.clamp(min=0), sinks + (p - sinks) % ring)

    _store(kv, st["new"], slot(mine))
    pinned = torch.arange(sinks, device="cuda").expand(n, sinks)
    recent = first - window + 1 + torch.arange(window + count - 1, device="cuda")
    seen = torch.cat((pinned, recent), 1)  # positions of the keys; those of `recent` below `sinks` are there already
    live = torch.cat((torch.ones_like(pinned, dtype=torch.bool), recent >= sinks), 1)
    pinned_key = torch.arange(seen.shape[1], device="cuda") < sinks
    allowed = live[:, None] & (seen[:, None] <= mine[..., None]) & (pinned_key | (seen[:, None] > mine[..., None] - window))
    at, seq = slot(seen), torch.arange(n, device="cuda")[:, None]
    k = _values(kv["k"][seq, :, at], kv["ks"][seq, :, at]).transpose(1, 2).reshape(n * kvheads, -1, hd)
    v = _values(kv["v"][seq, :, at], kv["vs"][seq, :, at]).transpose(1, 2).reshape(n * kvheads, -1, hd)
    q = st["q"].reshape(n, count, kvheads, group, hd).transpose(1, 2).reshape(n * kvheads, count * group, hd)
    score = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(hd)
    score = score.reshape(n, kvheads, count, group, -1).masked_fill_(~allowed[:, None, :, None], -math.inf)
    score = torch.exp(score - score.amax(-1, keepdim=True))
    score = (score / score.sum(-1, keepdim=True)).reshape(n * kvheads, count * group, -1)
    out = torch.bmm(score, v).reshape(n, kvheads, count, group, hd).transpose(1, 2).reshape(st["q"].shape)
    return dict(out=out, **kv)


def _shared(st):
    c, kv, prefix = st["case"], st["kv"], st["prefix"]
    n, kvheads, group, hd, length = c["seqs"], c["kvheads"], c["per_kv"], c["head_dim"], c["length"]
    lengths = st["lengths"].long()
    _store(kv, st["new"], lengths[:, None] - 1)
    q = st["q"].reshape(n, kvheads, group, hd)
    common = q.transpose(0, 1).reshape(kvheads, n * group, hd)
    pk, pv = (_values(prefix[a][0], prefix[a + "s"][0]) for a in "kv")
    k, v = (_values(kv[a], kv[a + "s"]).reshape(n * kvheads, length, hd) for a in "kv")
    far = torch.bmm(common, pk.transpose(1, 2).contiguous()).reshape(kvheads, n, group, -1).transpose(0, 1)
    near = torch.bmm(q.reshape(n * kvheads, group, hd), k.transpose(1, 2).contiguous()).reshape(n, kvheads, group, length)
    past = torch.arange(length, device="cuda") >= lengths[:, None]
    near = near.masked_fill(past[:, None, None], -math.inf)
    score = torch.cat((far, near), -1) / math.sqrt(hd)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    far, near = p[..., :c["prefix"]], p[..., c["prefix"]:]
    out = torch.bmm(far.transpose(0, 1).reshape(kvheads, n * group, -1), pv).reshape(kvheads, n, group, hd).transpose(0, 1)
    out = out + torch.bmm(near.reshape(n * kvheads, group, length), v).reshape(n, kvheads, group, hd)
    return dict(out=out.reshape(st["q"].shape), **kv)


def _weights(st):
    c, kv = st["case"], st["kv"]
    n, kvheads, group, hd, length = c["seqs"], c["kvheads"], c["per_kv"], c["head_dim"], c["length"]
    lengths = st["lengths"].long()
    _store(kv, st["new"], lengths[:, None] - 1)
    k, v = (_values(kv[a], kv[a + "s"]).reshape(n * kvheads, length, hd) for a in "kv")
    q = st["q"].reshape(n * kvheads, group, hd)
    score = (torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(hd)).reshape(n, kvheads, group, length)
    past = torch.arange(length, device="cuda") >= lengths[:, None]
    score = score.masked_fill(past[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    st["weights"] += p.sum(2)
    out = torch.bmm(p.reshape(n * kvheads, group, length), v).reshape(st["q"].shape)
    return dict(out=out, weights=st["weights"], **kv)


def _evict(st):
    c, kv = st["case"], st["kv"]
    keep, length = c["keep"], c["length"]
    n = st["lengths"].long()[:, None, None]
    left = n.clamp(max=keep)
    slot = torch.arange(length, device="cuda")
    always = (slot < c["sinks"]) | (slot >= n - c["recent"]) | (n <= keep)
    rank = torch.where(always, torch.full_like(st["weights"], math.inf), st["weights"])
    rank = torch.where(slot < n, rank, torch.full_like(rank, -math.inf))
    order = torch.sort(rank, dim=-1, descending=True, stable=True)[1]  # of equal weights the lower slot goes first
    kept = torch.sort(order[..., :keep], dim=-1)[0]
    live = torch.arange(keep, device="cuda") < left
    weights = torch.zeros_like(st["weights"])
    weights[..., :keep] = torch.where(live, st["weights"].gather(-1, kept), torch.zeros_like(st["weights"][..., :keep]))
    for name in ("k", "v"):
        rows = kv[name].gather(2, kept[..., None].expand(-1, -1, -1, c["head_dim"]))
        kv[name][:, :, :keep] = torch.where(live[..., None], rows, kv[name][:, :, :keep])
        scales = kv[name + "s"].gather(2, kept)
        kv[name + "s"][:, :, :keep] = torch.where(live, scales, kv[name + "s"][:, :, :keep])
    kept = torch.where(live, kept, torch.full_like(kept, -1)).int()
    return dict(weights=weights, lengths=left[:, 0, 0].int(), kept=kept, **kv)


PLAIN = dict(window=_window, shared=_shared, weights=_weights, evict=_evict)


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    c = case
    n, kvheads, hd = c["seqs"], c["kvheads"], c["head_dim"]
    row = 2 * (hd + 4)  # bytes of a slot and kv head, K and V
    if c["kind"] == "evict":
        mean = 0.75 * c["length"]  # the mean of the lengths drawn between a half and the whole
        left = min(c["keep"], mean)
        return dict(bytes=n * kvheads * (2 * left * row + 8 * mean + 4 * c["keep"]), flops=0.0)
    heads, count = kvheads * c["per_kv"], c.get("count", 1)
    io = 4.0 * n * count * hd * (2 * heads + 2 * kvheads) + n * count * kvheads * row
    if c["kind"] == "window":
        seen = c["sinks"] + c["window"]
        return dict(bytes=io + n * kvheads * row * (seen + count - 1), flops=4.0 * n * count * heads * hd * seen)
    mean = 0.625 * c["length"]  # of the lengths drawn between a quarter and the whole
    if c["kind"] == "shared":
        return dict(bytes=io + kvheads * row * (c["prefix"] + n * mean), flops=4.0 * n * heads * hd * (c["prefix"] + mean))
    return dict(bytes=io + n * kvheads * mean * (row + 8), flops=4.0 * n * heads * hd * mean)


# ---- the same in 64 bits, one sequence and kv head at a time ----------------------------------------------------------
def _cached(rows):
    """Cache rows as values in 64 bits. The quantiser is defined in 32 bits, so its codes are made there."""
    codes, scales = _quantised(rows)
    return codes.double() * scales.double()[..., None]


def _softmax_rows(q, k, hidden=None):
    s = torch.matmul(q, k.T.contiguous()) / math.sqrt(q.shape[-1])
    return torch.softmax(s if hidden is None else s.masked_fill(hidden, -math.inf), -1)


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    n, kvheads, hd = c["seqs"], c["kvheads"], c["head_dim"]
    if c["kind"] == "evict":
        weights = torch.zeros_like(s["weights"], dtype=torch.float64)
        for i, length in enumerate(s["lengths"].tolist()):
            for h in range(kvheads):
                w = s["weights"][i, h, :length].tolist()
                middle = sorted(range(c["sinks"], length - c["recent"]), key=lambda j: (-w[j], j))
                cut = middle[max(0, c["keep"] - c["sinks"] - c["recent"]):] if length > c["keep"] else []
                kept = sorted(set(range(length)) - set(cut))
                weights[i, h, :len(kept)] = torch.tensor([w[j] for j in kept], device="cuda").double()
        return dict(weights=weights, lengths=None, kept=None, k=None, v=None, ks=None, vs=None)
    group, count = c["per_kv"], c.get("count", 1)
    k, v = (_cached(r) for r in s["rows"])
    nk, nv = (_cached(r) for r in s["new"])
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if c["kind"] == "weights" else None
    if c["kind"] == "shared":
        pk, pv = (_cached(r)[0] for r in s["prefix_rows"])
    for i in range(n):
        hidden = None
        if c["kind"] == "window":
            first, ring = int(s["positions"][i]), _slots(c) - c["sinks"]
            mine = torch.arange(first, first + count, device="cuda")
            low = max(c["sinks"], first - c["window"] + 1)
            seen = torch.cat((torch.arange(c["sinks"], device="cuda"), torch.arange(low, first + count, device="cuda")))
            at = torch.where(seen < c["sinks"], seen, c["sinks"] + (seen - c["sinks"]) % ring)
            put = torch.where(mine < c["sinks"], mine, c["sinks"] + (mine - c["sinks"]) % ring)
            k[i, put], v[i, put] = nk[i], nv[i]
            back = mine[:, None] - seen[None]
            hidden = ((back < 0) | ((back >= c["window"]) & (seen >= c["sinks"]))).repeat_interleave(group, 0)
            ki, vi = k[i, at], v[i, at]
        else:
            length = int(s["lengths"][i])
            k[i, length - 1], v[i, length - 1] = nk[i, 0], nv[i, 0]
            ki, vi = k[i, :length], v[i, :length]
            if c["kind"] == "shared":
                ki, vi = torch.cat((pk, ki)), torch.cat((pv, vi))
        for h in range(kvheads):
            q = s["q"][i, :, h * group:(h + 1) * group].reshape(count * group, hd).double()
            p = _softmax_rows(q, ki[:, h], hidden)
            out[i, :, h * group:(h + 1) * group] = torch.matmul(p, vi[:, h].contiguous()).reshape(count, group, hd)
            if weights is not None:
                weights[i, h, :p.shape[1]] += p.sum(0)
    rest = dict(k=None, v=None, ks=None, vs=None)
    return dict(out=out, weights=weights, **rest) if weights is not None else dict(out=out, **rest)
