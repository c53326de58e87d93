"""Serving many requests from one paged int8 cache: tables and slots built on the GPU, heads normed and rotated, rows
stored by slot, and attention of ragged new tokens over the pages.

Each case is a dict of plain values. Kinds:

- ``tables``     `PagedCache.extend`, then `PagedCache.trim`: requests of different lengths get pages for their new tokens,
                 a slot and a position for every token, and the tokens are taken back (a step whose tokens were not kept);
- ``heads``      `rotate_heads`: every head of q and k normed over its own values, times 1 + gain, its first `rotary`
                 dimensions rotated by the token's position (dimension j with j + rotary / 2);
- ``store``      `PagedCache.store`: the K and V rows of a ragged batch of tokens into their slots;
- ``attention``  `PagedCache.attention`: the new tokens of every request (one, a draft or a prompt piece) over what the
                 request has in the cache up to the token itself, or the last `window` positions of that.

A page holds `page` positions of every kv head: int8 codes with one fp32 scale per row (row x: top = max|x|, scale =
top / 127, code = round(x * (127 / top)), both quotients rounded to 32 bits). Slot s is position s % page of page
s / page. Where `own` is true a state holds the framework's cache, else the same codes and scales as tensors
[pages, kvheads, page, ...]; everything else in a state is the same on both sides.
"""
import math
import random

import torch

own = False


# ---- the cases --------------------------------------------------------------------------------------------------
def listed():
    return [
        # a small decode batch, one new token each: the smallest step of a serving loop
        dict(name="tables_decode_32", kind="tables", decode=32, pieces=0, chunk=0, context=4096, page=16),
        # a large batch of long requests, most of them decoding, prompt pieces among them
        dict(name="tables_mixed_500", kind="tables", decode=480, pieces=20, chunk=1024, context=8192, page=16),
        # one token at the released geometry (8 heads, 4 kv heads of 64)
        dict(name="heads_1", kind="heads", tokens=1, heads=8, kvheads=4, head_dim=64, rotary=64, fused=False),
        # an odd batch, narrow heads rotated in part, q and k in the rows of one projection
        dict(name="heads_333_odd", kind="heads", tokens=333, heads=15, kvheads=5, head_dim=32, rotary=20, fused=True),
        # the prompt pieces of a step, grouped queries of 128
        dict(name="heads_8191", kind="heads", tokens=8191, heads=32, kvheads=8, head_dim=128, rotary=128, fused=True),
        # a decode batch
        dict(name="store_64", kind="store", tokens=64, kvheads=8, head_dim=128, page=16),
        # the prompt pieces of a step, some tokens without a slot
        dict(name="store_8191", kind="store", tokens=8191, kvheads=8, head_dim=128, page=16),
        # one conversation, one token, at the released geometry: the smallest call
        dict(name="attention_decode_1", kind="attention", decode=1, pieces=0, chunk=0, context=700, window=0, kvheads=4,
             per_kv=2, head_dim=64, page=16),
        # a full serving batch of different ages, one token each, grouped queries
        dict(name="attention_decode_64", kind="attention", decode=64, pieces=0, chunk=0, context=8192, window=0, kvheads=8,
             per_kv=4, head_dim=128, page=16),
        # drafts of up to five tokens to verify over a window; three query heads per kv head, odd everything
        dict(name="attention_draft_7", kind="attention", decode=0, pieces=7, chunk=5, context=999, window=501, kvheads=5,
             per_kv=3, head_dim=32, page=32),
        # decoding requests and prompt pieces of others in one call
        dict(name="attention_mixed_51", kind="attention", decode=48, pieces=3, chunk=1024, context=4096, window=0,
             kvheads=8, per_kv=4, head_dim=128, page=64),
        # a prompt piece far into one long document
        dict(name="attention_prompt", kind="attention", decode=0, pieces=1, chunk=2000, context=16000, window=0, kvheads=8,
             per_kv=4, head_dim=128, page=16),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]; odd and even alike."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "heads", "store", "attention", "attention", "attention"])
    hd, kvheads, per_kv = rng.choice([32, 64, 128]), rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 6, 8])
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "tables":
        return dict(kind=kind, decode=_log(rng, 1, 500), pieces=rng.choice([0, 1, 3, 10, 20]), chunk=_log(rng, 2, 1024),
                    context=_log(rng, 16, 8192), page=page)
    if kind == "heads":
        heads = min(32, kvheads * per_kv)
        most = 8191 * 40 * 128 // ((heads + kvheads) * hd)
        return dict(kind=kind, tokens=_log(rng, 1, min(8191, most)), heads=heads, kvheads=kvheads, head_dim=hd,
                    rotary=rng.choice([hd, hd, hd // 2, hd - 12]), fused=rng.random() < 0.5)
    if kind == "store":
        return dict(kind=kind, tokens=_log(rng, 1, 8191), kvheads=kvheads, head_dim=hd, page=page)
    form = rng.choice(["decode", "draft", "prompt", "mixed"])
    c = dict(kind=kind, decode=0, pieces=0, chunk=0, context=_log(rng, 16, 16000),
             window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), kvheads=kvheads, per_kv=per_kv, head_dim=hd, page=page)
    width = kvheads * hd
    if form in ("decode", "mixed"):
        c["decode"] = _log(rng, 1, max(1, min(64 if form == "decode" else 48, 64 * 8 * 128 * 8192 // (width * c["context"]))))
    if form == "draft":
        c["chunk"] = rng.randint(2, 8)
        c["pieces"] = _log(rng, 1, max(1, min(64, 16 * 8 * 128 * 8192 // (width * c["context"]))))
    if form in ("prompt", "mixed"):
        # no more products than half the largest listed case
        most = 1000 * 8 * 4 * 128 * 8000 // (width * per_kv * (c["context"] + 512))
        c["chunk"] = _log(rng, 9, max(9, min(2000, most)))
        c["pieces"] = rng.randint(1, max(1, min(4, most // c["chunk"])))
    return c


def _requests(c):
    """(new tokens, positions in the cache) of every request of a case, pieces and decoding ones in no order."""
    rng = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    counts = [1] * c["decode"] + [rng.randint((c["chunk"] + 1) // 2, c["chunk"]) for _ in range(c["pieces"])]
    rng.shuffle(counts)
    return counts, [rng.randint(c["context"] // 4, c["context"]) for _ in counts]


# ---- inputs -----------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _places(gen, counts, page, spare):
    """Every request's table (int32 [requests, width], -1 past its pages) over pages in no order, and the number of pages."""
    need = [(n + page - 1) // page for n in counts]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    width = max(need) + 1
    start = torch.tensor([0] + need, device="cuda").cumsum(0)
    j = torch.arange(width, device="cuda")
    at = start[:-1, None] + j
    return torch.where(j < torch.tensor(need, device="cuda")[:, None], order[at.clamp(max=pages - 1)], -1).int(), pages


def _slots(tables, positions, page):
    """Slots int32 of positions [requests, n]."""
    return (tables.gather(1, (positions // page).long()) * page + positions % page).int()


def _inputs(c, seed):
    """Everything but the cache's handle, from the seed alone."""
    g = _gen(seed)
    if c["kind"] == "heads":
        n, hd, heads, kvheads = c["tokens"], c["head_dim"], c["heads"], c["kvheads"]
        if c["fused"]:  # rows of one projection: q, k and v of a token side by side
            rows = _normal(g, n, (heads + 2 * kvheads) * hd)
            q, k = rows[:, :heads * hd], rows[:, heads * hd:(heads + kvheads) * hd]
        else:
            q, k = _normal(g, n, heads * hd), _normal(g, n, kvheads * hd)
        half = c["rotary"] // 2
        freq = 500000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        return dict(q=q, k=k, q_gain=0.2 * _normal(g, hd), k_gain=0.2 * _normal(g, hd), freq=freq,
                    # positions of requests far into their contexts
                    positions=torch.randint(0, 131072, (n,), generator=g, device="cuda", dtype=torch.int32))
    if c["kind"] == "store":
        n = c["tokens"]
        pages = (n + c["page"] - 1) // c["page"] * 2
        slots = torch.randperm(pages * c["page"], generator=g, device="cuda")[:n].int()
        slots = torch.where(torch.rand(n, generator=g, device="cuda") < 0.02, -1, slots)  # padded tokens
        return dict(k=_normal(g, n, c["kvheads"], c["head_dim"]), v=_normal(g, n, c["kvheads"], c["head_dim"]),
                    slots=slots, pages=pages)
    counts, past = _requests(c)
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    s = dict(counts=_ints(counts), tokens=starts[-1])
    if c["kind"] == "tables":  # requests of any age
        s["past"], s["mix"] = (torch.randint(lo, hi + 1, (len(counts),), generator=g, device="cuda", dtype=torch.int32)
                               for lo, hi in ((c["context"] // 4, c["context"]), (0, 64)))
        most = [(c["context"] + n + c["page"] - 1) // c["page"] for n in counts]
        return dict(s, width=max(most), pages=sum(most))
    total = [a + b for a, b in zip(counts, past)]
    s["past"], s["starts"] = _ints(past), _ints(starts)
    kvheads, hd = c["kvheads"], c["head_dim"]
    s["tables"], s["pages"] = _places(g, total, c["page"], 5)
    s["rows"] = tuple(_normal(g, s["pages"] * c["page"], kvheads, hd) for _ in "kv")
    s["q"] = _normal(g, starts[-1], kvheads * c["per_kv"], hd)
    return s


def _quantised(rows):
    """(codes, scales) of fp32 rows."""
    top = rows.abs().amax(-1, keepdim=True)
    live = top > 0
    inv = torch.where(live, (127.0 / top.double()).float(), torch.zeros_like(top))
    scale = torch.where(live, (top.double() / 127.0).float(), torch.ones_like(top))
    return torch.round(rows * inv).clamp(-127, 127).to(torch.int8), scale[..., 0]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _cache(c, pages):
    """An empty cache: the framework's, or a dict of tensors."""
    if own:
        from openneedle_amd.paged import PagedCache
        return PagedCache(1, pages, c["page"], c.get("kvheads", 1), c.get("head_dim", 32))
    if c["kind"] == "tables":  # the pages that are free, the next one last; a place behind them for what goes nowhere
        stack = torch.arange(pages - 1, -2, -1, dtype=torch.int32, device="cuda")
        return dict(stack=stack, top=torch.tensor(pages, device="cuda"))
    shape = (pages + 1, c["kvheads"], c["page"])  # the last page for rows without a slot
    k, v = (torch.zeros(shape + (c["head_dim"],), dtype=torch.int8, device="cuda") for _ in "kv")
    ks, vs = (torch.zeros(shape, device="cuda") for _ in "kv")
    return dict(k=k, v=v, ks=ks, vs=vs)


class _Address:
    """Device memory as torch takes it; the tensor keeps this object, which keeps the cache."""

    def __init__(self, at):
        self.at = at
        self.__cuda_array_interface__ = dict(data=(at.ptr, False), typestr="|i1", shape=(at.nbytes,), version=2)


def _rows_of(kv, c):
    """The framework cache's codes and scales as tensors over its own memory: a page's block of a kv head holds its K
    codes, V codes, K scales and V scales."""
    n, hd = c["page"], c["head_dim"]
    raw = torch.as_tensor(_Address(kv.device_pages(0)), device="cuda").view(kv.pages, kv.kvheads, n * (2 * hd + 8))
    k, v, ks, vs = raw.split((n * hd, n * hd, 4 * n, 4 * n), -1)
    return dict(k=k.unflatten(-1, (n, hd)), v=v.unflatten(-1, (n, hd)), ks=ks.view(torch.float32), vs=vs.view(torch.float32))


def prepare(case, seed):
    c, s = case, _inputs(case, seed)
    s["case"] = c
    if c["kind"] == "heads":
        s["q_out"], s["k_out"] = (torch.empty(t.shape, device="cuda") for t in (s["q"], s["k"]))
    else:
        s["kv"] = _cache(c, s["pages"])
    if c["kind"] == "store":
        s["rows"] = _rows_of(s["kv"], c) if own else {a: t[:-1] for a, t in s["kv"].items()}
    if c["kind"] == "tables":
        n = len(s["counts"])
        s["lengths"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        s["tables"] = torch.full((n, s["width"]), -1, dtype=torch.int32, device="cuda")
        s["out"] = dict(starts=torch.empty(n + 1, dtype=torch.int32, device="cuda"), firsts=torch.empty_like(s["counts"]),
                        slots=torch.empty(s["tokens"], dtype=torch.int32, device="cuda"),
                        positions=torch.empty(s["tokens"], dtype=torch.int32, device="cuda"))
        # the requests as they came to be: each longer than it is now, then cut, so that pages lie in no order
        room = (torch.minimum(s["past"] + s["mix"], s["past"] + s["counts"]))
        big = dict(s, counts=room, tokens=int(room.sum()))
        big["out"] = dict(s["out"], slots=torch.empty(big["tokens"], dtype=torch.int32, device="cuda"),
                          positions=torch.empty(big["tokens"], dtype=torch.int32, device="cuda"))
        _extend(big)
        _trim(s)
    if c["kind"] == "attention":
        s["out"] = torch.empty_like(s["q"])
        rows = s.pop("rows")
        counts, past = _requests(c)
        groups = {}  # requests of as many new tokens each, for the plain form
        for i, n in enumerate(counts):
            groups.setdefault(n, []).append(i)
        first = s["starts"].tolist()
        s["groups"] = [(n, torch.tensor(r, device="cuda"), torch.tensor([[first[i] + j for j in range(n)] for i in r],
                        device="cuda"), n + max(past[i] for i in r)) for n, r in sorted(groups.items())]
        s["count"], s["length"] = max(counts), max(a + b for a, b in zip(counts, past))
        if own:
            every = torch.arange(s["pages"] * c["page"], dtype=torch.int32, device="cuda")
            s["kv"].store(0, rows[0].data_ptr(), rows[1].data_ptr(), len(every), every.data_ptr(), stream=_stream())
        else:
            _put(s["kv"], rows, torch.arange(s["pages"] * c["page"], device="cuda"), c["page"])
        torch.cuda.synchronize()  # the rows are freed
    torch.cuda.synchronize()
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if kind == "tables":
        _extend(state)
        _trim(state)
        return dict(tables=state["tables"], lengths=state["lengths"], **state["out"])
    return (OWN if own else PLAIN)[kind](state)


def _extend(st):
    if not own:
        return _plain_extend(st)
    o = st["out"]
    st["kv"].extend(len(st["counts"]), st["counts"].data_ptr(), st["tokens"], st["lengths"].data_ptr(),
                    st["tables"].data_ptr(), st["width"], o["starts"].data_ptr(), o["firsts"].data_ptr(),
                    o["slots"].data_ptr(), o["positions"].data_ptr(), stream=_stream())


def _trim(st):
    if not own:
        return _plain_trim(st)
    st["kv"].trim(len(st["past"]), st["past"].data_ptr(), st["lengths"].data_ptr(), st["tables"].data_ptr(), st["width"],
                  stream=_stream())


def _own_heads(st):
    from openneedle_amd.heads import rotate_heads
    c = st["case"]
    rotate_heads(st["q"].data_ptr(), st["k"].data_ptr(), c["heads"], c["kvheads"], c["head_dim"], c["tokens"],
                 st["positions"].data_ptr(), st["freq"].data_ptr(), c["rotary"], d_q_gain=st["q_gain"].data_ptr(),
                 d_k_gain=st["k_gain"].data_ptr(), eps=1e-6, q_stride=st["q"].stride(0), k_stride=st["k"].stride(0),
                 d_q_out=st["q_out"].data_ptr(), d_k_out=st["k_out"].data_ptr(), stream=_stream())
    return dict(q=st["q_out"], k=st["k_out"])


def _own_store(st):
    st["kv"].store(0, st["k"].data_ptr(), st["v"].data_ptr(), st["case"]["tokens"], st["slots"].data_ptr(),
                   stream=_stream())
    return st["rows"]


def _own_attention(st):
    c = st["case"]
    st["kv"].attention(0, st["q"].data_ptr(), st["out"].data_ptr(), c["kvheads"] * c["per_kv"], len(st["counts"]),
                       st["tokens"], st["count"], st["starts"].data_ptr(), st["past"].data_ptr(), st["tables"].data_ptr(),
                       st["tables"].shape[1], st["length"], window=c["window"], stream=_stream())
    return st["out"]


def _plain_extend(st):
    """Pages from the top of the stack, request by request and page by page; a request past its table's width, or once
    the pages do not suffice, gets none and its tokens no slot. Without a wait for the GPU."""
    page, kv, tables = st["case"]["page"], st["kv"], st["tables"]
    n = st["lengths"].long()
    behind = st["counts"].long().cumsum(0)
    begin = behind - st["counts"]
    old, new = (n + page - 1) // page, (n + st["counts"] + page - 1) // page
    need = torch.where(new <= st["width"], new - old, 0)
    dealt = need.cumsum(0)
    granted = (new <= st["width"]) & ((need == 0) | (dealt <= kv["top"]))
    j = torch.arange(st["width"], device="cuda")
    take = granted[:, None] & (j >= old[:, None]) & (j < new[:, None])
    source = kv["top"] - 1 - ((dealt - need)[:, None] + j - old[:, None])
    tables.copy_(torch.where(take, kv["stack"][source.clamp(0, len(kv["stack"]) - 1)], tables))
    kv["top"] -= take.sum()
    t = torch.arange(st["tokens"], device="cuda")
    r = torch.searchsorted(behind, t, right=True)
    position = torch.where(granted[r], n[r] + t - begin[r], -1)
    at = position.clamp(min=0)
    o = st["out"]
    o["positions"].copy_(position)
    o["slots"].copy_(torch.where(position >= 0, tables[r, at // page] * page + at % page, -1))
    o["firsts"].copy_(torch.where(granted, n, -1))
    o["starts"][0] = 0
    o["starts"][1:].copy_(behind)
    st["lengths"] += torch.where(granted, st["counts"], 0)


def _plain_trim(st):
    """The first past[r] tokens of a request are kept; the pages behind them go back, the last one first."""
    page, kv, tables = st["case"]["page"], st["kv"], st["tables"]
    n = st["lengths"].long()
    keep = torch.minimum(n, st["past"].long())
    left, held = (keep + page - 1) // page, (n + page - 1) // page
    back = (held - left).cumsum(0)
    j = torch.arange(st["width"], device="cuda")
    gone = (j >= left[:, None]) & (j < held[:, None])
    to = kv["top"] + back[-1] - 1 - ((back - held + left)[:, None] + j - left[:, None])
    kv["stack"][torch.where(gone, to, len(kv["stack"]) - 1)] = tables
    tables.masked_fill_(gone, -1)
    kv["top"] += back[-1]
    st["lengths"].copy_(keep)


def _plain_heads(st):
    c = st["case"]
    half, hd = c["rotary"] // 2, c["head_dim"]
    angle = st["positions"].double()[:, None] * st["freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotated(x, gain):
        x = x.unflatten(-1, (-1, hd))
        x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)) * (1.0 + gain)
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), -1).flatten(1)

    return dict(q=rotated(st["q"], st["q_gain"]), k=rotated(st["k"], st["k_gain"]))


def _put(kv, rows, slots, page):
    """Rows [n, kvheads, head_dim] into slots [n] of a cache of tensors; those of slot -1 into its last page."""
    p, i = torch.where(slots >= 0, slots // page, kv["k"].shape[0] - 1), slots % page
    for name, x in zip("kv", rows):
        codes, scales = _quantised(x)
        kv[name][p, :, i] = codes
        kv[name + "s"][p, :, i] = scales


def _plain_store(st):
    _put(st["kv"], (st["k"], st["v"]), st["slots"], st["case"]["page"])
    return st["rows"]


def _plain_attention(st):
    c, kv, out = st["case"], st["kv"], st["out"]
    kvheads, group, hd, page = c["kvheads"], c["per_kv"], c["head_dim"], c["page"]
    for count, requests, tokens, length in st["groups"]:  # the requests of `count` new tokens, padded to the longest
        n, width = len(requests), (length + page - 1) // page
        at = st["tables"][requests, :width].long().clamp(min=0)
        k, v = ((kv[a][at].float() * kv[a + "s"][at][..., None]).transpose(1, 2).reshape(n * kvheads, width * page, hd)
                for a in "kv")
        q = st["q"][tokens].reshape(n, count, kvheads, group, hd).transpose(1, 2).reshape(n * kvheads, count * group, hd)
        score = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(hd)
        mine = st["past"].long()[requests][:, None] + torch.arange(count, device="cuda")
        j = torch.arange(width * page, device="cuda")
        hidden = j > mine[..., None]
        if c["window"]:
            hidden = hidden | (j <= mine[..., None] - c["window"])
        score = score.reshape(n, kvheads, count, group, -1).masked_fill_(hidden[:, None, :, None], -math.inf)
        score = torch.exp(score - score.amax(-1, keepdim=True))
        score = (score / score.sum(-1, keepdim=True)).reshape(n * kvheads, count * group, -1)
        got = torch.bmm(score, v).reshape(n, kvheads, count, group, hd).transpose(1, 2)
        out[tokens.flatten()] = got.reshape(n * count, kvheads * group, hd)
    return out


OWN = dict(heads=_own_heads, store=_own_store, attention=_own_attention)
PLAIN = dict(heads=_plain_heads, store=_plain_store, attention=_plain_attention)


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "heads":
        n, rows = c["tokens"], c["heads"] + c["kvheads"]
        return dict(bytes=n * (8.0 * rows * c["head_dim"] + 4) + 8 * c["head_dim"] + 4 * c["rotary"],
                    flops=8.0 * n * rows * c["head_dim"])
    if c["kind"] == "store":
        return dict(bytes=c["tokens"] * (4.0 + 2 * c["kvheads"] * (5 * c["head_dim"] + 4)),
                    flops=6.0 * c["tokens"] * c["kvheads"] * c["head_dim"])
    counts, past = _requests(c)
    if c["kind"] == "tables":
        # counts, lengths, first positions and where the tokens begin; a slot and a position a token; its page, and of
        # every new page its entry in the table and in the stack, written by both calls
        new = sum(counts) / c["page"]
        return dict(bytes=32.0 * len(counts) + 8.0 * sum(counts) + 4.0 * len(counts) + 16.0 * new, flops=0.0)
    window = c["window"] or 1 << 30
    heads, kvheads, hd = c["kvheads"] * c["per_kv"], c["kvheads"], c["head_dim"]
    keys = sum(min(n + past_n, window + n - 1) for n, past_n in zip(counts, past))  # of all requests
    pairs = sum(min(p + i + 1, window) for n, p in zip(counts, past) for i in range(n))  # of tokens and keys
    return dict(bytes=8.0 * sum(counts) * heads * hd + 2.0 * (hd + 4) * kvheads * keys, flops=4.0 * heads * hd * pairs)


# ---- the same in 64 bits, one request, token or head at a time --------------------------------------------------------
def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["kind"] == "tables":
        return None  # whole numbers
    hd = c["head_dim"]
    if c["kind"] == "store":  # the codes are defined in 32 bits
        out = dict(k=None, v=None)
        for name in "kv":
            scales = torch.zeros((s["pages"] * c["page"], c["kvheads"]), dtype=torch.float64, device="cuda")
            for h in range(c["kvheads"]):
                live = s["slots"] >= 0
                scales[s["slots"][live].long(), h] = s[name][live, h].double().abs().amax(-1) / 127
            out[name + "s"] = scales.reshape(s["pages"], c["page"], -1).transpose(1, 2)
        return out
    if c["kind"] == "heads":
        out = {}
        for name in "qk":
            x = s[name].double().reshape(c["tokens"], -1, hd)
            y = x / (x.pow(2).sum(-1, keepdim=True) / hd + 1e-6).sqrt() * (1 + s[name + "_gain"].double())
            z = y.clone()
            for j in range(c["rotary"] // 2):
                turn = torch.polar(torch.ones_like(s["freq"][:1]), s["positions"].double() * s["freq"][j])
                pair = torch.complex(y[..., j], y[..., j + c["rotary"] // 2]) * turn[:, None]
                z[..., j], z[..., j + c["rotary"] // 2] = pair.real, pair.imag
            out[name] = z.reshape(c["tokens"], -1)
        return out
    # the quantiser is defined in 32 bits, so the codes are made there
    k, v = (codes.double() * scales.double()[..., None] for codes, scales in map(_quantised, s["rows"]))
    counts, past = _requests(c)
    out, group, token = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), c["per_kv"], 0
    for r, (n, p) in enumerate(zip(counts, past)):
        slots = _slots(s["tables"][r:r + 1], torch.arange(p + n, device="cuda")[None], c["page"])[0].long()
        back = torch.arange(p, p + n, device="cuda")[:, None] - torch.arange(p + n, device="cuda")
        hidden = (back < 0) | (back >= (c["window"] or 1 << 30))
        for h in range(c["kvheads"]):
            kh, vh = k[slots, h], v[slots, h]
            for g in range(h * group, (h + 1) * group):
                x = torch.matmul(s["q"][token:token + n, g].double(), kh.T.contiguous()) / math.sqrt(hd)
                out[token:token + n, g] = torch.matmul(torch.softmax(x.masked_fill(hidden, -math.inf), -1), vh)
        token += n
    return out
