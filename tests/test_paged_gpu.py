"""The paged cache: tables against the model of tests/test_paged.py entry by entry, stores bit by bit, attention of ragged
tokens against the closed form in 64 bits with the tolerance of tests/test_span_gpu.py (many rows over the same keys: as
check_many_rows there, tiles of 32 positions), and a whole serving step, eager and captured.
"""
import ctypes as ct

import numpy as np
import pytest

import oracle
from openneedle_amd import _ffi
from openneedle_amd._ffi import GpuError
from openneedle_amd.device import DeviceArray, Graph, Stream, synchronize
from openneedle_amd.heads import rotary_frequencies, rotate_heads
from openneedle_amd.paged import PagedCache
from tests.test_paged import Pool
from tests.test_span_gpu import attend, check, upload

pytestmark = pytest.mark.gpu


def ints(a):
    return upload(a, np.int32)


class Tables:
    """A cache's tables on the device beside the host's model of them."""

    def __init__(self, pages, page, requests, width, kvheads=1, hd=32, layers=1):
        self.kv, self.model = PagedCache(layers, pages, page, kvheads, hd), Pool(pages, page, requests, width)
        self.requests, self.width = requests, width
        self.lengths, self.tables = ints(np.zeros(requests)), ints(np.full((requests, width), -1))

    def extend(self, counts, tokens, stream=None):
        out = [ints(np.full(n, 77)) for n in (self.requests + 1, self.requests, max(tokens, 1), max(tokens, 1))]
        self.kv.extend(self.requests, ints(counts), tokens, self.lengths, self.tables, self.width, *out, stream=stream)
        synchronize()
        got = [d.to_host(np.int32, n) for d, n in zip(out, (self.requests + 1, self.requests, tokens, tokens))]
        for g, w, name in zip(got, self.model.extend([int(c) for c in counts], tokens), ("starts", "firsts", "slots", "positions")):
            np.testing.assert_array_equal(g, w, name)
        self.same()
        return got

    def trim(self, keep):
        self.kv.trim(self.requests, ints(keep), self.lengths, self.tables, self.width)
        synchronize()
        self.model.trim([int(k) for k in keep])
        self.same()

    def same(self):
        np.testing.assert_array_equal(self.lengths.to_host(np.int32, self.requests), self.model.lengths)
        np.testing.assert_array_equal(self.tables.to_host(np.int32, (self.requests, self.width)), self.model.tables)
        assert self.kv.free_pages() == len(self.model.stack)


@pytest.mark.parametrize("page", [16, 32, 256])
def test_tables_by_steps(page):
    """Requests that come, grow, are cut and end, more of them than the pages hold at times."""
    rng = np.random.default_rng(page)
    t = Tables(90, page, 23, 9)
    for step in range(30):
        counts = rng.choice([-3, 0, 1, 1, 1, 2, page - 1, page, page + 1, 3 * page + 5, 10 * page], 23)
        total = int(np.maximum(counts, 0).sum())
        t.extend(counts, max(1, total + rng.integers(-40, 40)))
        keep = np.array(t.model.lengths) - rng.choice([0, 0, 1, 5, page, 2 ** 30, -7], 23)
        t.trim(keep)


@pytest.mark.parametrize("requests,most", [(1, 5000), (2, 1), (700, 40), (1024, 3), (1025, 3), (8192, 4)])
def test_tables_of_many_requests(requests, most):
    """One block and several, requests a thread from none to eight."""
    rng = np.random.default_rng(requests)
    t = Tables(requests * 3 + most // 8, 16, requests, most // 16 + 2)
    for _ in range(3):
        counts = rng.integers(0, most + 1, requests) * (rng.random(requests) < 0.8)
        t.extend(counts, int(counts.sum()) + 9)
        t.trim(np.maximum(np.array(t.model.lengths) - rng.integers(0, most // 2 + 2, requests), 0))
    t.trim(np.zeros(requests))
    assert t.kv.free_pages() == t.kv.pages


def test_extension_undone_by_trim():
    """A trim to the lengths before it leaves the stack of free pages as it was: the next extension deals the same."""
    t = Tables(150, 16, 40, 12)
    t.extend(np.arange(40) % 50, 2000)
    t.trim(np.arange(40) // 2)
    before, stack = list(t.model.lengths), list(t.model.stack)
    a = t.extend(np.full(40, 21), 840)
    t.trim(a[1])  # the first positions: -1 where a request got nothing
    assert t.model.lengths == before
    assert t.model.stack == stack
    for x, y in zip(a, t.extend(np.full(40, 21), 840)):
        np.testing.assert_array_equal(x, y)


def test_no_requests_and_no_tokens():
    t = Tables(5, 16, 3, 2)
    t.extend([0, 0, 0], 4)
    t.extend([1, 2, 3], 0)
    kv = t.kv
    out = [ints(np.full(n, 77)) for n in (1, 1, 3, 3)]
    kv.extend(0, None, 3, None, None, 1, out[0], None, out[2], out[3])
    synchronize()
    assert out[0].to_host(np.int32, 1)[0] == 0
    assert (out[2].to_host(np.int32, 3) == -1).all() and (out[3].to_host(np.int32, 3) == -1).all()
    kv.trim(0, None, None, None, 1)
    kv.reset()
    assert kv.free_pages() == 5


def test_tables_that_were_not_dealt_are_safe():
    """Lengths below zero and past the table, and pages outside the cache: no request, no slot."""
    kv = PagedCache(1, 6, 16, 1, 32)
    lengths, tables = ints([-5, 33, 2 ** 31 - 1, 16]), ints([[0, 1], [2, 3], [4, 5], [99, -1]])
    out = [ints(np.full(n, 77)) for n in (5, 4, 4, 4)]
    kv.extend(4, ints([1, 1, 1, 1]), 4, lengths, tables, 2, *out)
    synchronize()
    np.testing.assert_array_equal(out[1].to_host(np.int32, 4), [-1, -1, -1, 16])
    np.testing.assert_array_equal(out[2].to_host(np.int32, 4), [-1, -1, -1, 0])
    np.testing.assert_array_equal(lengths.to_host(np.int32, 4), [-5, 33, 2 ** 31 - 1, 17])
    kv.extend(4, ints([0, 0, 0, 15]), 15, lengths, ints([[0, 1], [2, 3], [4, 5], [99, 600]]), 2, out[0], out[1],
              *(ints(np.zeros(15)) for _ in "sp"))
    synchronize()
    kv.trim(4, ints([-1, -7, 2 ** 31 - 1, 20]), lengths, tables, 2)  # (the last one has 17 + 15)
    np.testing.assert_array_equal(lengths.to_host(np.int32, 4), [-5, 33, 2 ** 31 - 1, 20])
    many = ints([[9, 9, 9]] * 9)
    kv.trim(9, ints([0] * 9), ints([48] * 9), many, 3)
    assert kv.free_pages() == 6


# ---- rows ------------------------------------------------------------------------------------------------------------
class Rows:
    """A layer's rows on the host, [pages][kvheads][page] codes and scales."""

    def __init__(self, kv, layer=0):
        self.kv, self.layer = kv, layer
        shape = (kv.pages, kv.kvheads, kv.page_size)
        self.k, self.v = (np.zeros(shape + (kv.head_dim,), np.int8) for _ in "kv")
        self.ks, self.vs = (np.zeros(shape, np.float32) for _ in "kv")

    def fill(self, rng):
        self.k, self.v = (rng.integers(-127, 128, x.shape).astype(np.int8) for x in (self.k, self.v))
        self.ks, self.vs = (rng.uniform(0.01, 0.025, x.shape).astype(np.float32) for x in (self.ks, self.vs))
        self.push()
        return self

    def blocks(self):
        flat = self.k.shape[:2]
        parts = (self.k, self.v, self.ks.view(np.int8), self.vs.view(np.int8))
        return np.concatenate([p.reshape(flat + (-1,)) for p in parts], -1)

    def push(self):
        self.kv.device_pages(self.layer).upload(self.blocks())

    def put(self, slots, k, v):
        for codes, scales, rows in ((self.k, self.ks, k), (self.v, self.vs, v)):
            for i, s in enumerate(slots):
                if 0 <= s < self.kv.pages * self.kv.page_size:
                    c, x = oracle.kv_quantize(rows[i][None])
                    p, o = divmod(int(s), self.kv.page_size)
                    codes[p, :, o], scales[p, :, o] = c[0], x[0]

    def same(self):
        w = self.blocks()
        np.testing.assert_array_equal(self.kv.device_pages(self.layer).to_host(np.int8, w.shape), w)

    def at(self, table, positions, h):
        positions = np.asarray(positions, np.int64)
        p, o = np.asarray(table, np.int64)[positions // self.kv.page_size], positions % self.kv.page_size
        return ((self.k[p, h, o].astype(np.float64) * self.ks[p, h, o, None].astype(np.float64)),
                (self.v[p, h, o].astype(np.float64) * self.vs[p, h, o, None].astype(np.float64)))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("page,kvheads,tokens", [(16, 1, 1), (16, 5, 37), (64, 8, 300), (256, 3, 100)])
def test_store(hd, page, kvheads, tokens):
    """Slots in no order, some outside the cache; rows in one projection's rows; the second of two layers."""
    rng = np.random.default_rng(hd + tokens)
    pages = 2 * tokens // page + 3
    kv = PagedCache(2, pages, page, kvheads, hd)
    r, other = Rows(kv, 1).fill(rng), Rows(kv, 0).fill(rng)
    stride = 3 * kvheads * hd + 4
    rows = rng.normal(size=(tokens, stride)).astype(np.float32)
    rows[tokens // 2, :hd] = 0
    slots = rng.permutation(pages * page)[:tokens]
    slots[rng.random(tokens) < 0.2] = rng.choice([-1, -2 ** 31, pages * page, 2 ** 31 - 1])
    d = upload(rows)
    kv.store(1, d, d.view(kvheads * hd * 4, 16), tokens, ints(slots), k_stride=stride, v_stride=stride)
    synchronize()
    k, v = (rows[:, i * kvheads * hd:(i + 1) * kvheads * hd].reshape(tokens, kvheads, hd) for i in (0, 1))
    r.put(slots, k, v)
    r.same()
    other.same()


def test_store_far_into_a_large_cache():
    """Rows whose offsets pass 32 bits."""
    kv = PagedCache(1, 140000, 16, 16, 128)  # 9.5 GB
    rng = np.random.default_rng(3)
    slots = np.array([139999 * 16 + 15, 17, 70000 * 16])
    k, v = (rng.normal(size=(3, 16, 128)).astype(np.float32) for _ in "kv")
    kv.store(0, upload(k), upload(v), 3, ints(slots))
    # two requests: one of page 139999's last position in a table of its own, one through 70000 and 1
    rows = 16 * (2 * 128 + 8)
    for i, s in enumerate(slots):
        page, off = divmod(int(s), 16)
        for h in (0, 15):
            raw = kv.device_pages(0).view((page * 16 + h) * rows, rows).to_host(np.int8, rows)
            c, x = oracle.kv_quantize(k[i, h][None, None])
            np.testing.assert_array_equal(raw[:16 * 128].reshape(16, 128)[off], c[0, 0])
            assert raw[2 * 16 * 128:].view(np.float32)[off] == x[0, 0]
    # position 15 of page 139999 and position 0 of page 70000 alone have codes: zeros have scale 0 and weight 1 / n
    out = ints(np.zeros((2, 16, 128)))
    q = np.zeros((2, 16, 128), np.float32)
    kv.attention(0, upload(q), out, 16, 2, 2, 1, ints([0, 1, 2]), ints([15, 31]), ints([[139999, -1], [70000, 1]]), 2)
    synchronize()
    got = out.to_host(np.float32, (2, 16, 128))
    vals = [c[0].astype(np.float64) * x[0][:, None] for c, x in (oracle.kv_quantize(v[i][None]) for i in range(3))]
    np.testing.assert_allclose(got[0], vals[0] / 16, rtol=1e-6, atol=1e-9)
    np.testing.assert_allclose(got[1], (vals[1] + vals[2]) / 32, rtol=1e-6, atol=1e-8)


# ---- attention ---------------------------------------------------------------------------------------------------------
class Batch:
    """Requests over pages in no order; `past` positions each before `counts` new tokens."""

    def __init__(self, rng, kvheads, group, hd, counts, past, page=16, spare=3, extra_width=1):
        self.counts, self.past, self.group = list(counts), list(past), group
        need = [-(-(c + max(p, 0)) // page) for c, p in zip(counts, past)]
        pages = sum(need) + spare
        order = rng.permutation(pages)
        self.width = max([*need, 0]) + extra_width
        self.tables = np.full((len(counts), self.width), -1)
        at = 0
        for r, n in enumerate(need):
            self.tables[r, :n] = order[at:at + n]
            at += n
        self.kv = PagedCache(1, pages, page, kvheads, hd)
        self.rows = Rows(self.kv).fill(rng)
        self.starts = np.concatenate([[0], np.cumsum(counts)])
        self.q = rng.normal(size=(int(self.starts[-1]), kvheads * group, hd)).astype(np.float32)

    def run(self, window=0, length=0, count=None, tail=0, stream=None, firsts=None):
        """`tail` rows of no request behind the last one's; returned too."""
        q = np.concatenate([self.q, np.ones((tail, *self.q.shape[1:]), np.float32)])
        out = DeviceArray.from_host(np.full(q.shape, np.nan, np.float32))
        self.held = [upload(q), ints(self.starts), ints(self.past if firsts is None else firsts), ints(self.tables)]
        n = len(self.counts)
        self.kv.attention(0, self.held[0], out, q.shape[1], n, len(q), max(self.counts) if count is None else count,
                          *self.held[1:], self.width, length, window, stream=stream)
        synchronize()
        return out.to_host(np.float32, q.shape)

    def check(self, got, window=0, rows=None, gone=(), many=False):
        """`gone`: pages that are none. `rows`: (request, token)s, default all."""
        kvh, page = self.kv.kvheads, self.kv.page_size
        for r, (n, p) in enumerate(zip(self.counts, self.past)):
            for i in range(n):
                if rows is not None and (r, i) not in rows:
                    continue
                token = self.starts[r] + i
                seen = np.arange(max(0, p + i - window + 1) if window else 0, p + i + 1) if p >= 0 else np.arange(0)
                seen = np.array([j for j in seen if self.tables[r, j // page] not in gone], np.int64) if gone else seen
                for h in range(kvh):
                    k, v = self.rows.at(self.tables[r], seen, h) if len(seen) else (np.zeros((0, 1)),) * 2
                    for g in range(self.group):
                        want, tol, w = attend(self.q[token, h * self.group + g], k, v)
                        if many and len(seen):
                            pg, o = self.tables[r][seen // page], seen % page
                            vs = np.abs(self.rows.vs[pg, h, o].astype(np.float64))
                            codes = np.abs(self.rows.v[pg, h, o].astype(np.float64))
                            for t in np.unique(seen // 32):
                                mine = seen // 32 == t
                                tol = tol + 2.0 ** -27 * (w[mine] * vs[mine]).max() * codes[mine].sum(0)
                        check(got[token, h * self.group + g], want, tol, f"request {r} token {i} head {h * self.group + g}")


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kvheads,group", [(1, 1), (2, 2), (2, 3), (1, 8), (3, 5), (1, 16)])
def test_one_token_each(hd, kvheads, group):
    """Lengths around the tiles and pages, a request without tokens, one at a negative position; rows behind the last
    request's stay as they were."""
    rng = np.random.default_rng(hd + 10 * kvheads + group)
    b = Batch(rng, kvheads, group, hd, [1, 1, 1, 0, 1, 1, 1, 1, 1, 1], [0, 1, 14, 9, 15, 16, -1, 63, 64, 700])
    got = b.run(tail=3)
    b.check(got[:len(b.q)])
    assert np.isnan(got[len(b.q):]).all()


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_pages_of_every_size(hd, page):
    rng = np.random.default_rng(hd + page)
    b = Batch(rng, 2, 4, hd, [1, 2, 1], [3 * page + 5, page - 1, 5 * page], page=page)
    b.check(b.run())


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("window", [1, 5, 63, 64, 65, 300])
def test_window(hd, window):
    rng = np.random.default_rng(hd + window)
    b = Batch(rng, 2, 2, hd, [1, 1, 5, 1, 3, 1], [0, 63, 64, 65, 300, 1000], page=32)
    b.check(b.run(window), window)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("length", [0, 1, 3000, 40000])
def test_several_pieces(hd, length):
    """Long caches of few requests, cut into pieces; some requests have one piece, or none. The hint changes nothing that
    is right."""
    rng = np.random.default_rng(hd + length)
    b = Batch(rng, 1, 2, hd, [1, 1, 2, 1, 0, 1], [2999, 10, 1500, -4, 0, 700], extra_width=2500)
    b.check(b.run(length=length))
    b.check(b.run(window=900, length=length), 900)


MANY_PIECES = [(32, 66100), (64, 32768), (64, 32767), (128, 16400)]  # rows of so many values, and the longest request's positions


@pytest.mark.parametrize("hd,past", MANY_PIECES)
def test_more_pieces_than_a_wave_has_lanes(hd, past):
    """One long request by itself and beside short ones, with a length given and cut for the tables' width."""
    rng = np.random.default_rng(hd + past)
    b = Batch(rng, 1, 2, hd, [1], [past], page=64)
    b.check(b.run(length=past + 1))
    b.check(b.run())
    b = Batch(rng, 1, 2, hd, [1, 1, 2, 0, 1], [257, -1, past, 4, 0], page=64)
    b.check(b.run(length=past + 2))


ORDERED = [(40, 8), (64, 5), (65, 4), (130, 3), (511, 1)]  # requests and kv heads


@pytest.mark.parametrize("requests,kvheads", ORDERED)
def test_requests_in_the_order_of_their_lengths(requests, kvheads):
    """More blocks than compute units: every request is taken once, whatever lengths they share, tokens or not, padded or
    past their tables."""
    rng = np.random.default_rng(requests)
    past = [int(x) for x in rng.choice([0, 1, 60, 61, 61, 61, 200, 300, 300, 1100, -1, -7], requests)]
    counts = [int(c) for c in rng.choice([1, 1, 1, 1, 2, 0], requests)]
    b = Batch(rng, kvheads, 2, 32, counts, past, page=32)
    assert b.width * 32 >= 1152
    got = b.run(length=1152)
    assert np.isfinite(got).all()
    b.check(got)
    firsts = list(past)
    firsts[3], firsts[-2] = 2 ** 31 - 1, 32 * b.width
    b.past = [p if f == p else -1 for p, f in zip(past, firsts)]
    b.check(b.run(length=1152, firsts=firsts))
    same = Batch(rng, kvheads, 2, 32, [1] * requests, [77] * requests, page=32, extra_width=40)
    same.check(same.run(length=1152))


def test_the_same_numbers_again():
    """Records of a call do not reach into the next one, whatever its requests are."""
    rng = np.random.default_rng(12)
    b = Batch(rng, 2, 2, 64, [1, 3, 1], [5000, 2500, 40])
    first = b.run(length=6000)
    b.check(first)
    few = b.run(length=6000, firsts=[20, 30, -1])
    keep, b.past = b.past, [20, 30, -1]
    b.check(few)
    b.past = keep
    np.testing.assert_array_equal(b.run(length=6000), first)


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_pages_that_are_none(hd):
    """Pages of -1 and outside the cache inside a request are not attended; a request without any attends nothing."""
    rng = np.random.default_rng(hd)
    b = Batch(rng, 2, 3, hd, [1, 4, 1, 2], [200, 150, 40, 90])
    whole = b.tables.copy()
    b.tables[0, 3], b.tables[0, 12], b.tables[1, 0], b.tables[1, 9] = -1, 2 ** 31 - 1, 10 ** 6, -2 ** 31
    b.tables[2] = -1
    got = b.run()
    assert not got[b.starts[2]].any()
    gone = {int(x) for x in (whole[0, 3], whole[0, 12], whole[1, 0], whole[1, 9], *whole[2, :3])}
    b.tables = whole
    b.check(got, gone=gone)


def test_what_is_not_attended_does_not_matter():
    """Positions behind a token and before its window, pages of no request and rows behind the last position hold
    infinite and NaN scales."""
    for counts, past, window in (([1, 1], [50, 333], 0), ([1, 3], [200, 333], 100), ([40, 70], [200, 333], 100), ([90, 2], [0, 40], 0)):
        rng = np.random.default_rng(6)
        b = Batch(rng, 2, 2, 64, counts, past, page=32, spare=4)
        live = np.zeros(b.rows.ks.shape, bool)
        for r, (n, p) in enumerate(zip(counts, past)):
            for j in range(max(0, p - window + 1) if window else 0, p + n):
                live[b.tables[r, j // 32], :, j % 32] = True
        dead = np.where(rng.random(live.shape) < 0.5, np.nan, np.inf).astype(np.float32)
        b.rows.ks, b.rows.vs = np.where(live, b.rows.ks, dead), np.where(live, b.rows.vs, dead[::-1])
        b.rows.push()
        b.check(b.run(window), window, many=max(counts) > 9)


def test_non_finite_queries():
    rng = np.random.default_rng(8)
    b = Batch(rng, 2, 4, 64, [1, 30], [400, 100])
    b.q[0, 1, 3], b.q[5, 6, 9] = np.nan, np.inf
    got = b.run()
    assert not got[0, 1].any() and not got[5, 6].any()
    b.q[0, 1], b.q[5, 6] = 0, 0
    clean = b.run()
    b.check(clean, many=True)
    got[0, 1], got[5, 6] = clean[0, 1], clean[5, 6]
    b.check(got, many=True)


def test_starts_and_firsts_that_do_not_fit():
    """Tokens past q, and requests past their tables, are no access outside: zeros, or rows as they were."""
    rng = np.random.default_rng(9)
    b = Batch(rng, 1, 2, 64, [1, 1, 1], [20, 40, 10])
    b.starts = np.array([0, 1, 2, 900])
    got = b.run(firsts=[20, 48 + 16 * b.width, 2 ** 31 - 1])
    b.check(got, rows=[(0, 0)])
    assert not got[1:].any()
    b.starts = np.array([-5, 1, 0, 3])
    b.run()
    b.starts = np.array([0, 1, 2, 3])
    got = b.run(count=0)
    assert np.isnan(got).all()


def test_refusals():
    kv = PagedCache(2, 10, 16, 2, 64)
    with DeviceArray(1 << 16) as d:
        ok = dict(layer=0, d_q=d, d_out=d, heads=4, requests=1, tokens=2, count=2, d_starts=d, d_firsts=d, d_tables=d, width=3)
        for change, word in [(dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(heads=3), "multiple"), (dict(heads=34), "16 query"),
                             (dict(count=3), "count"), (dict(requests=8193), "8192"), (dict(width=0), "width"), (dict(d_q=None), "null"),
                             (dict(d_tables=None), "null"), (dict(window=-1), "window"), (dict(d_q=d.ptr + 4), "16 bytes"),
                             (dict(d_out=d.ptr + 8), "16 bytes"), (dict(length=-1), "length"), (dict(tokens=2 ** 25 + 1, count=1), "2^25")]:
            with pytest.raises(GpuError, match=word.replace("^", r"\^")):
                kv.attention(**{**ok, **change})
        for call, word in [(lambda: kv.store(2, d, d, 1, d), "layer"), (lambda: kv.store(0, d, None, 1, d), "null"),
                           (lambda: kv.store(0, d, d, 1, None), "null"), (lambda: kv.store(0, d, d, 1, d, k_stride=64), "stride"),
                           (lambda: kv.store(0, d, d.ptr + 4, 1, d), "16 bytes"), (lambda: kv.store(0, d, d, -1, d), "tokens"),
                           (lambda: kv.extend(1, None, 1, d, d, 1, d, d, d, d), "null"), (lambda: kv.extend(1, d, 1, d, d, 0, d, d, d, d), "width"),
                           (lambda: kv.extend(1, d, 1, d, d, 1, d, d, None, d), "null"), (lambda: kv.trim(1, None, d, d, 1), "null"),
                           (lambda: kv.device_pages(2), "layer"), (lambda: kv.store_rotated(0, d, d, d, 4, 1, d, None), "null"),
                           (lambda: kv.store_rotated(0, d, d, None, 4, 1, d, d), "null"),
                           (lambda: kv.store_rotated(0, d, d, d, 4, 1, d, d, d, rotary=66), "rotary")]:
            with pytest.raises(GpuError, match=word):
                call()
    with pytest.raises(GpuError, match="page_size"):
        PagedCache(1, 10, 17, 1, 64)


# ---- a step ------------------------------------------------------------------------------------------------------------
class Server:
    """What a serving program keeps: a step is extend, rotate and store, attend, all on one stream, from the counts on
    the device alone."""

    def __init__(self, rng, requests, tokens, heads, kvheads, hd, pages, page, width, stream):
        self.rng, self.stream, self.hd, self.heads, self.kvheads = rng, stream, hd, heads, kvheads
        self.requests, self.tokens, self.width = requests, tokens, width
        self.kv = PagedCache(1, pages, page, kvheads, hd)
        self.model, self.rows = Pool(pages, page, requests, width), Rows(self.kv)
        self.freq = rotary_frequencies(10000.0, hd)
        self.gains = [rng.normal(size=hd).astype(np.float32) * 0.2 for _ in "qk"]
        self.d = dict(freq=upload(self.freq, np.float64), qg=upload(self.gains[0]), kg=upload(self.gains[1]),
                      qkv=DeviceArray(tokens * (heads + 2 * kvheads) * hd * 4), q=DeviceArray(tokens * heads * hd * 4),
                      k=DeviceArray(tokens * kvheads * hd * 4), out=DeviceArray(tokens * heads * hd * 4),
                      counts=ints(np.zeros(requests)), lengths=ints(np.zeros(requests)), tables=ints(np.full((requests, width), -1)),
                      starts=ints(np.zeros(requests + 1)), firsts=ints(np.zeros(requests)), slots=ints(np.zeros(tokens)),
                      positions=ints(np.zeros(tokens)))

    def issue(self, count):
        d, row = self.d, (self.heads + 2 * self.kvheads) * self.hd
        q = d["qkv"].ptr
        k, v = q + self.heads * self.hd * 4, q + (self.heads + self.kvheads) * self.hd * 4
        self.kv.extend(self.requests, d["counts"], self.tokens, d["lengths"], d["tables"], self.width, d["starts"], d["firsts"],
                       d["slots"], d["positions"], stream=self.stream)
        self.kv.store_rotated(0, q, k, v, self.heads, self.tokens, d["positions"], d["slots"], d["freq"], self.hd,
                              d["qg"], d["kg"], q_stride=row, k_stride=row, v_stride=row, d_q_out=d["q"], d_k_out=d["k"],
                              stream=self.stream)
        self.kv.attention(0, d["q"], d["out"], self.heads, self.requests, self.tokens, count, d["starts"], d["firsts"],
                          d["tables"], self.width, self.width * self.kv.page_size, stream=self.stream)

    def feed(self, counts):
        rows = self.rng.normal(size=(self.tokens, (self.heads + 2 * self.kvheads) * self.hd)).astype(np.float32)
        self.d["qkv"].upload(rows)
        self.d["counts"].upload(np.asarray(counts, np.int32))
        for name in ("out", "q", "k"):
            self.d[name].fill(0xFF)
        synchronize()
        return rows

    def verify(self, counts, rows, many):
        synchronize()
        starts, firsts, slots, positions = self.model.extend([int(c) for c in counts], self.tokens)
        for name, want in (("starts", starts), ("firsts", firsts), ("slots", slots), ("positions", positions), ("lengths", self.model.lengths),
                           ("tables", np.ravel(self.model.tables))):
            np.testing.assert_array_equal(self.d[name].to_host(np.int32, len(want)), want, name)
        q, k, out = (self.d[n].to_host(np.float32, (self.tokens, h, self.hd)) for n, h in
                     (("q", self.heads), ("k", self.kvheads), ("out", self.heads)))
        live = np.array(positions) >= 0
        v = rows.reshape(self.tokens, -1, self.hd)[:, self.heads + self.kvheads:]
        assert np.isnan(q[~live]).all()
        self.rows.put([s if ok else -1 for s, ok in zip(slots, live)], k, v)
        self.rows.same()  # the stored rows are the quantiser's of k and v, bit for bit
        from tests.test_heads_gpu import heads_of
        x = rows.reshape(self.tokens, -1, self.hd)
        for got, part, gain in ((q, x[:, :self.heads], self.gains[0]), (k, x[:, self.heads:self.heads + self.kvheads], self.gains[1])):
            want, tol = heads_of(part[live], np.array(positions)[live], gain, self.freq, 1e-6)
            assert (np.abs(got[live] - want) <= tol).all()
        b = Batch.__new__(Batch)
        b.kv, b.rows, b.group, b.tables, b.starts, b.q = self.kv, self.rows, self.heads // self.kvheads, np.array(self.model.tables), starts, q
        b.counts = [max(int(c), 0) if f >= 0 else 0 for c, f in zip(counts, firsts)]
        b.past = firsts
        b.check(out, many=many)
        for r, f in enumerate(firsts):
            if f < 0:
                assert not out[starts[r]:starts[r + 1]].any()
        assert np.isnan(out[starts[-1]:]).all()

    def step(self, counts, count):
        rows = self.feed(counts)
        self.issue(count)
        self.verify(counts, rows, count > 8)


def test_serving_steps():
    """Prompts, decode steps, a mix of both, drafts taken back, a request that ends and one that comes, and more than the
    pages hold."""
    rng = np.random.default_rng(21)
    s = Server(rng, 5, 120, 4, 2, 64, 30, 16, 20, Stream())
    s.step([50, 7, 0, 33, 1], 50)
    for _ in range(3):
        s.step([1, 1, 0, 1, 1], 1)
    s.step([1, 4, 60, 1, 5], 60)
    keep = [n - (2 if r in (1, 4) else 0) for r, n in enumerate(s.model.lengths)]
    keep[0] = 0
    s.kv.trim(5, ints(keep), s.d["lengths"], s.d["tables"], s.width, stream=s.stream)
    s.model.trim(keep)
    s.step([20, 1, 1, 1, 1], 20)
    s.step([1, 100, 1, 0, 1], 120)
    for _ in range(2):
        s.step([0, 100, 1, 90, 1], 120)  # the pages end


def test_serving_step_captured():
    """One graph serves every step: counts, lengths and tables change on the device between its replays, eager calls of
    other sizes between them; two graphs share the cache's scratch."""
    rng = np.random.default_rng(22)
    stream = Stream()
    s = Server(rng, 4, 40, 4, 2, 64, 400, 16, 90, stream)
    s.step([30, 1, 3, 0], 30)
    graphs = []
    for count in (40, 1):
        s.step([1, 1, 1, 1], count)  # what is captured has run once
        s.feed([0] * 4)
        with Graph.capture(stream) as g:
            s.issue(count)
        graphs.append(g)
    steps = [([1, 1, 1, 1], 1), ([5, 0, 1, 31], 0), ([1, 1, 0, 1], 1), ([0, 40, 0, 0], 0), ([1, 1, 1, 1], 0), ([1, 1, 1, 1], 1)]
    for i, (counts, which) in enumerate(steps):
        rows = s.feed(counts)
        graphs[which].launch(stream)
        s.verify(counts, rows, which == 0)
        if i == 2:  # outgrows the records in between; the graphs keep theirs
            other = Batch(rng, 2, 2, 64, [1, 9], [1200, 800])
            q, out = upload(other.q), DeviceArray.from_host(np.zeros(other.q.shape, np.float32))
            s.kv.attention(0, q, out, 4, 2, 10, 9, ints(other.starts), ints([0, 0]), ints(np.zeros((2, 5000))), 5000)
            synchronize()
        s.step([1, 0, 1, 2], 2)
    for g in graphs:
        g.close()


RECORDED = dict(hd=64, requests=3, tokens=130, kvheads=2, group=2, width=375, page=16)  # of a captured step
RECORDED_COUNTS = (1, 130)  # most tokens of a request, in the order in which the steps are captured
OUTGROWN = dict(tokens=700, count=400)  # of a later eager call


def test_graphs_whose_calls_have_records():
    """Steps cut into pieces, in blocks of 16 rows and of 128, captured in two graphs, each with scratch that the next call
    outgrows; then they are replayed in turn beside eager calls, which share the larger scratch, every output checked."""
    rng = np.random.default_rng(24)
    c, stream = RECORDED, Stream()
    s = Server(rng, c["requests"], c["tokens"], c["kvheads"] * c["group"], c["kvheads"], c["hd"], 200, c["page"], c["width"], stream)
    for counts in [[130, 0, 0]] * 6 + [[0, 130, 0]] * 3 + [[0, 0, 5]]:  # stored, not attended
        rows = s.feed(counts)
        s.issue(0)
        synchronize()
        _, _, slots, positions = s.model.extend(counts, s.tokens)
        v = rows.reshape(s.tokens, -1, s.hd)[:, s.heads + s.kvheads:]
        s.rows.put([x if p >= 0 else -1 for x, p in zip(slots, positions)], s.d["k"].to_host(np.float32, (s.tokens, s.kvheads, s.hd)), v)
    graphs = {}
    for count, counts in zip(RECORDED_COUNTS, ([1, 1, 1], [3, 60, 1])):
        s.step(counts, count)
        s.feed([0] * 3)
        with Graph.capture(stream) as graphs[count]:
            s.issue(count)

    def outgrow():
        b = Batch.__new__(Batch)
        b.kv, b.rows, b.group, b.tables, b.width = s.kv, s.rows, c["group"], np.array(s.model.tables), s.width
        b.counts, b.past = [OUTGROWN["count"], 299, 1], [380, 90, 4]
        b.starts = np.concatenate([[0], np.cumsum(b.counts)])
        b.q = rng.normal(size=(OUTGROWN["tokens"], s.heads, s.hd)).astype(np.float32)
        b.check(b.run(length=s.width * s.kv.page_size), rows={(r, i) for r, n in enumerate(b.counts) for i in range(0, n, 37)}, many=True)

    outgrow()
    for counts, count in (([1, 1, 1], 1), ([70, 1, 2], 130), ([1, 0, 1], 1), ([0, 0, 0], 130), ([1, 1, 0], 1), ([1, 90, 39], 130), ([1, 1, 1], 1)):
        rows = s.feed(counts)
        graphs[count].launch(stream)
        s.verify(counts, rows, count > 8)
        s.step([1, 0, 2], 2)
        if count > 8:
            outgrow()
    for g in graphs.values():
        g.close()


def test_a_capture_that_grows_the_scratch_comes_first():
    """A first call captured in a relaxed capture, which may allocate: what it captures has not run when the same call is
    made eagerly, before the graph's first replay and after it."""
    rng = np.random.default_rng(26)
    stream, lib = Stream(), _ffi.lib()
    for counts, past in (([1, 1], [3000, 900]), ([130, 1], [1200, 900])):
        b = Batch(rng, 2, 2, 64, counts, past)
        held = [upload(b.q), ints(b.starts), ints(b.past), ints(b.tables)]
        out = DeviceArray.from_host(np.full(b.q.shape, np.nan, np.float32))

        def call():
            b.kv.attention(0, held[0], out, 4, 2, len(b.q), max(counts), *held[1:], b.width, 3001, stream=stream)

        rows = {(r, i) for r, n in enumerate(counts) for i in range(0, n, 13)}
        assert lib.hipStreamBeginCapture(ct.c_void_p(stream.ptr), 2) == 0
        try:
            call()
        finally:
            g = Graph()
            g.ptr = lib.needle2_gpu_graph_end(stream.ptr)
        assert g.ptr
        for replay in (False, True, True, False):
            out.fill(0xFF)
            synchronize()
            if replay:
                g.launch(stream)
            else:
                call()
            synchronize()
            b.check(out.to_host(np.float32, b.q.shape), rows=rows, many=max(counts) > 9)
        g.close()


@pytest.mark.parametrize("counts,past", [([1, 0, 2], [20, 40, 10]), ([100, 0, 100], [20, 40, 70])])
def test_starts_outside_the_batch_are_its_ends(counts, past):
    """A negative start is the batch's first row, one past its rows their end: the requests between them as ever."""
    rng = np.random.default_rng(25)
    b = Batch(rng, 1, 2, 64, counts, past)
    right = b.starts
    for first, last in ((-5, 900), (-2 ** 31, 2 ** 31 - 1), (-1, right[-1])):
        b.starts = np.array([first, right[1], right[2], last])
        got = b.run()
        b.starts = right
        b.check(got, many=max(counts) > 9)


@pytest.mark.parametrize("n", [2, 100])
def test_a_start_behind_the_next_one(n):
    """Starts that go back: a request whose end lies before its start has no tokens, the others have the rows from their
    start to their end (a row of two of them is one's or the other's)."""
    rng = np.random.default_rng(n)
    b = Batch(rng, 1, 2, 64, [n, 0, n], [20, 40, 10])
    b.starts = np.array([0, n, n // 2, n // 2 + n])
    got = b.run()
    assert np.isnan(got[n // 2 + n:]).all() and np.isfinite(got[:n // 2 + n]).all()
    b.check(got, rows={(0, i) for i in range(n // 2)} | {(2, i) for i in range(n - n // 2, n)}, many=n > 9)


def test_two_streams_two_caches():
    """Calls of two caches at once, on streams of their own."""
    rng = np.random.default_rng(23)
    a, b = (Batch(rng, 2, 4, 128, [1, 17, 1], [900, 300, 2000]) for _ in "ab")
    streams = [Stream(), Stream()]
    outs = []
    for x, st in zip((a, b), streams):
        x.held = [upload(x.q), ints(x.starts), ints(x.past), ints(x.tables)]
        outs.append(DeviceArray.from_host(np.full(x.q.shape, np.nan, np.float32)))
    for _ in range(5):
        for x, st, out in zip((a, b), streams, outs):
            x.kv.attention(0, x.held[0], out, 8, 3, len(x.q), 17, *x.held[1:], x.width, 2100, stream=st)
    synchronize()
    for x, out in zip((a, b), outs):
        x.check(out.to_host(np.float32, x.q.shape), many=True)
