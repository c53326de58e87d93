"""Attention of many new tokens over the paged cache: prompt pieces in blocks of 128 rows, alone and beside decoding
requests, at the edges of blocks, tiles, pages and pieces. Tolerance: tests/test_paged_gpu.py (tiles of 32 positions).
"""
import numpy as np
import pytest

from openneedle_amd.device import synchronize
from tests.test_paged_gpu import Batch, ints, upload

pytestmark = pytest.mark.gpu


# (kv heads, heads of each, new tokens, positions before them): grown(...) of them are in blocks of 128 rows
SHAPES = [
    (1, 1, [65], [0]), (1, 1, [129], [31]), (2, 2, [64, 100], [0, 500]), (1, 4, [32, 33, 1, 17, 16], [7, 0, 300, 64, 31]),
    (2, 3, [43, 0, 86, 22], [1, 5, 33, 0]), (1, 8, [16, 9, 17, 8], [1000, 0, 3, 12]), (1, 16, [8, 9, 5, 4], [95, 96, 97, 0]),
    (1, 5, [1, 26, 200, 1, 13, 14], [600, 0, 32, 0, 40, 41])]


def grown(hd, group, counts):
    """More tokens for narrower rows, of which more are in blocks of 16 rows."""
    return [c * 128 // hd if c * group > 64 else c for c in counts]


def some(rng, counts, n):
    """(request, token)s: the first and last of every request, those around blocks of 128 rows, and others."""
    rows = set()
    for r, c in enumerate(counts):
        if c:
            rows |= {(r, 0), (r, c - 1)} | {(r, int(i)) for i in rng.integers(0, c, n)}
    return rows


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kvheads,group,counts,past", SHAPES)
def test_pieces_and_decoding_requests(hd, kvheads, group, counts, past):
    """Requests of few rows beside longer ones; blocks of one row and of all; fresh prompts and later pieces."""
    rng = np.random.default_rng(hd + group + sum(counts))
    counts = grown(hd, group, counts)
    b = Batch(rng, kvheads, group, hd, counts, past)
    got = b.run(tail=2)
    b.check(got[:-2], rows=some(rng, counts, 12), many=True)
    assert np.isnan(got[-2:]).all()


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 256])
def test_every_row_of_a_piece(hd, page):
    rng = np.random.default_rng(hd + page)
    b = Batch(rng, 1, 2, hd, [150], [page + 7], page=page)
    b.check(b.run(), many=True)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("window", [1, 16, 31, 32, 33, 100, 1000])
def test_window(hd, window):
    rng = np.random.default_rng(hd + window)
    counts = grown(hd, 2, [90, 1, 130])
    b = Batch(rng, 1, 2, hd, counts, [0, 700, 333], page=32)
    b.check(b.run(window), window, rows=some(rng, counts, 30), many=True)


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_pieces_of_long_contexts(hd):
    """Keys cut into pieces that are joined; row tiles with fewer pieces, requests with one, one that attends nothing."""
    rng = np.random.default_rng(hd)
    counts = grown(hd, 2, [70, 1, 2, 40])
    b = Batch(rng, 1, 2, hd, counts, [6000, 3000, -1, 20], page=64)
    for length in (0, 100, 6070, 50000):
        got = b.run(length=length)
        b.check(got, rows=some(rng, counts, 6), many=True)
        assert not got[b.starts[2]:b.starts[3]].any()
    one = Batch(rng, 1, 1, hd, [130], [9000])
    one.check(one.run(), rows=some(rng, [130], 8), many=True)
    np.testing.assert_array_equal(one.run(), one.run())


def test_one_request_of_fewer_tokens_than_announced():
    """The count is a bound: a request of one token, or of none, where up to 200 may come."""
    rng = np.random.default_rng(3)
    for n in (1, 7, 33):
        b = Batch(rng, 2, 2, 64, [n], [300])
        b.starts = np.array([0, n])
        got = b.run(count=200, tail=200)
        b.check(got[:n], many=True)
        assert np.isnan(got[n:]).all()
    b.starts = np.array([0, 0])
    assert np.isnan(b.run(count=200, tail=200)).all()


@pytest.mark.parametrize("requests", [63, 64, 65, 300, 512, 513, 700])
def test_many_requests(requests):
    """Blocks find their requests among more than a wave looks at at once; most of them have no tokens, or few; some are of
    the same length, one is padded."""
    rng = np.random.default_rng(requests)
    counts = [int(c) for c in rng.choice([0, 1, 2, 3], requests)]
    for r in rng.choice(requests, 5, replace=False):
        counts[r] = int(rng.integers(193, 400))
    counts[0], counts[-1] = 210, 299
    past = [int(p) for p in rng.integers(0, 40, requests)]
    counts[20:23], past[20:23] = [257] * 3, [33] * 3
    counts[40], past[40] = 250, -3
    b = Batch(rng, 1, 1, 32, counts, past)
    big = {(r, i) for r, c in enumerate(counts) if c > 60 for i in (0, 31, 64, c - 1)}
    small = {(r, i) for r, c in enumerate(counts[:60]) if c <= 60 for i in range(c)}
    b.check(b.run(), rows=big | small, many=True)


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_pages_that_are_none(hd):
    rng = np.random.default_rng(hd)
    counts = grown(hd, 2, [80, 70, 66])
    b = Batch(rng, 1, 2, hd, counts, [200, 0, 40])
    assert b.tables.shape[1] > 12
    whole = b.tables.copy()
    holes = [(0, 3), (0, 4), (0, 12), (1, 0), (1, 4)]
    for i, at in enumerate(holes):
        b.tables[at] = (-1, 2 ** 31 - 1, 10 ** 6, -2 ** 31, b.kv.pages)[i]
    b.tables[2] = -1
    got = b.run()
    assert not got[b.starts[2]:].any()
    gone = {int(whole[at]) for at in holes} | {int(x) for x in whole[2] if x >= 0}
    b.tables = whole
    b.check(got, gone=gone, rows=some(rng, counts[:2], 40), many=True)


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_zero_rows_and_uneven_values(hd):
    """V rows of zeros, whose scale is 1, far above the others'; V scales that differ by powers of two; scores far apart;
    entries of q far above the rest over zero K codes."""
    rng = np.random.default_rng(hd)
    b = Batch(rng, 1, 2, hd, grown(hd, 2, [70, 1]), [150, 90])
    zero = rng.random(b.rows.vs.shape) < 0.1
    b.rows.v[zero], b.rows.vs[zero] = 0, 1.0
    b.rows.vs[~zero] *= 2.0 ** -rng.integers(0, 20, (~zero).sum())
    b.rows.k[..., 5] = 0
    b.rows.push()
    b.q *= 4
    b.q[::3, :, 5] = 1e8
    b.check(b.run(), many=True)


def test_offsets_past_32_bits():
    """A prompt piece whose pages lie on both sides of 4 GiB of a layer."""
    import oracle
    from openneedle_amd.paged import PagedCache
    rng = np.random.default_rng(5)
    kv = PagedCache(1, 140000, 16, 16, 128)  # 9.5 GB
    pages = np.array([139999, 3, 70000, 64000, 139000, 1, 2, 99999, 0])
    n = 16 * len(pages) - 20
    slots = pages[np.arange(n + 20) // 16] * 16 + np.arange(n + 20) % 16
    k, v = (rng.normal(size=(n + 20, 16, 128)).astype(np.float32) for _ in "kv")
    kv.store(0, upload(k), upload(v), n + 20, ints(slots))
    q = rng.normal(size=(n, 16, 128)).astype(np.float32)
    out = upload(np.zeros_like(q))
    kv.attention(0, upload(q), out, 16, 1, n, n, ints([0, n]), ints([20]), ints(pages), len(pages))
    synchronize()
    got = out.to_host(np.float32, q.shape)
    kd, vd = (np.stack([c.astype(np.float64) * s[..., None] for c, s in (oracle.kv_quantize(r[None]) for r in x)]) for x in (k, v))
    from tests.test_span_gpu import attend, check
    for i in (0, 5, 63, n - 1):
        for h in (0, 7, 15):
            kk, vv = kd.reshape(n + 20, 16, 128)[:21 + i, h], vd.reshape(n + 20, 16, 128)[:21 + i, h]
            want, tol, _ = attend(q[i, h], kk, vv)
            check(got[i, h], want, tol + 2.0 ** -27 * np.abs(vv).max(), f"token {i} head {h}")
